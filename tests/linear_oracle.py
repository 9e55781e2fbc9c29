"""Linear attention with one decay a head in 64 bits, with the bounds that the kernels' roundings allow: S_t = e^g_t S_{t-1} + v_t k_t^T,
y_t = scale S_t q_t.  Tensors are torch, on any device."""
import torch

U32 = 2.0 ** -24    # half a step of f32, relative
UBF = 2.0 ** -8     # half a step of bf16, relative


def recurrence(lens, q, k, v, g, state, scale, round_rows):
    """Outputs, end states and how far a row-by-row kernel may be from either: (y, S, bound of y, bound of S).

    The kernel forms e^g to two steps of f32 (its exponential's bound), S with one rounding in f32 and, `round_rows`, one to bf16 a row; a sum of 128
    products in f32 loses at most 130 roundings of the sum of their magnitudes; y is rounded to bf16 once."""
    rows, heads, d = v.shape
    share = heads // q.shape[1]
    q, k = (t.double().repeat_interleave(share, 1) for t in (q, k))
    v, g = v.double(), g.double().expand(rows, heads)
    y, yb = (torch.zeros(rows, heads, d, dtype=torch.float64, device=v.device) for _ in range(2))
    ends, endb = [], []
    first = 0
    for b, n in enumerate(lens):
        s = state[b].double()
        e = torch.zeros_like(s)
        for t in range(first, first + n):
            decay = torch.exp(g[t])[:, None, None]
            kept = torch.where(decay > 0, decay * s, 0.0)
            carried = torch.where(decay > 0, decay * e, 0.0)
            s = kept + v[t][:, :, None] * k[t][:, None, :]
            e = carried + 4 * U32 * kept.abs() + U32 * s.abs()
            if round_rows:
                e = e + UBF * (s.abs() + e)
            dot = (s * q[t][:, None, :])
            y[t] = scale * dot.sum(-1)
            at = abs(scale) * ((e * q[t][:, None, :].abs()).sum(-1) + 130 * U32 * (dot.abs() + e * q[t][:, None, :].abs()).sum(-1))
            yb[t] = at + (UBF + U32) * (y[t].abs() + at) + 1e-38
        ends.append(s)
        endb.append(e)
        first += n
    return y, torch.stack(ends), yb, torch.stack(endb) + 1e-38


def inputs(lens, heads, qk_heads, seed, device, decay="token", size=1.0):
    gen = torch.Generator().manual_seed(seed)
    rows = sum(lens)
    q, k = (torch.nn.functional.normalize(torch.randn(rows, qk_heads, 128, generator=gen), dim=-1).bfloat16() for _ in range(2))
    v = torch.randn(rows, heads, 128, generator=gen).bfloat16()
    if decay == "token":
        g = -size * torch.nn.functional.softplus(torch.randn(rows, heads, generator=gen))
    else:
        g = -size * torch.rand(heads, generator=gen)
    state = 0.5 * torch.randn(len(lens), heads, 128, 128, generator=gen)
    return [t.to(device) for t in (q, k, v, g, state)]


def cu_of(lens, device):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=device)


def chunked(lens, q, k, v, g, state, scale, bf16_state):
    """The same, with the bounds of the chunked form.  M, the recurrence of the magnitudes, is what every rounding is relative to: products of
    bf16 are exact; a chunk's sums of up to 64 terms (and the scores' of 128) in the tensor core's f32 lose at most four half steps a term; a factor's
    exponential and the sums of log decays eight; a chunk that passes over an older one's sums six.  w V is exact to f32 in three parts (24 bits), to 2^-16
    in two; P as an operand is exact to 2^-16 (two roundings of bf16: 2^-8 of 2^-8); of S and of the scaled q the tensor core takes 11 bits, cut off: 2^-10 of what
    came into the chunk from before it, each."""
    rows, heads, d = v.shape
    share = heads // q.shape[1]
    q, k = (t.double().repeat_interleave(share, 1) for t in (q, k))
    v, g = v.double(), g.double().expand(rows, heads)
    y, yb = (torch.zeros(rows, heads, d, dtype=torch.float64, device=v.device) for _ in range(2))
    ends, endb = [], []
    first = 0
    for b, n in enumerate(lens):
        s = state[b].double()
        m = s.abs()
        part = (4 * 64 + 8 + 6 * ((n + 63) // 64)) * U32 + (UBF * UBF if bf16_state else 4 * U32)
        for t in range(first, first + n):
            decay = torch.exp(g[t])[:, None, None]
            if (t - first) % 64 == 0:
                before = m
            before = decay * before
            s = decay * s + v[t][:, :, None] * k[t][:, None, :]
            m = decay * m + (v[t][:, :, None] * k[t][:, None, :]).abs()
            y[t] = scale * (s * q[t][:, None, :]).sum(-1)
            at = abs(scale) * ((m * (part + UBF * UBF + (4 * 128 + 4 * 64 + 16) * U32) + before * 2.0 ** -9) * q[t][:, None, :].abs()).sum(-1)
            yb[t] = at + (UBF + U32) * (y[t].abs() + at) + 1e-38
        e = part * m
        ends.append(s)
        endb.append(e + (UBF if bf16_state else U32) * (s.abs() + e) + 1e-38)
        first += n
    return y, torch.stack(ends), yb, torch.stack(endb)
