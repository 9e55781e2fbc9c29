"""The gated linear recurrence and its gradients in 64 bits, row by row, and how far f32 arithmetic may be from them.

Bounds.  With u = 2^-24: a gate a and its complement are formed to within 6 u of themselves (an exponential to one unit in the last place, 2 u; the sigmoid's
reciprocal and products add 4 u), each multiplication and addition of the recurrence adds u.  To first order the error of h_t is then at most 10 u times the
sum over its contributions of (the steps each went through + 2), which the recurrences H_t = a_t H_{t-1} + |b_t| and N_t = a_t (N_{t-1} + H_{t-1}) give."""
import torch

U = 2.0 ** -24


def half_step(t, dtype):
    """Half a step of `dtype` at t, and of its smallest normal number."""
    f = torch.finfo(dtype)
    return t.abs().clamp(min=f.tiny) * (f.eps / 2)


def gates(g, gate, input):
    g = g.double()
    if gate == "decay":
        a, rest, slope = torch.exp(g), -torch.expm1(g), torch.exp(g)
    else:
        a, rest = torch.sigmoid(g), torch.sigmoid(-g)
        slope = a * rest
    return a, rest if input == "complement" else torch.ones_like(a), slope


def rows(a, b, h, mag, steps):
    """All h_t of h_t = a_t h_{t-1} + b_t and the bound of each one's error; `mag` and `steps` are those of the starting state."""
    out, bound = [], []
    for t in range(a.shape[0]):
        steps = a[t] * (steps + mag)
        mag = a[t] * mag + b[t].abs()
        h = a[t] * h + b[t]
        out.append(h)
        bound.append(10 * U * (steps + 2 * mag))
    if not out:
        return a, a
    return torch.stack(out), torch.stack(bound)


def forward(lens, g, x, state, gate, input):
    """(h, bound, end states, their bound) of packed rows g, x [rows][channels] and states [batch][channels]."""
    hs, bs, ends, ebs = [], [], [], []
    first = 0
    for i, n in enumerate(lens):
        a, c, _ = gates(g[first:first + n], gate, input)
        s = state[i].double()
        h, b = rows(a, c * x[first:first + n].double(), s, s.abs(), torch.zeros_like(s))
        hs.append(h), bs.append(b)
        ends.append(h[-1] if n else s), ebs.append(b[-1] if n else torch.zeros_like(s))
        first += n
    return torch.cat(hs), torch.cat(bs), torch.stack(ends), torch.stack(ebs)


def backward(lens, g, x, state, dout, dstate, gate, input):
    """[(value, bound)] of dg, dx and the start states' gradient."""
    dgs, dxs, dss = [], [], []
    first = 0
    for i, n in enumerate(lens):
        at = slice(first, first + n)
        first += n
        after = dstate[i].double() if dstate is not None else torch.zeros_like(state[i]).double()
        if n == 0:
            dss.append((after, torch.zeros_like(after)))
            dgs.append((g[at].double(), g[at].double())), dxs.append((x[at].double(), x[at].double()))  # none
            continue
        a, c, slope = gates(g[at], gate, input)
        xd, s = x[at].double(), state[i].double()
        h, hb = rows(a, c * xd, s, s.abs(), torch.zeros_like(s))
        before, before_b = torch.cat([s[None], h[:-1]]), torch.cat([torch.zeros_like(s)[None], hb[:-1]])
        step = torch.cat([torch.ones_like(a[:1]), a.flip(0)[:-1]])
        d, db = rows(step, dout[at].double().flip(0), after, after.abs(), torch.zeros_like(after))
        d, db = d.flip(0), db.flip(0)
        other = xd if input == "complement" else torch.zeros_like(xd)
        inner = before - other
        dgs.append((d * slope * inner, slope * (db * inner.abs() + d.abs() * before_b) + 16 * U * d.abs() * slope * (before.abs() + other.abs())))
        dxs.append((c * d, c * db + 8 * U * (c * d).abs()))
        dss.append((a[0] * d[0], a[0] * db[0] + 10 * U * (a[0] * d[0]).abs()))
    cat = lambda parts: tuple(torch.cat([p[j] for p in parts]) for j in range(2))
    return cat(dgs), cat(dxs), tuple(torch.stack([p[j] for p in dss]) for j in range(2))


def close(got, want, bound, what=""):
    """Within the bound and one rounding to got's type."""
    over = (got.double() - want).abs() - (1.01 * bound + half_step(want.abs() + bound, got.dtype))
    assert not torch.isnan(got).any(), what
    assert (over <= 0).all(), over.numel() and f"{what}: {int((over > 0).sum())} values, the worst by {float(over.max()):.3g} of {float(want.flatten()[over.argmax()]):.3g}"
