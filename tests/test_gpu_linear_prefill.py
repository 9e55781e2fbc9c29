"""The chunked prefill of linear attention with one decay a head, against the recurrence in 64 bits (bounds in linear_oracle.py)."""
import importlib

import pytest

import linear_oracle as lo

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lin():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return importlib.import_module("glm53f-afd_b200.linear")


def status():
    torch.cuda.synchronize()
    return importlib.import_module("glm53f-afd_b200.core").device_status()


def offsets(lens, heads):
    return torch.arange(len(lens), dtype=torch.int64, device="cuda") * (heads * 128 * 128)


def check(got, want, bound):
    far = (got.double() - want).abs() - bound
    assert bool((far <= 0).all()), float(far.max())


def workspace(lin, heads, batch, max_len):
    return torch.empty(max(16, lin.prefill_workspace_bytes(heads, batch, max_len)), dtype=torch.uint8, device="cuda")


CASES = [
    # lens, heads, qk_heads, state, decay, size
    ([9], 1, 1, "f32", "token", 0.1),
    ([64], 1, 1, "f32", "token", 1.0),
    ([65], 2, 1, "bf16", "head", 0.05),
    ([1, 63, 64, 65, 0, 130], 3, 3, "f32", "token", 0.02),
    ([200, 17, 128, 2], 4, 2, "bf16", "token", 0.3),
    ([300], 2, 2, "f32", "token", 6.0),
    ([500], 1, 1, "f32", "head", 0.0),
]


@pytest.mark.parametrize("lens,heads,qk_heads,state,decay,size", CASES)
def test_against_64_bits(lin, lens, heads, qk_heads, state, decay, size):
    q, k, v, g, s = lo.inputs(lens, heads, qk_heads, 3, "cuda", decay, size)
    s = s.to(torch.float32 if state == "f32" else torch.bfloat16)
    rows = sum(lens)
    out = torch.full((rows + 70, heads, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    so, before = torch.full_like(s, 9.0), s.clone()
    lin.prefill_varlen(heads, rows, lo.cu_of(lens, "cuda"), max(lens), q, k, v, g, s, offsets(lens, heads), qk_heads=qk_heads, state_out=so, scale=0.5, out=out)
    assert status() == 0
    y, ends, yb, endb = lo.chunked(lens, q, k, v, g, s, 0.5, state == "bf16")
    check(out[:rows], y, yb)
    check(so, ends, endb)
    assert (out[rows:] == 7.0).all() and torch.equal(s, before)
    lin.prefill_varlen(heads, rows, lo.cu_of(lens, "cuda"), max(lens), q, k, v, g, s, offsets(lens, heads), qk_heads=qk_heads, scale=0.5, out=out)
    assert torch.equal(s, so)


@pytest.mark.parametrize("lens,heads,state", [([1100, 70, 0, 600], 2, "f32"), ([4000], 1, "bf16")])
def test_segments(lin, lens, heads, state):
    """Few chains over a workspace: several segments at once; in place, into other states, and with a workspace that is too small for any."""
    q, k, v, g, s = lo.inputs(lens, heads, heads, 5, "cuda", "token", 0.01)
    s = s.to(torch.float32 if state == "f32" else torch.bfloat16)
    rows, cu, off = sum(lens), lo.cu_of(lens, "cuda"), offsets(lens, heads)
    ws = workspace(lin, heads, len(lens), max(lens))
    assert ws.numel() > 2 * heads * len(lens) * 65536
    y, ends, yb, endb = lo.chunked(lens, q, k, v, g, s, 0.5, state == "bf16")
    results = []
    for w in (ws, ws[:heads * len(lens) * 65536 * 2 + 1024], ws[:16], None):
        out, own = torch.full((rows + 64, heads, 128), 7.0, dtype=torch.bfloat16, device="cuda"), s.clone()
        lin.prefill_varlen(heads, rows, cu, max(lens), q, k, v, g, own, off, scale=0.5, out=out, workspace=w)
        assert status() == 0
        check(out[:rows], y, yb)
        check(own, ends, endb)
        assert (out[rows:] == 7.0).all()
        other = torch.full_like(s, 9.0)
        lin.prefill_varlen(heads, rows, cu, max(lens), q, k, v, g, s, off, state_out=other, scale=0.5, out=out, workspace=w)
        assert torch.equal(own, other)
        results.append((out, own))
    assert torch.equal(results[2][0], results[3][0]) and torch.equal(results[2][1], results[3][1])


def test_strided_rows_and_unaligned_states(lin):
    lens, heads = [100, 33], 3
    for state in (torch.float32, torch.bfloat16):
        q, k, v, g, s = lo.inputs(lens, heads, heads, 7, "cuda", "token", 0.05)
        rows, width = sum(lens), heads * 128
        fused = torch.full((rows, 3 * width + 40), float("nan"), dtype=torch.bfloat16, device="cuda")
        parts = [fused[:, i * width:(i + 1) * width] for i in range(3)]
        for part, t in zip(parts, (q, k, v)):
            part.copy_(t.reshape(rows, width))
        wide = torch.zeros(rows, heads + 5, device="cuda")
        wide[:, 2:2 + heads] = g
        per = heads * 128 * 128
        pool = torch.zeros(3 * per + 3, dtype=state, device="cuda")
        off = torch.tensor([2 * per + 3, 1], dtype=torch.int64, device="cuda")
        for b in range(2):
            pool[int(off[b]):int(off[b]) + per] = s[b].reshape(-1).to(state)
        first = torch.stack([pool[int(o):int(o) + per].view(heads, 128, 128) for o in off.cpu()])
        y, ends, yb, endb = lo.chunked(lens, q, k, v, g, first, 128 ** -0.5, state == torch.bfloat16)
        big = torch.zeros(rows, 2 * width, dtype=torch.bfloat16, device="cuda")
        guard = pool.clone()
        lin.prefill_varlen(heads, rows, lo.cu_of(lens, "cuda"), 100, *parts, wide[:, 2:2 + heads], pool, off, out=big[:, width:])
        assert status() == 0
        check(big[:, width:].reshape(rows, heads, 128), y, yb)
        assert (big[:, :width] == 0).all()
        for b in range(2):
            o = int(off[b])
            check(pool[o:o + per].view(heads, 128, 128), ends[b], endb[b])
            guard[o:o + per] = pool[o:o + per]
        assert torch.equal(pool, guard)


def test_another_sequences_nan_stays_there(lin):
    """Chunks reach over a sequence's end: what lies behind must not come in, whatever it is."""
    lens, heads = [40, 90, 70], 2
    q, k, v, g, s = lo.inputs(lens, heads, heads, 9, "cuda", "token", 0.1)
    y, ends, yb, endb = lo.chunked(lens, q, k, v, g, s, 1.0, False)
    for bad in (float("nan"), float("inf")):
        q2, k2, v2, g2, s2 = (t.clone() for t in (q, k, v, g, s))
        for t in (q2, k2, v2, g2):
            t[40:130] = bad
        s2[1] = bad
        out = torch.empty(200, heads, 128, dtype=torch.bfloat16, device="cuda")
        lin.prefill_varlen(heads, 200, lo.cu_of(lens, "cuda"), 90, q2, k2, v2, g2, s2, offsets(lens, heads), scale=1.0, out=out)
        assert status() == 0
        for a, b in ((0, 40), (130, 200)):
            check(out[a:b], y[a:b], yb[a:b])
        for i in (0, 2):
            check(s2[i], ends[i], endb[i])


@pytest.mark.parametrize("at", [0, 1, 30, 63, 64, 90])
def test_a_decay_of_minus_infinity_forgets(lin, at):
    """Nothing of before the row is left, and the rows behind it are as exact as ever."""
    lens, heads = [100], 2
    q, k, v, g, s = lo.inputs(lens, heads, heads, 11, "cuda", "token", 0.1)
    g[at, 0] = -float("inf")
    g[at, 1] = -5000.0
    v[:at] *= 1e3
    out, so = torch.empty(100, heads, 128, dtype=torch.bfloat16, device="cuda"), torch.empty_like(s)
    lin.prefill_varlen(heads, 100, lo.cu_of(lens, "cuda"), 100, q, k, v, g, s, offsets(lens, heads), state_out=so, scale=1.0, out=out)
    g[at] = -1e9
    y, ends, yb, endb = lo.chunked(lens, q, k, v, g, s, 1.0, False)
    check(out, y, yb)
    check(so, ends, endb)


def test_prompt_then_steps(lin):
    """A prompt through the prefill, further rows through the row-by-row form, against one recurrence over all of them."""
    heads, n, more = 4, 150, 6
    q, k, v, g, s = lo.inputs([n + more], heads, 2, 13, "cuda", "token", 0.05)
    out, state = torch.empty(n + more, heads, 128, dtype=torch.bfloat16, device="cuda"), s.clone()
    off = offsets([1], heads)
    lin.prefill_varlen(heads, n, lo.cu_of([n], "cuda"), n, q, k, v, g, state, off, qk_heads=2, out=out[:n])
    for t in range(n, n + more):
        at = slice(t, t + 1)
        lin.decode_batch(heads, 1, lo.cu_of([1], "cuda"), q[at], k[at], v[at], g[at], state, off, qk_heads=2, out=out[at])
    y, ends, yb, endb = lo.chunked([n + more], q, k, v, g, s, 128 ** -0.5, False)
    check(out, y, yb)
    check(state, ends, endb[:] * 1.1)  # (the steps' own roundings: under 6 x 6 half steps beside the 276 counted)


def test_another_stream_and_a_replayed_graph(lin):
    lens, heads = [700, 90], 2
    q, k, v, g, s = lo.inputs(lens, heads, 1, 15, "cuda", "head", 0.01)
    cu, off, rows = lo.cu_of(lens, "cuda"), offsets(lens, heads), sum(lens)
    ws = workspace(lin, heads, 2, 700)
    want, want_s = torch.empty(rows, heads, 128, dtype=torch.bfloat16, device="cuda"), s.clone()
    for _ in range(3):
        lin.prefill_varlen(heads, rows, cu, 700, q, k, v, g, want_s, off, qk_heads=1, out=want, workspace=ws)
    torch.cuda.synchronize()
    got, got_s = torch.empty_like(want), s.clone()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        lin.prefill_varlen(heads, rows, cu, 700, q, k, v, g, got_s, off, qk_heads=1, out=got, workspace=ws)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(got_s, want_s)
