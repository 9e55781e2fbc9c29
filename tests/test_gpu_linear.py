"""The row-by-row form of linear attention with one decay a head, against the recurrence in 64 bits (bounds in linear_oracle.py)."""
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


def offsets(lens, heads):
    return torch.arange(len(lens), dtype=torch.int64, device="cuda") * (heads * 128 * 128)


def check(got, want, bound):
    far = (got.double() - want).abs() - bound
    assert bool((far <= 0).all()), float(far.max())


CASES = [
    # lens, heads, qk_heads, state, decay, size
    ([1], 1, 1, "f32", "token", 1.0),
    ([1, 1, 1], 3, 1, "bf16", "head", 0.1),
    ([4, 1, 0, 7, 16], 5, 5, "f32", "token", 0.1),
    ([8, 3, 2], 6, 2, "bf16", "token", 3.0),
    ([65], 2, 2, "bf16", "head", 0.02),
]


@pytest.mark.parametrize("lens,heads,qk_heads,state,decay,size", CASES)
@pytest.mark.parametrize("write", [True, False])
def test_rows_against_64_bits(lin, lens, heads, qk_heads, state, decay, size, write):
    q, k, v, g, s = lo.inputs(lens, heads, qk_heads, 3, "cuda", decay, size)
    s = s.to(torch.float32 if state == "f32" else torch.bfloat16)
    rows = sum(lens)
    out = torch.full((rows + 2, heads, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    before = s.clone()
    so = torch.full_like(s, 9.0) if write else None
    lin.decode_batch(heads, rows, lo.cu_of(lens, "cuda"), q, k, v, g, s, offsets(lens, heads), qk_heads=qk_heads, state_out=so, scale=0.25, out=out)
    y, ends, yb, endb = lo.recurrence(lens, q, k, v, g, s, 0.25, state == "bf16")
    check(out[:rows], y, yb)
    assert (out[rows:] == 7.0).all() and torch.equal(s, before)
    if write:
        check(so, ends, endb)


@pytest.mark.parametrize("state", ["f32", "bf16"])
def test_windows_are_single_rows_bit_for_bit(lin, state):
    """One call over a window, a verify and a commit of k rows, and k single-row calls: the same outputs and states."""
    lens, heads = [5, 16, 3], 4
    q, k, v, g, s = lo.inputs(lens, heads, 2, 5, "cuda")
    s = s.to(torch.float32 if state == "f32" else torch.bfloat16)
    rows, cu, off = sum(lens), lo.cu_of(lens, "cuda"), offsets(lens, heads)
    out = torch.zeros(rows, heads, 128, dtype=torch.bfloat16, device="cuda")
    lin.decode_batch(heads, rows, cu, q, k, v, g, s, off, qk_heads=2, state_out=None, out=out)
    keep = [2, 16, 1]
    kept = s.clone()
    lin.decode_batch(heads, rows, cu, q, k, v, g, kept, off, qk_heads=2, keep=torch.tensor(keep, dtype=torch.int32, device="cuda"))
    serial, one = s.clone(), torch.zeros_like(out)
    first = 0
    for b, n in enumerate(lens):
        for t in range(keep[b]):
            at = slice(first + t, first + t + 1)
            lin.decode_batch(heads, 1, lo.cu_of([1], "cuda"), q[at], k[at], v[at], g[at], serial, off[b:b + 1], qk_heads=2, out=one[at])
        assert torch.equal(out[first:first + keep[b]], one[first:first + keep[b]])
        first += n
    assert torch.equal(kept, serial)


@pytest.mark.parametrize("state", ["f32", "bf16"])
def test_strided_rows_shared_offsets_and_unaligned_states(lin, state):
    """q, k, v as parts of one projection's rows, a pool of states in any order and at any element, gates in a wider tensor."""
    lens, heads = [2, 4], 3
    q, k, v, g, s = lo.inputs(lens, heads, heads, 7, "cuda")
    rows, width = 6, heads * 128
    fused = torch.full((rows, 3 * width + 40), 5.0, dtype=torch.bfloat16, device="cuda")
    parts = [fused[:, i * width:(i + 1) * width] for i in range(3)]
    for part, t in zip(parts, (q, k, v)):
        part.copy_(t.reshape(rows, width))
    wide = torch.zeros(rows, heads + 5, device="cuda")
    wide[:, 2:2 + heads] = g
    per = heads * 128 * 128
    pool = torch.zeros(3 * per + 3, dtype=torch.float32 if state == "f32" else torch.bfloat16, device="cuda")
    off = torch.tensor([2 * per + 3, 1], dtype=torch.int64, device="cuda")
    for b in range(2):
        pool[int(off[b]):int(off[b]) + per] = s[b].reshape(-1).to(pool.dtype)
    want_in = torch.stack([pool[int(o):int(o) + per].view(heads, 128, 128) for o in off.cpu()])
    y, ends, yb, endb = lo.recurrence(lens, q, k, v, g, want_in, 128 ** -0.5, state == "bf16")
    big = torch.zeros(rows, 2 * width, dtype=torch.bfloat16, device="cuda")
    guard = pool.clone()
    lin.decode_batch(heads, rows, lo.cu_of(lens, "cuda"), *parts, wide[:, 2:2 + heads], pool, off, out=big[:, width:])
    check(big[:, width:].reshape(rows, heads, 128), y, yb)
    assert (big[:, :width] == 0).all()
    for b in range(2):
        o = int(off[b])
        check(pool[o:o + per].view(heads, 128, 128), ends[b], endb[b])
        guard[o:o + per] = pool[o:o + per]
    assert torch.equal(pool, guard)


def test_a_decay_of_minus_infinity_forgets(lin):
    lens, heads = [3], 2
    q, k, v, g, s = lo.inputs(lens, heads, heads, 9, "cuda")
    g[1] = -float("inf")
    out = torch.empty(3, heads, 128, dtype=torch.bfloat16, device="cuda")
    so = torch.empty_like(s)
    lin.decode_batch(heads, 3, lo.cu_of(lens, "cuda"), q, k, v, g, s, offsets(lens, heads), state_out=so, out=out)
    y, ends, yb, endb = lo.recurrence(lens, q, k, v, g, s, 128 ** -0.5, False)
    check(out, y, yb)
    check(so, ends, endb)


def test_another_stream_and_a_replayed_graph(lin):
    lens, heads = [1] * 4, 8
    q, k, v, g, s = lo.inputs(lens, heads, 4, 11, "cuda")
    cu, off = lo.cu_of(lens, "cuda"), offsets(lens, heads)
    want_s, want = s.clone(), torch.empty(4, heads, 128, dtype=torch.bfloat16, device="cuda")
    for _ in range(3):
        lin.decode_batch(heads, 4, cu, q, k, v, g, want_s, off, qk_heads=4, out=want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got_s, got = s.clone(), torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        lin.decode_batch(heads, 4, cu, q, k, v, g, got_s, off, qk_heads=4, out=got)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(got_s, want_s)
