"""Linear attention and the verification of drafted tokens at the edges of what their documentation allows: offsets beyond 32 bits, calls beside one another, a state that
several requests read, sequences of every kind of length in one batch."""
import importlib

import pytest

import linear_oracle as lo
from test_gpu_accept import rule

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
PER = 128 * 128


@pytest.fixture(scope="module")
def mods():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return {n: importlib.import_module("glm53f-afd_b200." + n) for n in ("core", "linear", "spec")}


def status(mods):
    torch.cuda.synchronize()
    return mods["core"].device_status()


@pytest.mark.parametrize("prefill", [False, True])
def test_rows_and_states_beyond_32_bits(mods, prefill):
    """Rows 2^24 + 8 elements apart, a state that begins 2^31 elements in: the same bits as close together."""
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    lens, heads, far = [130], 1, (1 << 24) + 8
    q, k, v, g, s = lo.inputs(lens, heads, heads, 11, "cuda", "token", 0.05)
    rows, cu = 130, lo.cu_of(lens, "cuda")
    wide = torch.zeros(rows * far, dtype=torch.bfloat16, device="cuda")
    apart = [wide.as_strided((rows, 128), (far, 1), 128 * i) for i in range(4)]
    for a, t in zip(apart, (q, k, v)):
        a.copy_(t.reshape(rows, 128))
    states = torch.zeros((1 << 31) + 2 * PER, dtype=torch.bfloat16, device="cuda")
    off = torch.tensor([(1 << 31) + 40], dtype=torch.int64, device="cuda")
    own = s.reshape(-1).bfloat16()
    states[int(off):int(off) + PER] = own
    out, at0 = torch.zeros(rows, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    near = own.clone()
    if prefill:
        mods["linear"].prefill_varlen(heads, rows, cu, rows, *apart[:3], g, states, off, out=apart[3])
        mods["linear"].prefill_varlen(heads, rows, cu, rows, q, k, v, g, near, at0, out=out)
    else:
        mods["linear"].decode_batch(heads, rows, cu, *apart[:3], g, states, off, out=apart[3])
        mods["linear"].decode_batch(heads, rows, cu, q, k, v, g, near, at0, out=out)
    assert status(mods) == 0
    assert torch.equal(apart[3], out) and torch.equal(states[int(off):int(off) + PER], near)
    assert not states[:int(off)].any() and not states[int(off) + PER:].any()


def test_judged_rows_beyond_32_bits(mods):
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GB")
    rows, vocab, far = 9, 1003, 1 << 28
    gen = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.zeros(rows * far, dtype=torch.bfloat16, device="cuda")
    target = wide.as_strided((rows, vocab), (far, 1), 5)
    target.copy_((torch.randn(rows, vocab, device="cuda", generator=gen) * 3).bfloat16())
    u = torch.rand(rows, device="cuda", generator=gen) * 0.9
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    tokens[1:] = target.float().argmax(-1)[:-1].int()
    lens, heat = [1, 8], torch.tensor([1.0, 0.0], device="cuda")
    keep, nxt = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    mods["spec"].accept_batch(lo.cu_of(lens, "cuda"), tokens, target, u, keep, nxt, temperature=heat)
    assert status(mods) == 0
    assert (keep.tolist(), nxt.tolist()) == rule(lens, tokens, target, u, False, None, heat) and keep.tolist() == [1, 8]


def test_calls_beside_one_another(mods):
    """Two prefills in segments and two rounds of judging on two streams, each with its own workspace: the bits of the same calls alone, time after time."""
    lin, spec, heads, lens = mods["linear"], mods["spec"], 3, [2100, 500]
    rows, cu = sum(lens), lo.cu_of(lens, "cuda")
    off = torch.arange(2, dtype=torch.int64, device="cuda") * (heads * PER)
    jobs = []
    for seed in (1, 2):
        q, k, v, g, s = lo.inputs(lens, heads, heads, seed, "cuda", "token", 0.02)
        ws = torch.empty(lin.prefill_workspace_bytes(heads, 2, max(lens)), dtype=torch.uint8, device="cuda")
        assert ws.numel() > 0
        gen = torch.Generator(device="cuda").manual_seed(seed)
        target = torch.randn(24, 20000, device="cuda", generator=gen) * 2
        tokens, u = torch.randint(0, 20000, (24,), dtype=torch.int32, device="cuda", generator=gen), torch.rand(24, device="cuda", generator=gen) * 0.99
        jobs.append((q, k, v, g, s, ws, target, tokens, u))
    windows = lo.cu_of([8, 8, 8], "cuda")

    def run(job):
        q, k, v, g, s, ws, target, tokens, u = job
        so, out = torch.empty_like(s), torch.empty(rows, heads, 128, dtype=torch.bfloat16, device="cuda")
        keep, nxt = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
        lin.prefill_varlen(heads, rows, cu, max(lens), q, k, v, g, s, off, state_out=so, out=out, workspace=ws)
        spec.accept_batch(windows, tokens, target, u, keep, nxt)
        return so, out, keep, nxt

    alone = []
    for job in jobs:
        alone.append(run(job))
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(5):
        together = []
        torch.cuda.synchronize()
        for stream, job in zip(streams, jobs):
            with torch.cuda.stream(stream):
                together.append(run(job))
        torch.cuda.synchronize()
        for got, want in zip(together, alone):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert status(mods) == 0


def test_requests_that_read_one_state(mods):
    """Windows that branch off the same state, which stays as it is."""
    lens, heads = [3, 8, 1, 5], 2
    q, k, v, g, s = lo.inputs(lens, heads, heads, 5, "cuda", "token", 0.1)
    state, rows = s[:1].contiguous(), sum(lens)
    off, before = torch.zeros(4, dtype=torch.int64, device="cuda"), s[:1].clone()
    out = torch.empty(rows, heads, 128, dtype=torch.bfloat16, device="cuda")
    mods["linear"].decode_batch(heads, rows, lo.cu_of(lens, "cuda"), q, k, v, g, state, off, state_out=None, out=out)
    first = 0
    for n in lens:
        one, part = torch.empty(n, heads, 128, dtype=torch.bfloat16, device="cuda"), slice(first, first + n)
        mods["linear"].decode_batch(heads, n, lo.cu_of([n], "cuda"), q[part], k[part], v[part], g[part], state, off[:1], state_out=None, out=one)
        assert torch.equal(one, out[part])
        first += n
    assert status(mods) == 0 and torch.equal(state, before)


@pytest.mark.parametrize("lens,heads,max_len", [([0] * 40 + [700, 3, 64] * 3 + [1] * 30, 2, 700), ([5000] + [40] * 70, 1, 5000), ([300, 4200, 0, 129], 4, 4200), ([2000, 900], 3, 5)])
def test_many_lengths_in_one_batch(mods, lens, heads, max_len):
    """More sequences than a warp's lanes, empty ones, a long one among short ones in segments, and a longest length that was given too small."""
    q, k, v, g, s = lo.inputs(lens, heads, heads, 9, "cuda", "token", 0.02)
    rows, batch = sum(lens), len(lens)
    off = torch.arange(batch, dtype=torch.int64, device="cuda").flip(0) * (heads * PER)
    size = mods["linear"].prefill_workspace_bytes(heads, batch, max(lens))
    ws = torch.empty(size, dtype=torch.uint8, device="cuda") if size else None
    out, so = torch.full((rows + 64, heads, 128), 7.0, dtype=torch.bfloat16, device="cuda"), torch.full_like(s, 9.0)
    mods["linear"].prefill_varlen(heads, rows, lo.cu_of(lens, "cuda"), max_len, q, k, v, g, s, off, state_out=so, scale=0.5, out=out, workspace=ws)
    assert status(mods) == 0
    y, ends, yb, endb = (lo.recurrence if max_len <= 8 else lo.chunked)(lens, q, k, v, g, s.flip(0), 0.5, False)  # (handfuls of rows go row by row)
    assert bool(((out[:rows].double() - y).abs() <= yb).all()) and bool(((so.flip(0).double() - ends).abs() <= endb).all())
    assert (out[rows:] == 7.0).all()
