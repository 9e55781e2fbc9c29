"""Chunked prefill of the linear attention: a sequence's last, short chunk reaches over rows that are another sequence's or nobody's.  Whatever lies there, the
results are the bits that they are with zeros there."""
import importlib

import pytest

import linear_oracle as lo

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
PER = 128 * 128


@pytest.fixture(scope="module")
def lin():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return importlib.import_module("glm53f-afd_b200.linear")


def status():
    torch.cuda.synchronize()
    return importlib.import_module("glm53f-afd_b200.core").device_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("whole", [0, 1, 2, 5])
@pytest.mark.parametrize("rest", [1, 2, 7, 8, 9, 31, 33, 48, 62, 63])
def test_what_lies_behind_a_sequence_stays_there(lin, rest, whole, dtype):
    heads, n, behind = 40, 64 * whole + rest, 70
    rows = n + behind  # a sequence, and rows of none
    q, k, v, g, s = lo.inputs([n, behind], heads, heads, rest + whole, "cuda", "token", 0.05)
    state, off, cu = s[:1].to(dtype), torch.zeros(1, dtype=torch.int64, device="cuda"), lo.cu_of([n], "cuda")
    got = []
    for fill in (0.0, float("nan"), float("inf"), -float("inf")):
        for t in (q, k, v, g):
            t[n:] = fill
        out, end = torch.full((rows, heads, 128), 7.0, dtype=torch.bfloat16, device="cuda"), torch.empty_like(state)
        lin.prefill_varlen(heads, rows, cu, max(n, 64), q, k, v, g, state, off, state_out=end, out=out)
        assert status() == 0
        assert (out[n:] == 7.0).all()
        got.append((out[:n], end))
    assert all(torch.equal(a, b) for one in got[1:] for a, b in zip(one, got[0]))
    assert torch.isfinite(got[0][0]).all() and torch.isfinite(got[0][1]).all()


def test_a_whole_batch_beside_nan(lin):
    """Every other sequence is NaN; many blocks a SM, so that they start at different times."""
    lens, heads = [1 + 37 * i % 200 for i in range(60)], 8
    q, k, v, g, s = lo.inputs(lens, heads, heads, 3, "cuda", "token", 0.05)
    rows, cu = sum(lens), lo.cu_of(lens, "cuda")
    off = torch.arange(len(lens), dtype=torch.int64, device="cuda") * (heads * PER)
    got = []
    for bad in (0.0, float("nan")):
        q2, k2, v2, s2 = (t.clone() for t in (q, k, v, s))
        first, mine = 0, []
        for i, n in enumerate(lens):
            if i % 2:
                for t in (q2, k2, v2):
                    t[first:first + n] = bad
            else:
                mine += range(first, first + n)
            first += n
        out = torch.empty(rows, heads, 128, dtype=torch.bfloat16, device="cuda")
        lin.prefill_varlen(heads, rows, cu, max(lens), q2, k2, v2, g, s2, off, out=out)
        assert status() == 0
        got.append((out[mine], s2[::2]))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert torch.isfinite(got[0][0]).all()
