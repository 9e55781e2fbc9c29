"""Prefill of handfuls of rows, which go row by row: a bf16 state is FP32 from the first row to the last and rounded once, and more chains take more rows that way."""
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


# One to eight rows over few chains; up to 16, 24 and 32 over two, three and more waves of them; one more than goes that way.
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens,heads,qk_heads", [([5], 2, 1), ([1, 8, 0, 3], 4, 4), ([1], 1, 1), ([16] * 20 + [9], 8, 2), ([24, 3] * 10, 16, 16), ([20] * 75, 8, 4), ([32, 1, 17] * 25, 8, 8),
                                                 ([9, 2], 2, 2), ([33, 32] * 38, 8, 8)])
def test_against_64_bits(lin, lens, heads, qk_heads, dtype):
    q, k, v, g, s = lo.inputs(lens, heads, qk_heads, 31, "cuda", "token", 0.2)
    state, rows, batch = s.to(dtype), sum(lens), len(lens)
    off = torch.arange(batch, dtype=torch.int64, device="cuda").flip(0) * (heads * PER)
    out, end = torch.full((rows + 3, heads, 128), 7.0, dtype=torch.bfloat16, device="cuda"), torch.full_like(state, 9.0)
    lin.prefill_varlen(heads, rows, lo.cu_of(lens, "cuda"), max(lens), q, k, v, g, state, off, qk_heads=qk_heads, state_out=end, scale=0.7, out=out)
    torch.cuda.synchronize()
    assert importlib.import_module("glm53f-afd_b200.core").device_status() == 0
    bf16 = dtype == torch.bfloat16
    by_rows = max(lens) <= 8 * min(4, -(-heads * batch // torch.cuda.get_device_properties(0).multi_processor_count))
    if by_rows:
        y, ends, yb, endb = lo.recurrence(lens, q, k, v, g, state.flip(0), 0.7, False)
        if bf16:
            endb = endb + lo.UBF * (ends.abs() + endb)  # rounded once, at the end
    else:
        y, ends, yb, endb = lo.chunked(lens, q, k, v, g, state.flip(0), 0.7, bf16)
    assert bool(((out[:rows].double() - y).abs() <= yb).all()) and bool(((end.flip(0).double() - ends).abs() <= endb).all())
    assert (out[rows:] == 7.0).all()
