"""Chunked prefill of the linear attention: the state and the factored rows of q are f32 operands of which the tensor core takes 11 bits and cuts the rest off.  The cuts
all go one way; what they take on the mean is made up for, so that outputs are no smaller on the mean than they should be."""
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


def run(lin, lens, q, k, v, g, s, scale):
    heads, rows = v.shape[1], sum(lens)
    out, end = torch.empty(rows, heads, 128, dtype=torch.bfloat16, device="cuda"), torch.empty_like(s)
    off = torch.arange(len(lens), dtype=torch.int64, device="cuda") * (heads * PER)
    lin.prefill_varlen(heads, rows, lo.cu_of(lens, "cuda"), max(max(lens), 64), q, k, v, g, s, off, state_out=end, scale=scale, out=out)
    torch.cuda.synchronize()
    assert importlib.import_module("glm53f-afd_b200.core").device_status() == 0
    return out.double()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens,size,carried", [([64] * 40, 0.01, 1.0), ([640], 0.01, 1.0), ([2000], 0.001, 0.0), ([900, 1100], 0.02, 0.5)])
def test_outputs_are_not_smaller_on_the_mean(lin, lens, size, carried, dtype):
    """The slope of the outputs against the definition's.  The mean cut of either operand is within 5 % of 3.52e-4 of it for values spread over a few powers of two (of the mantissa's
    density only the deviation from 1 / m counts): 3.6e-5 for both.  The roundings to bf16 (1.7e-3 each, independent) average out over 256,000 or more values, weighed by their
    squares: 1.7e-3 sqrt(3 / 256,000) = 5.8e-6, five times that 2.9e-5.  Cut off and left so it is -1.6e-4 to -6.6e-4."""
    heads = 4
    q, k, v, g, s = lo.inputs(lens, heads, heads, 21, "cuda", "token", size)
    s = (carried * s).to(dtype)
    got, want = run(lin, lens, q, k, v, g, s, 128 ** -0.5), lo.chunked(lens, q, k, v, g, s, 128 ** -0.5, dtype == torch.bfloat16)[0]
    assert abs(float((got * want).sum() / (want * want).sum()) - 1) <= 6.5e-5


@pytest.mark.parametrize("scale", [1.0, -0.25, 1.75])
def test_what_is_not_cut_is_left_alone(lin, scale):
    """A bf16 state, decays of 0 and a factor of three bits: both operands fit 11 bits, so S q is exact but for the sum of 128 products (four half steps of f32 a term) and
    its rounding to bf16."""
    lens, heads = [64, 9, 33], 3
    q, k, v, g, s = lo.inputs(lens, heads, heads, 22, "cuda", "head", 0.0)
    s, v = s.bfloat16(), torch.zeros_like(v)
    got = run(lin, lens, q, k, v, torch.zeros_like(g), s, scale)
    first = 0
    for b, n in enumerate(lens):
        dots = s[b].double()[None] * q[first:first + n].double()[:, :, None, :]
        want, size = scale * dots.sum(-1), abs(scale) * dots.abs().sum(-1)
        bound = 4 * 128 * lo.U32 * size
        assert bool(((got[first:first + n] - want).abs() <= bound + lo.UBF * (want.abs() + bound)).all())
        # ... and so it is the nearest bf16 number nearly everywhere
        assert float((got[first:first + n] == want.bfloat16().double()).double().mean()) > 0.98
        first += n
