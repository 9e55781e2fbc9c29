"""`Int4Mat.quantise` of weights that lie in memory otherwise than row by row."""
import importlib

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def proj():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return importlib.import_module("glm53f-afd_b200.proj")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("zeros", [False, True])
def test_strides(proj, dtype, zeros):
    n, k = 75, 256
    w = torch.randn(n, k, device="cuda").to(dtype)
    want = proj.Int4Mat.quantise(w, group=64, zeros=zeros)
    x = torch.randn(3, k, device="cuda").bfloat16()
    a = torch.empty(3, n, device="cuda")
    proj.int4(x, k, want, 3, a, n, out_f32=True)
    apart = torch.zeros(n, 2 * k, device="cuda", dtype=dtype)
    apart[:, ::2] = w
    rows = torch.zeros(n, k + 8, device="cuda", dtype=dtype)
    rows[:, :k] = w
    for other in (w.t().contiguous().t(), apart[:, ::2], rows[:, :k]):
        assert not other.is_contiguous() and torch.equal(other, w)
        m = proj.Int4Mat.quantise(other, group=64, zeros=zeros)
        b = torch.empty(3, n, device="cuda")
        proj.int4(x, k, m, 3, b, n, out_f32=True)
        assert torch.equal(a, b)
