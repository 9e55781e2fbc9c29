"""Projections with bias, activation and residual in the epilogue, against 64 bits.

Bound: the product's f32 sum of k terms loses at most (k + 2) half steps of the sum of their magnitudes (the tensor core may add them in any
grouping); an activation's slope is at most 1.13 (gelu's), its own arithmetic loses 8 half steps of f32 of |y| or of 1 (exp, erfc and
the division a few each); the last rounding half a step of the result's type."""
import importlib
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U32, UBF = 2.0 ** -24, 2.0 ** -8


@pytest.fixture(scope="module")
def proj():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return importlib.import_module("glm53f-afd_b200.proj")


def act64(name, y):
    if name == "relu":
        return y.clamp(min=0)
    if name == "silu":
        return y * torch.sigmoid(y)
    if name == "gelu":
        return 0.5 * y * torch.erfc(-y / math.sqrt(2))
    if name == "gelu_tanh":
        return y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    return torch.sigmoid(y) if name == "sigmoid" else y


def status():
    torch.cuda.synchronize()
    return importlib.import_module("glm53f-afd_b200.core").device_status()


def make(groups, rows, n, k, bias, residual, f32, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(groups, rows, k, generator=gen).bfloat16().cuda()
    w = (k ** -0.5 * torch.randn(groups, n, k, generator=gen)).bfloat16().cuda()
    b = None if bias is None else torch.randn(groups, n, generator=gen).to(bias).cuda()
    kind = torch.float32 if f32 else torch.bfloat16
    r = torch.randn(groups, rows, n, generator=gen).to(kind).cuda() if residual else None
    return x, w, b, r, kind


def expect(x, w, b, r, act, f32):
    y = x.double() @ w.double().transpose(1, 2)
    size = x.double().abs() @ w.double().abs().transpose(1, 2)
    if b is not None:
        y = y + b.double()[:, None]
        size = size + b.double().abs()[:, None]
    z = act64(act, y)
    bound = 1.13 * (x.shape[2] + 2) * U32 * size + (0 if act == "none" else 8 * U32 * (1 + y.abs()))
    if r is not None:
        z = z + r.double()
    bound = bound + 2 * U32 * z.abs()
    return z, bound + (U32 if f32 else UBF) * (z.abs() + bound) + 1e-38


def check(got, want, bound):
    far = (got.double() - want).abs() - bound
    assert bool((far <= 0).all()), float(far.max())


SHAPES = [
    # groups, rows, n, k, f32 out: one block a tile, clusters that split k, odd rows, SM pairs, pairs whose k runs in segments
    (1, 1, 8, 64, False), (1, 16, 4096, 1024, True), (1, 16, 256, 4096, False), (1, 37, 264, 2048, False), (2, 33, 512, 128, True),
    (1, 64, 256, 4096, True), (1, 96, 19008, 128, False), (1, 90, 200, 64, True), (1, 97, 1000, 64, False), (2, 130, 8192, 128, False), (1, 333, 4096, 512, True),
    (1, 333, 8192, 128, False), (1, 200, 256, 4096, False), (1, 200, 256, 4096, True), (1, 700, 4096, 1024, False), (1, 513, 256, 2048, False),
]


@pytest.mark.parametrize("groups,rows,n,k,f32", SHAPES)
@pytest.mark.parametrize("act,bias,residual", [("none", torch.bfloat16, True), ("silu", torch.float32, True), ("gelu", None, False), ("sigmoid", torch.bfloat16, True)])
def test_against_64_bits(proj, groups, rows, n, k, f32, act, bias, residual):
    x, w, b, r, kind = make(groups, rows, n, k, bias, residual, f32, 5)
    out = torch.full((groups * rows * n + 8,), 7.0, dtype=kind, device="cuda")
    proj.fused(x, k, rows * k, proj.Bf16Mat.dense(w), rows, out, n, rows * n, f32, bias=b, activation=act, residual=r)
    assert status() == 0
    want, bound = expect(x, w, b, r, act, f32)
    check(out[:-8].view(groups, rows, n), want, bound)
    assert (out[-8:] == 7.0).all()


@pytest.mark.parametrize("act", ["relu", "gelu_tanh", "gelu", "silu", "sigmoid"])
def test_activations_over_their_range(proj, act):
    """y from -40 to 40 by the bias alone (x = 0), f32 results."""
    n = 4096
    x, w = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, n, 64, dtype=torch.bfloat16, device="cuda")
    y = torch.linspace(-40, 40, n, device="cuda")
    out = torch.empty(n, device="cuda")
    proj.fused(x, 64, 64, proj.Bf16Mat.dense(w), 1, out, n, n, True, bias=y.view(1, n), activation=act)
    want = act64(act, y.double())
    # The exponential's argument is rounded: a relative error of the result of |argument| half steps (|y| <= 40; the cubic's up to 1.6 (40 + 0.045 40^3) < 4,700 where
    # the result is below the smallest f32 anyway, below 90 where it is not; erfc's argument squared 2 * 88).
    # And e^x is infinite in f32 from x = ln(2^128) = 88.72 on: y / (1 + e^x) is 0 there where the definition has at most |y| e^-88.72 = |y| 2^-128.
    check(out, want, (200 + 4 * 90) * U32 * want.abs() + 2.0 ** -148 + 2.0 ** -128 * y.double().abs())


@pytest.mark.parametrize("rows,n,k,f32", [(16, 256, 4096, False), (40, 512, 256, True), (300, 512, 256, False), (300, 512, 256, True)])
def test_in_place_residual_and_strided_rows(proj, rows, n, k, f32):
    """out += x w^T + bias on rows of a wider tensor; the same bits as into another tensor, the rest of the rows untouched."""
    x, w, b, r, kind = make(1, rows, n, k, torch.bfloat16, True, f32, 9)
    mat = proj.Bf16Mat.dense(w)
    apart = torch.empty(rows, n, dtype=kind, device="cuda")
    proj.fused(x, k, 0, mat, rows, apart, n, 0, f32, bias=b, activation="relu", residual=r)
    for pad in (24, 13):
        wide = torch.full((rows, n + pad), 3.0, dtype=kind, device="cuda")
        wide[:, 8:8 + n] = r[0]
        proj.fused(x, k, 0, mat, rows, wide, n + pad, 0, f32, out_offset=8, bias=b, activation="relu", residual=wide, residual_offset=8)
        assert status() == 0
        assert torch.equal(wide[:, 8:8 + n], apart)
        assert (wide[:, :8] == 3.0).all() and (wide[:, 8 + n:] == 3.0).all()


def test_residual_of_other_strides(proj):
    """Residual rows of another stride, one broadcast row included (ldr is at least a row, so a broadcast is over groups)."""
    groups, rows, n, k = 2, 150, 512, 128
    x, w, b, _, kind = make(groups, rows, n, k, torch.float32, False, False, 11)
    r = torch.randn(rows, n + 16, device="cuda").bfloat16()
    out = torch.empty(groups, rows, n, dtype=kind, device="cuda")
    proj.fused(x, k, rows * k, proj.Bf16Mat.dense(w), rows, out, n, rows * n, bias=b, residual=r, ldr=n + 16, r_gstride=0)
    want, bound = expect(x, w, b, r[:, :n].expand(groups, rows, n), "none", False)
    check(out, want, bound)


def test_without_an_epilogue_the_plain_projections_bits(proj):
    for groups, rows, n, k, f32 in ((1, 16, 256, 4096, True), (1, 64, 4096, 256, False), (1, 333, 4096, 512, False), (1, 200, 256, 4096, False)):
        x, w, _, _, kind = make(groups, rows, n, k, None, False, f32, 13)
        a, b = (torch.empty(groups * rows * n, dtype=kind, device="cuda") for _ in range(2))
        proj.bf16(x, k, 0, proj.Bf16Mat.dense(w), rows, a, n, 0, f32)
        proj.fused(x, k, 0, proj.Bf16Mat.dense(w), rows, b, n, 0, f32)
        assert torch.equal(a, b)


def test_a_rows_result_does_not_depend_on_the_others(proj):
    n, k = 512, 4096
    x, w, b, r, kind = make(1, 400, n, k, torch.float32, True, True, 15)
    mat = proj.Bf16Mat.dense(w)
    whole = torch.empty(400, n, device="cuda")
    proj.fused(x, k, 0, mat, 400, whole, n, 0, True, bias=b, activation="gelu", residual=r)
    for rows in (1, 16, 17, 90, 128, 129):
        some = torch.empty(rows, n, device="cuda")
        proj.fused(x, k, 0, mat, rows, some, n, 0, True, bias=b, activation="gelu", residual=r)
        assert torch.equal(some, whole[:rows]), rows


@pytest.mark.parametrize("act,at_minus_inf,at_inf", [("relu", 0.0, math.inf), ("gelu", 0.0, math.inf), ("silu", None, math.inf), ("gelu_tanh", None, math.inf), ("sigmoid", 0.0, 1.0)])
def test_infinities_and_nan(proj, act, at_minus_inf, at_inf):
    """By the bias, at few rows and on SM pairs.  (Where the formula has minus infinity times zero, either that or the limit, 0.)"""
    for rows in (3, 130):
        x, w = torch.zeros(rows, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(64, 64, dtype=torch.bfloat16, device="cuda")
        y = torch.zeros(64, device="cuda")
        y[0], y[9], y[17], y[33], y[34] = -math.inf, math.inf, math.nan, 3e38, -3e38
        out = torch.empty(rows, 64, device="cuda")
        proj.fused(x, 64, 0, proj.Bf16Mat.dense(w), rows, out, 64, 0, True, bias=y, activation=act)
        low, high, nan, big, small = (out[:, i] for i in (0, 9, 17, 33, 34))
        assert nan.isnan().all() and (high == at_inf).all() and (big == (1.0 if act == "sigmoid" else y[33])).all() and (small == 0).all()
        assert ((low == at_minus_inf) if at_minus_inf is not None else (low.isnan() | (low == 0))).all()
        assert torch.isfinite(out[:, 40:]).all()
