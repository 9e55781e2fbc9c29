"""Projections with 4-bit weights on the GPU against 64 bits.

Bounds.  x (q - z) is exact.  The tensor core adds 16 such products and a sum at a time and keeps 24 bits or more of the largest, so a group's sum is within 16 / 16 + 1 = 2 units of 2^-23 of
its terms' magnitudes for every 16 k, the scaled sums add another 2^-24 for each of k / 32 groups at most and as many where parts of k meet: k / 4 units of 2^-24 of sum |x w| and 64 more for short k."""
import importlib

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def proj():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return importlib.import_module("glm53f-afd_b200.proj")


def weight(n, k, group, zeros, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 16, (n, k), generator=gen, device="cuda", dtype=torch.uint8)
    scales = (torch.randn(n, k // group, generator=gen, device="cuda") * k ** -0.5).bfloat16()
    z = torch.randint(0, 16, (n, k // group), generator=gen, device="cuda", dtype=torch.uint8) if zeros else None
    zero = 8.0 if z is None else z.double().repeat_interleave(group, 1)
    w = (q.double() - zero) * scales.double().repeat_interleave(group, 1)
    return q[:, ::2] | (q[:, 1::2] << 4), scales, z, w


def compare(out, x, w):
    want, size = x.double() @ w.T, x.double().abs() @ w.abs().T
    k = x.shape[1]
    bound = (k / 4 + 64) * 2.0 ** -24 * size
    step = torch.finfo(out.dtype).eps / 2 * (want.abs() + bound)
    assert not out.isnan().any()
    over = (out.double() - want).abs() - bound - step
    assert (over <= 0).all(), (float(over.max()), int((over > 0).sum()))
    if out.dtype == F32:  # the projections' own bound on f32 results
        assert (out.double() - want).norm() <= 1e-5 * want.norm()


ROWS = [1, 2, 7, 8, 9, 16, 17, 33, 64, 100, 129, 300]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("group,zeros", [(32, False), (32, True), (64, False), (64, True), (128, False), (128, True)])
def test_row_counts(proj, rows, group, zeros):
    n, k = 328, 640
    codes, scales, z, w = weight(n, k, group, zeros)
    m = proj.Int4Mat.pack(codes, scales, z, group=group)
    x = torch.randn(rows, k, device="cuda").bfloat16()
    for f32 in (False, True):
        out = torch.full((rows, n), 7.0, dtype=F32 if f32 else BF, device="cuda")
        proj.int4(x, k, m, rows, out, n, out_f32=f32)
        compare(out, x, w)


@pytest.mark.parametrize("n,k,group", [(1, 64, 64), (1, 64, 32), (7, 128, 128), (16, 192, 64), (17, 96 * 2, 32), (129, 128, 128), (64, 4096, 128), (300, 8192, 32), (24640, 4096, 128), (40, 16384, 64),
                                       (5, 65536, 128), (3001, 256, 32), (20000, 64, 64)])
@pytest.mark.parametrize("rows", [1, 5, 40, 200])
def test_shapes(proj, n, k, group, rows):
    codes, scales, z, w = weight(n, k, group, n % 2 == 1)
    m = proj.Int4Mat.pack(codes, scales, z, group=group)
    x = torch.randn(rows, k, device="cuda").bfloat16()
    out = torch.empty(rows, n, dtype=F32, device="cuda")
    proj.int4(x, k, m, rows, out, n, out_f32=True)
    compare(out, x, w)
    again = torch.empty_like(out)
    proj.int4(x, k, m, rows, again, n, out_f32=True)
    assert torch.equal(out, again)


@pytest.mark.parametrize("rows", [1, 6, 50, 140])
def test_strides_offsets_and_what_lies_between(proj, rows):
    n, k, ldx, ldo = 75, 256, 264, 83
    codes, scales, z, w = weight(n, k, 64, True)
    m = proj.Int4Mat.pack(codes, scales, z, group=64)
    room = torch.full((8 + rows * ldx,), float("nan"), device="cuda").bfloat16()
    x = room[8:].view(rows, ldx)
    x[:, :k] = torch.randn(rows, k, device="cuda")
    for dtype in (BF, F32):
        out = torch.full((5 + rows * ldo,), 7.0, dtype=dtype, device="cuda")
        proj.int4(room, ldx, m, rows, out, ldo, out_f32=dtype == F32, x_offset=8, out_offset=5)
        got = out[5:].view(rows, ldo)
        compare(got[:, :n], x[:, :k], w)
        assert (out[:5] == 7).all() and (got[:, n:] == 7).all()


def test_quantised_weights(proj):
    """The nearest codes: no further than half a scale and its rounding from the weight."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    w = torch.randn(100, 512, generator=gen, device="cuda")
    w[3, :128], w[4, 128:256] = 0.0, w[4, 128:256].abs()
    eye = torch.eye(512, device="cuda").bfloat16()
    for group in (32, 64, 128):
        for zeros in (False, True):
            m = proj.Int4Mat.quantise(w, group=group, zeros=zeros)
            back = torch.empty(512, 100, device="cuda")
            proj.int4(eye, 512, m, 512, back, 100, out_f32=True)
            back = back.T.reshape(100, -1, group)
            g = w.view(100, -1, group)
            span = (g.amax(-1).clamp(min=0) - g.amin(-1).clamp(max=0)) / 15 if zeros else g.abs().amax(-1) / 7
            # half a step, the scale's rounding at up to 15 steps, and with a zero point its own half step
            assert ((back - g).abs() <= span[..., None] * (0.5 + 15 * 2.0 ** -8 + (0.5 if zeros else 0)) + 1e-6).all()
            assert (back[3].flatten()[:128] == 0).all()


def test_infinities_stay_in_their_rows(proj):
    n, k = 90, 512
    codes, scales, z, w = weight(n, k, 128, True)
    m = proj.Int4Mat.pack(codes, scales, z)
    for rows in (4, 70):
        x = torch.randn(rows, k, device="cuda").bfloat16()
        x[1, 5], x[2, 100] = float("inf"), float("nan")
        out = torch.empty(rows, n, device="cuda")
        proj.int4(x, k, m, rows, out, n, out_f32=True)
        keep = [i for i in range(rows) if i not in (1, 2)]
        compare(out[keep], x[keep], w)
        assert not out[1].isfinite().any() and out[2].isnan().all()


def test_graphs_and_streams(proj):
    n, k = 1000, 1024
    codes, scales, z, w = weight(n, k, 128, False)
    m = proj.Int4Mat.pack(codes, scales, z)
    for rows in (3, 90):
        x = torch.randn(rows, k, device="cuda").bfloat16()
        out, want = torch.zeros(rows, n, device="cuda"), torch.zeros(rows, n, device="cuda")
        proj.int4(x, k, m, rows, want, n, out_f32=True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            proj.int4(x, k, m, rows, out, n, out_f32=True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        side = torch.cuda.Stream()
        out.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            proj.int4(x, k, m, rows, out, n, out_f32=True)
        side.synchronize()
        assert torch.equal(out, want)
    assert importlib.import_module("glm53f-afd_b200.core").device_status() == 0
