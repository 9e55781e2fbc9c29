"""Projections with 4-bit weights: up to eight rows have the bits of single ones, whatever k is, whether the rows fit in shared memory or come with the weights."""
import importlib

import pytest

torch = pytest.importorskip("torch")
from test_gpu_proj_int4 import BF, F32, compare, weight

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def proj():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return importlib.import_module("glm53f-afd_b200.proj")


# Eight rows fit up to k of 9,592, five up to 15,352, three up to 25,592, two up to 38,392 and one always.
@pytest.mark.parametrize("n,k,group,zeros", [(40, 64, 64, False), (300, 4096, 128, True), (40, 9536, 64, True), (40, 9600, 128, False), (33, 9600, 32, True), (3000, 12288, 128, False), (40, 15360, 64, False),
                                             (24, 16384, 128, True), (100, 28672, 32, False), (40, 38400, 128, False), (17, 65536, 64, True)])
def test_bits_of_single_rows(proj, n, k, group, zeros):
    codes, scales, z, w = weight(n, k, group, zeros)
    m = proj.Int4Mat.pack(codes, scales, z, group=group)
    gen = torch.Generator(device="cuda").manual_seed(3)
    ldx = k + 8
    room = torch.full((8, ldx), float("nan"), device="cuda").bfloat16()  # (what lies between the rows is not used)
    room[:, :k] = torch.randn(8, k, device="cuda", generator=gen)
    single = torch.empty(8, n, device="cuda")
    for r in range(8):
        proj.int4(room, ldx, m, 1, single[r], n, out_f32=True, x_offset=r * ldx)
    compare(single, room[:, :k], w)
    for rows in range(2, 9):
        for first in {0, 8 - rows}:
            for dtype in (F32, BF):
                out = torch.full((9, n), 7.0, dtype=dtype, device="cuda")
                proj.int4(room, ldx, m, rows, out, n, out_f32=dtype == F32, x_offset=first * ldx)
                assert torch.equal(out[:rows], single[first:first + rows].to(dtype)), (rows, first)
                assert (out[rows:] == 7).all()
    wide = room.clone()
    wide[3, 7], wide[5, k - 1] = float("inf"), float("nan")  # ... and rows do not mix
    out = torch.empty(8, n, device="cuda")
    proj.int4(wide, ldx, m, 8, out, n, out_f32=True)
    keep = [0, 1, 2, 4, 6, 7]
    assert torch.equal(out[keep], single[keep])
    assert importlib.import_module("glm53f-afd_b200.core").device_status() == 0
