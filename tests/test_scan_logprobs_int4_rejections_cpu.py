"""What the C entry points of the gated recurrence, the log probabilities and the 4-bit projections refuse on the host: status 1 before any launch, 0 where there is nothing to do.
No GPU is needed: the addresses are stand-ins that no path here reads."""
import pytest

A = 4096  # on 16 bytes


@pytest.fixture(scope="module")
def lib(pkg):
    pkg.build()
    return pkg.ffi.load()


STEP = dict(channels=64, batch=2, cu=A, keep=None, g=A, gs=64, x=A, xs=64, flags=0, si=A, so=A, off=A, out=A, os=64)
PREFILL = dict(channels=64, batch=2, cu=A, rows=9, most=5, g=A, gs=64, x=A, xs=64, flags=0, si=A, so=A, off=A, out=A, os=64, saves=None, ws=None, wn=0)
BACKWARD = dict(channels=64, batch=2, cu=A, rows=9, most=5, g=A, gs=64, x=A, xs=64, flags=0, saves=A, dy=A, dys=64, ds=None, di=None, off=A, dg=A, dgs=64, dx=A, dxs=64, ws=None, wn=0)
LOGPROBS = dict(rows=3, vocab=50, logits=A, kind=1, ld=50, tokens=A, t=None, lp=A, h=None, lse=None, top=0, ids=None, values=None)
GRADS = dict(rows=3, vocab=50, logits=A, kind=1, ld=50, tokens=A, t=None, lse=A, h=None, dlp=A, dh=None, d=A, dld=50)
INT4 = dict(x=A, ldx=128, w=A, n=10, k=128, group=64, zeros=0, rows=3, out=A, f32=0, ldo=10)
PACK = dict(codes=A, scales=A, zeros=None, n=10, k=128, group=64, packed=A)

COMMON = [dict(channels=0), dict(channels=-1), dict(channels=2 ** 30 + 1, gs=2 ** 31, xs=2 ** 31, os=2 ** 31, dys=2 ** 31, dgs=2 ** 31, dxs=2 ** 31), dict(batch=-1), dict(cu=None), dict(flags=16), dict(flags=-1), dict(g=None), dict(x=None),
          dict(gs=63), dict(xs=63), dict(g=A + 2), dict(x=A + 1), dict(g=A + 1, flags=4), dict(x=A + 1, flags=8), dict(off=None)]
RANGES = [dict(rows=-1), dict(most=-1), dict(most=10), dict(rows=2 ** 30 + 1), dict(wn=-1), dict(ws=A + 8, wn=1 << 20)]
CASES = {
    "scan_decode_batch": (STEP, COMMON + [dict(si=None), dict(si=A + 2), dict(so=A + 2), dict(so=None, out=None), dict(os=63), dict(out=A + 2)]),
    "scan_prefill_varlen": (PREFILL, COMMON + RANGES + [dict(si=None), dict(so=None), dict(so=A + 2), dict(os=63), dict(saves=A + 4)]),
    "scan_backward_varlen": (BACKWARD, COMMON + RANGES + [dict(saves=None), dict(dy=None), dict(dg=None), dict(dx=None), dict(dys=63), dict(dgs=63), dict(dxs=63), dict(ds=A + 2), dict(di=A + 1), dict(saves=A + 2)]),
    "logprobs": (LOGPROBS, [dict(rows=-1), dict(vocab=0), dict(vocab=2000001, ld=2000001), dict(logits=None), dict(kind=9), dict(kind=-1), dict(ld=49), dict(logits=A + 1), dict(tokens=None), dict(lp=None), dict(lp=None, tokens=None),
                            dict(tokens=A + 2), dict(t=A + 1), dict(h=A + 2), dict(lse=A + 3), dict(top=-1), dict(top=33, ids=A, values=A), dict(top=5), dict(top=5, ids=A), dict(top=5, values=A), dict(ids=A, values=A)]),
    "logprobs_backward": (GRADS, [dict(rows=-1), dict(vocab=0), dict(vocab=2000001, ld=2000001, dld=2000001), dict(logits=None), dict(kind=9), dict(ld=49), dict(dld=49), dict(d=None), dict(d=A + 1), dict(tokens=None), dict(lse=None), dict(dlp=None),
                                  dict(dh=A), dict(dh=A, h=A + 2), dict(t=A + 2), dict(lse=A + 2)]),
    "proj_int4": (INT4, [dict(rows=-1), dict(n=0), dict(n=2 ** 30 + 1, ldo=2 ** 31), dict(k=0), dict(k=96, group=32), dict(k=192, group=128, ldx=192), dict(k=65600, ldx=65600), dict(group=16), dict(group=0), dict(ldx=120), dict(ldx=132), dict(ldo=9), dict(x=None),
                         dict(x=A + 8), dict(w=None), dict(w=A + 8), dict(out=None), dict(out=A + 1), dict(out=A + 2, f32=1)]),
    "int4_pack": (PACK, [dict(n=0), dict(k=32, group=32), dict(group=48), dict(codes=None), dict(scales=None), dict(scales=A + 1), dict(packed=None), dict(packed=A + 8)]),
}


@pytest.mark.parametrize("name", CASES)
def test_refused(lib, name):
    base, wrong = CASES[name]
    for change in wrong:
        args = {**base, **{k: v for k, v in change.items() if k in base}}
        assert any(k in base for k in change)
        assert getattr(lib, "glm53f_kda_" + name)(*args.values(), None) == 1, (name, change)


def test_nothing_to_do(lib):
    for name, key in (("scan_decode_batch", "batch"), ("scan_prefill_varlen", "batch"), ("scan_backward_varlen", "batch"), ("logprobs", "rows"), ("logprobs_backward", "rows"), ("proj_int4", "rows")):
        assert getattr(lib, "glm53f_kda_" + name)(*{**CASES[name][0], key: 0}.values(), None) == 0, name


def test_sizes(lib):
    for args in ((0, 1, 9), (64, 0, 9), (64, 1, -1), (2 ** 30 + 1, 1, 9), (64, 1, 2 ** 30 + 1)):
        assert lib.glm53f_kda_scan_workspace_bytes(*args) == 0
    small = lib.glm53f_kda_scan_workspace_bytes(64, 1, 64)
    assert 0 < small < lib.glm53f_kda_scan_workspace_bytes(64, 1, 640) < lib.glm53f_kda_scan_workspace_bytes(65, 1, 640)
    assert lib.glm53f_kda_scan_saves_rows(3, 640) == 13 and lib.glm53f_kda_scan_saves_rows(0, 640) == lib.glm53f_kda_scan_saves_rows(1, -1) == 0
    for args in ((0, 64, 64, 0), (16, 32, 32, 0), (16, 128, 100, 0), (16, 192, 128, 0), (16, 65600, 64, 0)):
        assert lib.glm53f_kda_int4_bytes(*args) == 0
    # 17 weight rows are two tiles of 16: half a byte a weight, two a scale and one a zero point, each part rounded up to 256 bytes.
    codes, scales, zeros = 32 * 128 // 2, 32 * 2 * 2, 32 * 2
    up = lambda n: (n + 255) // 256 * 256
    assert lib.glm53f_kda_int4_bytes(17, 128, 64, 0) == up(codes) + up(scales)
    assert lib.glm53f_kda_int4_bytes(17, 128, 64, 1) == up(codes) + up(scales) + up(zeros)
