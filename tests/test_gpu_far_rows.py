"""Rows that lie further apart than 32 bits of elements reach: the bits of the same rows side by side."""
import importlib

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


@pytest.fixture(scope="module")
def mods():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return {n: importlib.import_module("glm53f-afd_b200." + n) for n in ("gated", "spec", "proj")}


def far(t, stride):
    """The same rows, `stride` elements apart."""
    rows, n = t.shape
    room = torch.empty((rows - 1) * stride + n, dtype=t.dtype, device="cuda").as_strided((rows, n), (stride, 1))
    return room.copy_(t)


def test_log_probabilities(mods):
    spec = mods["spec"]
    near = torch.randn(3, 1000, device="cuda").bfloat16()
    tokens, lse, h, lp = torch.tensor([5, 999, 0], dtype=I32, device="cuda"), *(torch.empty(3, device="cuda") for _ in range(3))
    results = []
    for logits in (near, far(near, 2 ** 31 + 8)):
        top = torch.empty(3, 4, dtype=I32, device="cuda"), torch.empty(3, 4, device="cuda")
        spec.logprobs(logits, tokens, lp, entropy=h, lse=lse, top=top)
        d = torch.empty_like(near) if logits is near else logits
        spec.logprobs_backward(logits, tokens, lse, lp, d, entropy=h, dentropy=h)
        results.append([t.clone() for t in (lp, h, lse, *top, d)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("rows", [3, 9])
def test_4_bit_projections(mods, rows):
    proj = mods["proj"]
    w = proj.Int4Mat.quantise(torch.randn(40, 128, device="cuda"), group=64)
    x, stride = torch.randn(rows, 128, device="cuda").bfloat16(), 2 ** 30 if rows == 3 else 2 ** 28 + 8
    near = torch.empty(rows, 40, device="cuda")
    proj.int4(x, 128, w, rows, near, 40, out_f32=True)
    apart = torch.empty((rows - 1) * stride + 128, dtype=BF, device="cuda")
    apart.as_strided((rows, 128), (stride, 1)).copy_(x)
    out = torch.empty((rows - 1) * stride + 40, device="cuda")
    proj.int4(apart, stride, w, rows, out, stride, out_f32=True)
    assert torch.equal(out.as_strided((rows, 40), (stride, 1)), near)


@pytest.mark.parametrize("channels", [64, 63])
def test_gated_recurrence(mods, channels):
    gated = mods["gated"]
    rows, stride = 70, 2 ** 25 + 8
    g, x, dy = -torch.rand(rows, channels, device="cuda"), torch.randn(rows, channels, device="cuda").bfloat16(), torch.randn(rows, channels, device="cuda").bfloat16()
    cu, off = torch.tensor([0, 68, 70], dtype=I32, device="cuda"), torch.tensor([2 ** 31 + 6, 0], device="cuda")
    states = torch.empty(2 ** 31 + 6 + channels, device="cuda")
    results = []
    for a, b, c in ((g, x, dy), (far(g, stride), far(x, stride), far(dy, stride))):
        like = (lambda t: torch.empty_like(t)) if a is g else (lambda t: far(t, stride))
        states[:channels], states[-channels:] = 0.5, -0.25
        out, dg, dx, again = like(x), like(g), like(x), like(x)
        saves = torch.empty(gated.saves_rows(2, rows), channels, device="cuda")
        gated.prefill_varlen(channels, rows, cu, 68, a, b, states, off, out=out, saves=saves)
        ends = states[:channels].clone(), states[-channels:].clone()
        gated.backward_varlen(channels, rows, cu, 68, a, b, saves, off, c, dg, dx, dstate=states, dstate_in=states)
        starts = states[:channels].clone(), states[-channels:].clone()
        gated.decode_batch(channels, rows, cu, a, b, states, off, state_out="in_place", out=again)
        results.append([t.clone() for t in (out, dg, dx, again, *ends, *starts, states[:channels], states[-channels:])])
    assert all(torch.equal(p, q) for p, q in zip(*results))
