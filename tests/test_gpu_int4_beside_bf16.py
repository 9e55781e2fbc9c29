"""Projections with 4-bit weights beside bf16 ones, whose blocks hold smaller parts of an SM's tensor memory: in turn in one stream, where a launch begins while the one before it drains, and
on two streams at once.  Every call's result has the bits that the call alone gives, wherever its tensor memory began."""
import importlib

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def proj():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return importlib.import_module("glm53f-afd_b200.proj")


@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, False), (128, True)])
@pytest.mark.parametrize("streams", [1, 2])
def test_bits(proj, group, zeros, streams):
    gen = torch.Generator(device="cuda").manual_seed(4)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    k = 1024
    calls = []  # (launch into a buffer, shape)
    for n, rows in ((3000, 9), (20000, 16), (1200, 17), (9000, 32), (504, 12), (4000, 64)):
        m, x = proj.Int4Mat.quantise(rn(n, k), group=group, zeros=zeros), rn(rows, k).bfloat16()
        calls.append((lambda out, m=m, x=x, n=n, rows=rows: proj.int4(x, k, m, rows, out, n, out_f32=True), (rows, n), 0))
        rows, n = min(rows, 16), n + 72
        w, x = proj.Bf16Mat.dense(rn(n, k).bfloat16()), rn(rows, k).bfloat16()
        calls.append((lambda out, w=w, x=x, n=n, rows=rows: proj.bf16(x, k, 0, w, rows, out, n, 0, out_f32=True), (rows, n), 1))
    want = []
    for call, shape, _ in calls:
        out = torch.empty(shape, device="cuda")
        torch.cuda.synchronize()
        call(out)
        torch.cuda.synchronize()
        want.append(out)
    rounds = 20
    got = [[torch.full(shape, 7.0, device="cuda") for _, shape, _ in calls] for _ in range(rounds)]
    torch.cuda.synchronize()
    on = [torch.cuda.Stream() for _ in range(streams)]
    for outs in got:
        for (call, _, kind), out in zip(calls, outs):
            with torch.cuda.stream(on[kind % streams]):
                call(out)
    torch.cuda.synchronize()
    for outs in got:
        for i, (a, b) in enumerate(zip(outs, want)):
            assert torch.equal(a, b), calls[i][1]
    assert importlib.import_module("glm53f-afd_b200.core").device_status() == 0
