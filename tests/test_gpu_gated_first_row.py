"""Sequences whose rows begin elsewhere than at row 0, divided over the GPU and walked: the rows before the first are no tile of anybody's."""
import importlib

import pytest

torch = pytest.importorskip("torch")
import gated_oracle as oracle
from test_gpu_gated import BF, F32, Case, cu_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mods():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return {n: importlib.import_module("glm53f-afd_b200." + n) for n in ("gated", "core")}


@pytest.mark.parametrize("first", [63, 64, 65, 200, 4096])
@pytest.mark.parametrize("channels,lens,behind", [(64, [3000], 0), (64, [3000], 70), (63, [2000, 0, 1], 5), (130, [0, 64, 1100], 200)], ids=lambda v: str(v).replace(" ", ""))
@pytest.mark.parametrize("gate,input,g,x", [("decay", "plain", F32, BF), ("sigmoid", "complement", BF, F32)])
def test_rows_before_the_first(mods, first, channels, lens, behind, gate, input, g, x):
    gated = mods["gated"]
    n, batch = sum(lens), len(lens)
    rows = first + n + behind
    c = Case(channels, [rows], gate, input, g, x)
    for t in (c.g, c.x, c.dout):  # what belongs to nobody is not used
        t[:first], t[first + n:] = float("nan"), float("nan")
    gen = torch.Generator(device="cuda").manual_seed(8)
    start, dstate = (torch.randn(batch, channels, device="cuda", generator=gen) for _ in range(2))
    cu, off = cu_of(lens, first), torch.arange(batch, dtype=torch.int64, device="cuda") * channels
    kinds = dict(gate=gate, input=input)
    results = []
    for divided in (True, False):
        size = gated.workspace_bytes(channels, batch, rows)
        ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda") if divided else None
        state, ds = start.clone(), torch.full_like(start, 5.0)
        out, dx = (torch.full((rows, channels), 5.0, dtype=x, device="cuda") for _ in range(2))
        dg = torch.full((rows, channels), 5.0, dtype=g, device="cuda")
        saves = torch.full((gated.saves_rows(batch, rows), channels), 3.0, device="cuda")
        gated.prefill_varlen(channels, rows, cu, max(lens), c.g, c.x, state, off, out=out, saves=saves, workspace=ws, **kinds)
        gated.backward_varlen(channels, rows, cu, max(lens), c.g, c.x, saves, off, c.dout, dg, dx, dstate=dstate, dstate_in=ds, workspace=ws, **kinds)
        assert mods["core"].device_status() == 0
        for t in (out, dg, dx):
            assert (t[:first] == 5).all() and (t[first + n:] == 5).all()
        results.append((out, state, dg, dx, ds))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    at = slice(first, first + n)
    h, hb, end, endb = oracle.forward(lens, c.g[at], c.x[at], start, gate, input)
    oracle.close(out[at], h, hb, "out")
    oracle.close(state, end, endb, "state")
    for got, want, name in zip((dg[at], dx[at], ds), oracle.backward(lens, c.g[at], c.x[at], start, c.dout[at], dstate, gate, input), ("dg", "dx", "ds")):
        oracle.close(got, *want, name)
