"""Sequences that are divided over the GPU (long ones of few channels, with a workspace): the bits of a walk, and what 64 bits give."""
import importlib

import pytest

torch = pytest.importorskip("torch")
import gated_oracle as oracle
from test_gpu_gated import BF, F32, Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gated():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return importlib.import_module("glm53f-afd_b200.gated")


SHAPES = [(64, [3000, 5, 0, 1300]), (63, [2000, 1]), (130, [64, 1100]), (192, [4096])]


def all_of(c, m, workspace):
    saves = c.saves(m)
    out, state = c.prefill(m, workspace, saves)
    return (out, state, saves, *c.backward(m, saves, workspace))


@pytest.mark.parametrize("channels,lens", SHAPES, ids=lambda v: str(v).replace(" ", ""))
@pytest.mark.parametrize("gate,input,g,x,pad", [("decay", "plain", F32, BF, 0), ("sigmoid", "complement", BF, BF, 0), ("decay", "complement", BF, F32, 3)])
def test_divided_and_walked(gated, channels, lens, gate, input, g, x, pad):
    c = Case(channels, lens, gate, input, g, x, pad=pad, apart=2)
    divided, walked = all_of(c, gated, c.workspace(gated)), all_of(c, gated, None)
    for a, b in zip(divided, walked):
        assert torch.equal(a, b)
    want, bound, ends, ends_bound = oracle.forward(lens, c.g, c.x, c.state, gate, input)
    oracle.close(divided[0], want, bound, "out")
    oracle.close(c.states(divided[1]), ends, ends_bound, "state")
    for got, (value, limit), what in zip((divided[3], divided[4], c.states(divided[5])), oracle.backward(lens, c.g, c.x, c.state, c.dout, c.dstate, gate, input), ("dg", "dx", "dstate")):
        oracle.close(got, value, limit, what)
