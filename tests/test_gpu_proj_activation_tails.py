"""The fused projection's activations on the device over the range in which they have results, tails down to the smallest subnormals and arguments near zero: f32
results of y by the bias alone (x = 0), at few rows and on SM pairs.

Bounds, in half steps of f32 (U): those of test_proj_activations_cpu.py, and what the approximating instructions add: 2^-22 of an exponential, which is squared (8),
a step of a reciprocal (2; through gelu's polynomial 6)."""
import importlib
import math

import numpy as np
import pytest

from test_proj_activations_cpu import U, exact, grid

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def results(name, y, rows):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    proj = importlib.import_module("glm53f-afd_b200.proj")
    n = (len(y) + 7) // 8 * 8
    bias = torch.zeros(n)
    bias[:len(y)] = torch.from_numpy(y)
    x, w = torch.zeros(rows, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, 64, dtype=torch.bfloat16, device="cuda")
    out = torch.empty(rows, n, device="cuda")
    proj.fused(x, 64, 0, proj.Bf16Mat.dense(w), rows, out, n, 0, True, bias=bias.cuda(), activation=name)
    assert bool((out.view(torch.int32) == out[:1].view(torch.int32)).all())
    return out[0, :len(y)].cpu().numpy().astype(np.float64)


@pytest.mark.parametrize("rows", [1, 130])
@pytest.mark.parametrize("name,lo", [("silu", -110.0), ("sigmoid", -110.0), ("gelu_tanh", -12.0)])
def test_sigmoids_and_their_products(name, lo, rows):
    y = grid(lo, 100.0)
    got, (want, z) = results(name, y, rows), exact(name, y)
    bound = ((10 if name == "gelu_tanh" else 2) * z + 18) * U * np.abs(want) + 2.0 ** -149
    if name == "sigmoid":
        bound += np.where(want < 2.0 ** -126 * (1 + 2.0 ** -14), 2.0 ** -125, 0.0)  # subnormal results are 0
    far = np.abs(got - want) - bound
    assert np.all(far <= 0), (y[far > 0][:5], got[far > 0][:5], want[far > 0][:5])


@pytest.mark.parametrize("rows", [1, 130])
def test_gelu(rows):
    y = grid(-13.5, 40.0)
    got, (want, square) = results("gelu", y, rows), exact("gelu", y)
    tail = np.array([0.5 * abs(v) * math.erfc(abs(v) / math.sqrt(2)) for v in y.astype(np.float64)])
    bound = (1.6e-7 + (4.2 * (0.361 * square + 1.5) + 10 * 1.5 * 1.4 + 24) * U) * tail + U * np.abs(want) + 2.0 ** -149
    far = np.abs(got - want) - bound
    assert np.all(far <= 0), (y[far > 0][:5], got[far > 0][:5], want[far > 0][:5])
