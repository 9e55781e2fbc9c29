"""The fused projection's activations (csrc/proj_gemm.cuh) compiled for the host, against 64 bits: relative errors where results are normal numbers, a step of the
smallest where they are not.  The approximating instructions are stood in for by exact ones with their flushing to zero.  No GPU."""
import math
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

SOURCE = os.path.join(os.path.dirname(__file__), "..", "glm53f-afd_b200", "csrc", "proj_gemm.cuh")
U = 2.0 ** -24
ACTS = {"silu": 2, "gelu": 3, "gelu_tanh": 4, "sigmoid": 5}

HARNESS = r"""
#include <cmath>
#include <cstdio>
#include <cstdlib>
enum { GLM53F_PROJ_NONE, GLM53F_PROJ_RELU, GLM53F_PROJ_SILU, GLM53F_PROJ_GELU, GLM53F_PROJ_GELU_TANH, GLM53F_PROJ_SIGMOID };
constexpr float kLog2e = 1.4426950408889634f;
static float flushed(double x) { return std::fabs(x) < 0x1p-126 ? (float)std::copysign(0.0, x) : (float)x; }
static float ex2_ftz(float x) { return flushed(std::exp2((double)flushed(x))); }
static float rcp_approx(float x) { return flushed(1.0 / (double)flushed(x)); }
SOURCE
int main(int, char** argv) {
    float y;
    while (fread(&y, 4, 1, stdin) == 1) {
        float r = 0;
        switch (atoi(argv[1])) {
            case 2: r = proj_act<2>(y); break;
            case 3: r = proj_act<3>(y); break;
            case 4: r = proj_act<4>(y); break;
            case 5: r = proj_act<5>(y); break;
        }
        fwrite(&r, 4, 1, stdout);
    }
}
"""


@pytest.fixture(scope="module")
def act(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    with open(SOURCE) as f:
        text = f.read()
    # From the first of the activations' functions up to the one that takes several values at once.
    start = min(m.start() for m in re.finditer(r"(template <[^>]*>\n)?__device__ __forceinline__ float proj_(?!bias)", text))
    body = text[start:text.index("// N values at once")].replace("__device__ __forceinline__", "static")
    body = re.sub(r'asm\("rcp.approx.f32.*?\)\);', "r = (float)(1.0 / (double)u);", body)
    where = tmp_path_factory.mktemp("activations")
    (where / "x.cpp").write_text(HARNESS.replace("SOURCE", body))
    subprocess.check_call([gxx, "-std=c++17", "-O1", "-ffp-contract=off", "-o", str(where / "x"), str(where / "x.cpp")])

    def run(name, y):
        out = subprocess.run([str(where / "x"), str(ACTS[name])], input=np.asarray(y, np.float32).tobytes(), capture_output=True, check=True).stdout
        return np.frombuffer(out, np.float32).astype(np.float64)

    return run


def exact(name, y):
    y = np.asarray(y, np.float32).astype(np.float64)
    sigmoid = lambda z: np.where(z < 0, np.exp(np.minimum(z, 0)) / (1 + np.exp(np.minimum(z, 0))), 1 / (1 + np.exp(-np.maximum(z, 0))))
    if name == "silu":
        return y * sigmoid(y), np.abs(y)
    if name == "sigmoid":
        return sigmoid(y), np.abs(y)
    if name == "gelu_tanh":
        z = 2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)
        return y * sigmoid(z), np.abs(z)
    return np.array([0.5 * v * math.erfc(-v / math.sqrt(2)) for v in y]), y * y


def grid(lo, hi):
    near = np.concatenate([np.geomspace(1e-37, 1, 4000), -np.geomspace(1e-37, 1, 4000)])
    return np.unique(np.concatenate([np.linspace(lo, hi, 40001), near, [0.0]]).astype(np.float32))


@pytest.mark.parametrize("name,lo", [("silu", -110.0), ("sigmoid", -110.0), ("gelu_tanh", -12.0)])
def test_sigmoids_and_their_products(act, name, lo):
    """The exponential's argument z has a constant and a product rounded (gelu_tanh's cubic eight more): 2 |z| (10 |z|) half steps of the result; its square
    root's own half step twice, the sum, the reciprocal and three products one each."""
    y = grid(lo, 100.0)
    got, (want, z) = act(name, y), exact(name, y)
    bound = ((10 if name == "gelu_tanh" else 2) * z + 8) * U * np.abs(want) + 2.0 ** -149
    if name == "sigmoid":
        bound += np.where(want < 2.0 ** -126 * (1 + 2.0 ** -14), 2.0 ** -125, 0.0)  # subnormal results are 0
    far = np.abs(got - want) - bound
    assert np.all(far <= 0), (y[far > 0][:5], got[far > 0][:5], want[far > 0][:5])


def test_gelu(act):
    """erfc's fit is within 1.6e-7.  The exponent 2 e = -z^2 log2 e + P - 1, z^2 = y^2 / 2, is rounded: e's product, its constant and the sum one half step
    of |e| each and e^2's twice: 3 x 2 ln 2 |e| half steps, |e| at most 0.361 y^2 + 1.5; P's coefficients and steps 10 half steps of 1.5; what is taken of the factors 8."""
    y = grid(-13.5, 40.0)
    got, (want, square) = act("gelu", y), exact("gelu", y)
    tail = np.array([0.5 * abs(v) * math.erfc(abs(v) / math.sqrt(2)) for v in y.astype(np.float64)])  # what is taken from max(y, 0)
    bound = (1.6e-7 + (4.2 * (0.361 * square + 1.5) + 10 * 1.5 * 1.4 + 8) * U) * tail + U * np.abs(want) + 2.0 ** -149
    far = np.abs(got - want) - bound
    assert np.all(far <= 0), (y[far > 0][:5], got[far > 0][:5], want[far > 0][:5])


@pytest.mark.parametrize("name", list(ACTS))
def test_at_the_ends(act, name):
    got = act(name, [np.inf, np.nan, 3e38, -3e38, -1e5])
    assert got[0] == (1.0 if name == "sigmoid" else np.inf) and np.isnan(got[1])
    assert got[2] == (1.0 if name == "sigmoid" else np.float32(3e38)) and got[3] == 0 and got[4] == 0
