"""The weights of a draw from logits (csrc/spec_accept.cu, logit_weight) compiled for the host: e^((l - max) / t) to the 1e-11 that its series leaves, 0 where that is
below e^-691, and never anything else, however small the temperature and however few steps of f32 lie between a logit and the largest.  No GPU."""
import math
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

SOURCE = os.path.join(os.path.dirname(__file__), "..", "glm53f-afd_b200", "csrc", "spec_accept.cu")

HARNESS = r"""
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
using std::fma;
static int __double2loint(double x) { int64_t b; memcpy(&b, &x, 8); return (int)(uint32_t)b; }
static int __double2hiint(double x) { int64_t b; memcpy(&b, &x, 8); return (int)(b >> 32); }
static double __hiloint2double(int hi, int lo) { int64_t b = (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo); double x; memcpy(&x, &b, 8); return x; }
constexpr int kCopies = 16;
SOURCE
int main() {
    static double power[32][kCopies];
    for (int j = 0; j < 32; ++j)
        for (int i = 0; i < kCopies; ++i) power[j][i] = exp2(j / 32.0);
    float x[3];
    while (fread(x, 4, 3, stdin) == 3) {  // l, max, t
        const double w = logit_weight(x[0], row_scale_of(x[1], x[2]), &power[0][5]);
        fwrite(&w, 8, 1, stdout);
    }
}
"""


@pytest.fixture(scope="module")
def weights(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    with open(SOURCE) as f:
        body = re.search(r"(constexpr double kTurns = .*?)__device__ __forceinline__ float finite_weight", f.read(), re.S).group(1)
    where = tmp_path_factory.mktemp("weights")
    (where / "x.cpp").write_text(HARNESS.replace("SOURCE", body.replace("__device__ __forceinline__", "static")))
    subprocess.check_call([gxx, "-std=c++17", "-O1", "-ffp-contract=off", "-o", str(where / "x"), str(where / "x.cpp")])

    def run(l, top, t):
        triples = np.stack(np.broadcast_arrays(np.float32(l), np.float32(top), np.float32(t)), -1).astype(np.float32)
        out = subprocess.run([str(where / "x")], input=triples.tobytes(), capture_output=True, check=True).stdout
        return np.frombuffer(out, np.float64)

    return run


def exact(l, top, t):
    x = (np.float64(np.float32(l)) - np.float64(np.float32(top))) / np.float64(np.float32(t))
    return x, np.exp(np.maximum(x, -700.0))


@pytest.mark.parametrize("top", [10.0, 100.0, 9000.0, -3.0, 1e-3, 1e30, 0.0])
@pytest.mark.parametrize("t", [1e-9, 1e-8, 1e-7, 1e-6, 1e-5, 1e-3, 0.6, 1.0, 40.0, 1e30])
def test_logits_a_few_steps_below_the_largest(weights, top, t):
    l, steps = np.float32(top), []
    for _ in range(40):
        steps.append(l)
        l = np.nextafter(l, np.float32(-np.inf))
    got = weights(steps, top, t)
    x, want = exact(np.array(steps), top, t)
    inside = x > -689.0
    assert got[0] == 1.0
    assert np.all((got >= 0) & (got <= 1 + 1e-11))
    assert np.all(got[x < -691.0] == 0)
    # x is formed with two roundings of 64 bits, of which e^x makes |x| times as much.
    assert np.all(np.abs(got - want)[inside] <= (1e-11 + 4 * 2.0 ** -53 * np.abs(x[inside])) * want[inside])


def test_over_the_whole_range(weights):
    r = np.random.default_rng(1)
    t = np.exp(r.uniform(math.log(1e-12), math.log(1e6), 200000)).astype(np.float32)
    top = (r.standard_normal(t.size) * np.exp(r.uniform(-5, 9, t.size))).astype(np.float32)
    l = np.minimum((top - t * r.uniform(0, 1500, t.size)).astype(np.float32), top)
    got = weights(l, top, t)
    x, want = exact(l, top, t)
    inside = x > -689.0
    assert inside.sum() > 10000 and (~inside).sum() > 10000
    assert np.all(np.abs(got - want)[inside] <= (1e-11 + 4 * 2.0 ** -53 * np.abs(x[inside])) * want[inside])
    assert np.all((got >= 0) & (got <= 1 + 1e-11)) and np.all(got[x < -691.0] == 0)


def test_masked_and_no_logits(weights):
    for l in (-math.inf, math.nan, -3.4e38):
        for t in (1e-9, 0.5, 1e5):
            assert weights([l], 3.0, t)[0] == 0.0
