"""The most (request, head) pairs that the linear attention's launches hold: one more is refused, not handed to a launch that the device cannot make.  Nothing is
read and nothing is launched, so no GPU."""
import importlib

import pytest

from test_refusals_cpu import LINEAR, PREFILL, STEP, call


@pytest.fixture(scope="module")
def ffi(pkg):
    m = importlib.import_module("glm53f-afd_b200.ffi")
    m.load()
    return m


@pytest.mark.parametrize("heads,qk_heads,batch", [(1, 1, 0x20000000), (1, 1, 0x3fffffff), (2, 1, 0x10000000), (64, 64, 0x800000), (4, 2, 0x0fffffff), (65535, 5, 8193)])
def test_more_pairs_than_blocks(ffi, heads, qk_heads, batch):
    assert heads * batch * 4 > 0x7fffffff  # four blocks a pair
    wide = dict(heads=heads, qk_heads=qk_heads, batch=batch, q_stride=qk_heads * 128, k_stride=qk_heads * 128, v_stride=heads * 128, out_stride=heads * 128, g_stride=heads)
    assert call(ffi.glm53f_kda_lin_decode_batch, STEP, LINEAR, **wide) == 1
    assert call(ffi.glm53f_kda_lin_prefill_varlen, PREFILL, LINEAR, **wide) == 1
