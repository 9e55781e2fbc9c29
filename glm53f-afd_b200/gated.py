"""Gated linear recurrence channel by channel, on torch CUDA tensors: h_t = a_t h_{t-1} + c_t x_t, out_t = h_t.

The vector-state companion of `linear`, for layers that keep one value a channel; not in the reference.  `gate` says what g is: "decay", a = e^g
with g a log decay, or "sigmoid", a = sigmoid(g) with g as its projection leaves it.  `input` says c: "plain", 1, or "complement", 1 - a.
Conventions are `core`'s: extents are checked on the host, a rejected launch raises `Invalid`, a CUDA error `CudaError`, launches
are asynchronous on the current torch stream, nothing is allocated.

g, x, out and their gradients are [rows][channels], f32 or bf16 (out and the gradients of x's and g's types), rows any stride apart, so slices of a fused
projection's rows will do.  States are f32, [channels] a request, at state_off[b] elements.  Gradients are calls of their own (`backward_varlen`),
not nodes of an autograd graph.
"""
from __future__ import annotations

import torch

from . import ffi
from .core import Invalid, _launched, _need, _ptr, _stream

GATES = {"decay": 0, "sigmoid": 1}       # GLM53F_KDA_SCAN_SIGMOID
INPUTS = {"plain": 0, "complement": 2}   # GLM53F_KDA_SCAN_COMPLEMENT
G_BF16, X_BF16 = 4, 8


def _matrix(t, what, rows, channels, dtype=None):
    """(address, row stride) of `rows` rows of `channels` values, f32 or bf16 (or of the type named)."""
    if t is None:
        raise Invalid(f"{what} is required")
    if not t.is_cuda:
        raise Invalid(f"{what} must be a CUDA tensor")
    if t.dtype not in (torch.float32, torch.bfloat16) if dtype is None else t.dtype != dtype:
        raise Invalid(f"{what} has dtype {t.dtype}")
    if t.dim() != 2 or t.shape[0] < rows or t.shape[1] != channels or (channels > 1 and t.stride(1) != 1):
        raise Invalid(f"{what} must be {rows} rows of {channels} values, each contiguous; got {tuple(t.shape)}, strides {tuple(t.stride())}")
    stride = t.stride(0) if t.shape[0] > 1 else channels
    if stride < channels:
        raise Invalid(f"{what}'s rows overlap")
    return (t.data_ptr() if rows else 256), stride  # (no rows: an address that is not used)


def _state(t, what, channels, max_state_off):
    if t is None or not t.is_cuda or t.dtype != torch.float32 or not t.is_contiguous():
        raise Invalid(f"{what} must be a contiguous CUDA tensor of float32")
    if max_state_off is not None and (max_state_off < 0 or t.numel() < max_state_off + channels):
        raise Invalid(f"{what}: a request's region exceeds the buffer")


def _apart_or_same(a, b, what):
    if b is not None and a is not None and b.data_ptr() != a.data_ptr():
        if b.data_ptr() < a.data_ptr() + a.numel() * 4 and a.data_ptr() < b.data_ptr() + b.numel() * 4:
            raise Invalid(f"{what} must be the same memory or memory of its own")


def _common(channels, rows, cu_rows, state_off, gate, input, max_len=0):
    if gate not in GATES or input not in INPUTS:
        raise Invalid(f"gate {gate!r}, input {input!r}: one of {', '.join(GATES)} and of {', '.join(INPUTS)}")
    if channels < 1 or channels > 0x7fffffff or rows < 0 or rows > 0x7fffffff:
        raise Invalid(f"{rows} rows of {channels} channels")
    if not 0 <= max_len <= rows:
        raise Invalid(f"max_len {max_len} of {rows} rows")
    _need(cu_rows, "cu_rows", (torch.int32,), 1)
    batch = cu_rows.numel() - 1
    _need(state_off, "state_off", (torch.int64,), batch)
    return batch


def _kinds(gate, input):
    """The flags that name a call's kinds, or what the native path takes for none."""
    return GATES.get(gate, -1) | INPUTS.get(input, -1)


def _flags(gate, input, g, x):
    return GATES[gate] | INPUTS[input] | (G_BF16 if g.dtype == torch.bfloat16 else 0) | (X_BF16 if x.dtype == torch.bfloat16 else 0)


def _here(*tensors):
    here = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.device.index != here:
            raise Invalid(f"a tensor on {t.device}, the current device is cuda:{here}")


def _workspace(t):
    if t is None or t.numel() == 0:
        return None, 0
    if not t.is_cuda or not t.is_contiguous() or t.data_ptr() % 16:
        raise Invalid("workspace must be a contiguous CUDA tensor that lies on 16 bytes")
    return t.data_ptr(), t.numel() * t.element_size()


def decode_batch(channels, rows, cu_rows, g, x, state, state_off, *, gate="decay", input="plain", keep=None, state_out="in_place", out=None,
                 max_state_off=None):
    """glm53f_kda_scan_decode_batch: the recurrence row by row, for single tokens and windows.  `rows` = total rows (host); `cu_rows`
    int32 [batch + 1], `state_off` int64 [batch] and `keep` int32 [batch] (the rows of each request that count; None: all) on the device.
    state_out: "in_place", None (a verify: not written) or a tensor; out=None writes no outputs (a commit of kept rows).  A verify and a commit
    of k rows leave the bits of k single-row calls."""
    code = ffi.host().scan(False, channels, rows, 0, cu_rows, g, x, state, state_off, _kinds(gate, input), keep, state_out, out, None, None, max_state_off)
    if code >= 0:
        return _launched(code, "glm53f_kda_scan_decode_batch")
    # Not the plain accepted call: the same checks here, with their errors.
    batch = _common(channels, rows, cu_rows, state_off, gate, input)
    gp, gs = _matrix(g, "g", rows, channels)
    xp, xs = _matrix(x, "x", rows, channels)
    op, os = (None, 0) if out is None else _matrix(out, "out", rows, channels, x.dtype)
    if keep is not None:
        _need(keep, "keep", (torch.int32,), batch)
    so = _state_out(state, state_out, channels, max_state_off)
    if so is None and out is None:
        raise Invalid("neither states nor outputs to write")
    _here(cu_rows, g, x, state, state_off, keep, so, out)
    _launched(ffi.glm53f_kda_scan_decode_batch(channels, batch, _ptr(cu_rows), _ptr(keep), gp, gs, xp, xs, _flags(gate, input, g, x), _ptr(state), _ptr(so),
                                               _ptr(state_off), op, os, _stream()), "glm53f_kda_scan_decode_batch")


def _state_out(state, state_out, channels, max_state_off):
    _state(state, "state", channels, max_state_off)
    so = state if isinstance(state_out, str) else state_out
    if so is not None and so is not state:
        _state(so, "state_out", channels, max_state_off)
        if so.numel() < state.numel():
            raise Invalid("state_out is smaller than the state")
        _apart_or_same(state, so, "state_out")
    return so


def workspace_bytes(channels, batch, rows):
    """The workspace with which `prefill_varlen` and `backward_varlen` divide sequences of more than 64 rows over the GPU."""
    return int(ffi.glm53f_kda_scan_workspace_bytes(channels, batch, rows))


def saves_rows(batch, rows):
    """Rows of the f32 [saves_rows][channels] tensor in which `prefill_varlen` leaves what `backward_varlen` starts from."""
    return int(ffi.glm53f_kda_scan_saves_rows(batch, rows))


def _saves(t, channels, batch, rows):
    if not t.is_cuda or t.dtype != torch.float32 or not t.is_contiguous() or t.numel() < saves_rows(batch, rows) * channels or t.data_ptr() % 8:
        raise Invalid(f"saves must be a contiguous CUDA tensor of at least {saves_rows(batch, rows)} x {channels} float32 values")


def prefill_varlen(channels, rows, cu_rows, max_len, g, x, state, state_off, *, gate="decay", input="plain", state_out="in_place", out=None, saves=None,
                   workspace=None, max_state_off=None):
    """glm53f_kda_scan_prefill_varlen: packed sequences, the longest of at most max_len rows.  out=None writes the end states only.  `saves`: f32
    [saves_rows(batch, rows)][channels], for a backward pass.  `workspace`: a CUDA uint8 tensor of `workspace_bytes` bytes, or None: results are the same
    bits, long sequences of few channels take longer."""
    code = ffi.host().scan(True, channels, rows, max_len, cu_rows, g, x, state, state_off, _kinds(gate, input), None, state_out, out, saves, workspace, max_state_off)
    if code >= 0:
        return _launched(code, "glm53f_kda_scan_prefill_varlen")
    batch = _common(channels, rows, cu_rows, state_off, gate, input, max_len)
    gp, gs = _matrix(g, "g", rows, channels)
    xp, xs = _matrix(x, "x", rows, channels)
    op, os = (None, 0) if out is None else _matrix(out, "out", rows, channels, x.dtype)
    so = _state_out(state, state_out, channels, max_state_off)
    if so is None:
        raise Invalid("a prefill writes the state")
    if saves is not None:
        _saves(saves, channels, batch, rows)
    wp, wn = _workspace(workspace)
    _here(cu_rows, g, x, state, state_off, so, out, saves, workspace)
    _launched(ffi.glm53f_kda_scan_prefill_varlen(channels, batch, _ptr(cu_rows), rows, max_len, gp, gs, xp, xs, _flags(gate, input, g, x), _ptr(state),
                                                 _ptr(so), _ptr(state_off), op, os, _ptr(saves), wp, wn, _stream()), "glm53f_kda_scan_prefill_varlen")


def backward_varlen(channels, rows, cu_rows, max_len, g, x, saves, state_off, dout, dg, dx, *, gate="decay", input="plain", dstate=None, dstate_in=None,
                    workspace=None, max_state_off=None):
    """glm53f_kda_scan_backward_varlen: from dout (x's type) and `dstate` (f32, the gradient of the end states at state_off; None: zero), writes dg (g's type), dx (x's) and
    `dstate_in` (the start states' gradient; None: not wanted; may be `dstate`).  g, x, saves, gate, input and the row ranges are those of the `prefill_varlen` call."""
    code = ffi.host().scan_backward(channels, rows, max_len, cu_rows, g, x, saves, state_off, _kinds(gate, input), dout, dg, dx, dstate, dstate_in, workspace,
                                    max_state_off)
    if code >= 0:
        return _launched(code, "glm53f_kda_scan_backward_varlen")
    batch = _common(channels, rows, cu_rows, state_off, gate, input, max_len)
    gp, gs = _matrix(g, "g", rows, channels)
    xp, xs = _matrix(x, "x", rows, channels)
    yp, ys = _matrix(dout, "dout", rows, channels, x.dtype)
    dgp, dgs = _matrix(dg, "dg", rows, channels, g.dtype)
    dxp, dxs = _matrix(dx, "dx", rows, channels, x.dtype)
    if saves is None:
        raise Invalid("saves is required")
    _saves(saves, channels, batch, rows)
    for t, name in ((dstate, "dstate"), (dstate_in, "dstate_in")):
        if t is not None:
            _state(t, name, channels, max_state_off)
    _apart_or_same(dstate, dstate_in, "dstate_in")
    wp, wn = _workspace(workspace)
    _here(cu_rows, g, x, saves, state_off, dout, dg, dx, dstate, dstate_in, workspace)
    _launched(ffi.glm53f_kda_scan_backward_varlen(channels, batch, _ptr(cu_rows), rows, max_len, gp, gs, xp, xs, _flags(gate, input, g, x), _ptr(saves), yp, ys,
                                                  _ptr(dstate), _ptr(dstate_in), _ptr(state_off), dgp, dgs, dxp, dxs, wp, wn, _stream()),
              "glm53f_kda_scan_backward_varlen")
