"""Linear attention with one decay a head, on torch CUDA tensors: S_t = e^g_t S_{t-1} + v_t k_t^T, y_t = scale S_t q_t.

The recurrence that hybrid decoders use where the KDA layers have a delta rule and a decay for every key channel; not in the
reference.  Conventions are `core`'s: extents are checked on the host, a rejected launch raises `Invalid`, a CUDA error
`CudaError`, launches are asynchronous on the current torch stream, nothing is allocated.

q and k are [rows][qk_heads][128], v and out [rows][heads][128] (bf16; the two inner dimensions may be one), rows any stride apart that
is a multiple of eight elements, so slices of a fused projection's rows will do.  g holds log decays, f32: [rows][heads], or
[heads] for decays that are the same in every row.  States are [heads][128 (v)][128 (k)] a request, f32 or bf16.
"""
from __future__ import annotations

import torch

from . import ffi
from .core import DK, DV, Invalid, _BF, _launched, _need, _ptr, _state_kind, _stream


def _row_tensor(t, what, rows, heads):
    """(address, row stride) of `rows` rows of heads x 128 bf16 values."""
    if t is None:
        raise Invalid(f"{what} is required")
    if not t.is_cuda:
        raise Invalid(f"{what} must be a CUDA tensor")
    if t.dtype not in _BF:
        raise Invalid(f"{what} has dtype {t.dtype}")
    width = heads * DK
    if t.dim() == 2:
        ok = t.shape[1] == width and t.stride(1) == 1
    else:
        ok = t.dim() == 3 and t.shape[1:] == (heads, DK) and t.stride(2) == 1 and (heads == 1 or t.stride(1) == DK)
    if not ok or t.shape[0] < rows:
        raise Invalid(f"{what} must be {rows} rows of {heads} x {DK} values, the row contiguous; got {tuple(t.shape)}, strides {tuple(t.stride())}")
    stride = t.stride(0) if t.shape[0] > 1 else width
    if stride % 8 or t.data_ptr() % 16:
        raise Invalid(f"{what} must lie on 16 bytes with a row stride that is a multiple of eight")
    if stride < width:
        raise Invalid(f"{what}'s rows overlap")
    return (t.data_ptr() if rows else 256), stride  # (no rows: an address that is not used)


def _tokens(heads, qk_heads, rows, cu_rows, q, k, v, g, state, state_off, out):
    if heads < 1 or qk_heads < 1 or heads % qk_heads:
        raise Invalid(f"{qk_heads} heads of q and k do not divide {heads} heads")
    _need(cu_rows, "cu_rows", (torch.int32,), 1)
    batch = cu_rows.numel() - 1
    _need(state_off, "state_off", (torch.int64,), batch)
    args = []
    for t, name, n in ((q, "q", qk_heads), (k, "k", qk_heads), (v, "v", heads)):
        args += _row_tensor(t, name, rows, n)
    if g is None or not g.is_cuda or g.dtype != torch.float32:
        raise Invalid("g must be a CUDA tensor of float32")
    if g.dim() == 1:
        ok, g_stride = g.shape[0] == heads and (heads == 1 or g.stride(0) == 1), 0
    else:
        ok = g.dim() == 2 and g.shape[0] >= rows and g.shape[1] == heads and (heads == 1 or g.stride(1) == 1)
        g_stride = (g.stride(0) if g.shape[0] > 1 else heads) if ok else 0
        ok = ok and (g_stride >= heads or rows <= 1)
        g_stride = max(g_stride, heads)
    if not ok:
        raise Invalid(f"g must be [{rows}][{heads}] or [{heads}], got {tuple(g.shape)}, strides {tuple(g.stride())}")
    args += [g.data_ptr() if g.numel() else 256, g_stride]
    if state is None or not state.is_cuda or not state.is_contiguous():
        raise Invalid("state must be a contiguous CUDA tensor")
    kind = _state_kind(state)
    o, o_stride = (None, 0) if out is None else _row_tensor(out, "out", rows, heads)
    here = torch.cuda.current_device()
    for t in (cu_rows, state_off, q, k, v, g, state, out):
        if t is not None and t.device.index != here:
            raise Invalid(f"a tensor on {t.device}, the current device is cuda:{here}")
    return batch, args, kind, o, o_stride


def _state_out(state, state_out, batch, heads, max_state_off):
    if max_state_off is not None and (max_state_off < 0 or state.numel() < max_state_off + heads * DV * DK):
        raise Invalid("state: a request's region exceeds the buffer")
    so = state if isinstance(state_out, str) else state_out
    if so is not None and so is not state:
        if so.dtype != state.dtype or so.numel() < state.numel() or not so.is_cuda or not so.is_contiguous() or so.device != state.device:
            raise Invalid("state_out must match the state's type and size")
        if so.data_ptr() != state.data_ptr():
            size = state.element_size()
            if so.data_ptr() < state.data_ptr() + state.numel() * size and state.data_ptr() < so.data_ptr() + so.numel() * size:
                raise Invalid("state_out must be the state itself or memory of its own")
    return so


def _scale(scale):
    return DK ** -0.5 if scale is None else float(scale)


def decode_batch(heads, rows, cu_rows, q, k, v, g, state, state_off, *, qk_heads=None, keep=None, state_out="in_place", scale=None, out=None,
                 max_state_off=None):
    """glm53f_kda_lin_decode_batch: the recurrence row by row, for single tokens and windows.  `rows` = total rows (host);
    `cu_rows` int32 [batch + 1], `state_off` int64 [batch] and `keep` int32 [batch] (the rows of each request that count; None: all)
    on the device.  state_out: "in_place", None (a verify: not written) or a tensor; out=None writes no outputs (a commit of kept
    rows).  A verify and a commit of k rows leave the bits of k single-row calls."""
    qk_heads = heads if qk_heads is None else qk_heads
    code = ffi.host().lin(False, heads, qk_heads, rows, 0, cu_rows, q, k, v, g, state, state_off, keep, state_out, scale, out, None, max_state_off)
    if code >= 0:
        return _launched(code, "glm53f_kda_lin_decode_batch")
    # Not the plain accepted call: the same checks here, with their errors.
    batch, args, kind, o, o_stride = _tokens(heads, qk_heads, rows, cu_rows, q, k, v, g, state, state_off, out)
    if keep is not None:
        _need(keep, "keep", (torch.int32,), batch)
    so = _state_out(state, state_out, batch, heads, max_state_off)
    if so is None and out is None:
        raise Invalid("neither states nor outputs to write")
    _launched(ffi.glm53f_kda_lin_decode_batch(heads, qk_heads, batch, _ptr(cu_rows), _ptr(keep), *args, _ptr(state), _ptr(so), _ptr(state_off), kind,
                                              _scale(scale), o, o_stride, _stream()), "glm53f_kda_lin_decode_batch")


def prefill_workspace_bytes(heads, batch, max_len):
    """The workspace with which `prefill_varlen` runs sequences of up to max_len rows in as many segments as help."""
    return int(ffi.glm53f_kda_lin_prefill_workspace_bytes(heads, batch, max_len))


def prefill_varlen(heads, rows, cu_rows, max_len, q, k, v, g, state, state_off, *, qk_heads=None, state_out="in_place", scale=None, out=None,
                   workspace=None, max_state_off=None):
    """glm53f_kda_lin_prefill_varlen: chunked prefill of packed sequences, the longest of at most max_len rows.  `workspace`: a CUDA uint8
    tensor of `prefill_workspace_bytes` bytes, or None."""
    qk_heads = heads if qk_heads is None else qk_heads
    code = ffi.host().lin(True, heads, qk_heads, rows, max_len, cu_rows, q, k, v, g, state, state_off, None, state_out, scale, out, workspace, max_state_off)
    if code >= 0:
        return _launched(code, "glm53f_kda_lin_prefill_varlen")
    if not 0 <= max_len <= rows:
        raise Invalid(f"max_len {max_len} of {rows} rows")
    if out is None:
        raise Invalid("out is required")
    batch, args, kind, o, o_stride = _tokens(heads, qk_heads, rows, cu_rows, q, k, v, g, state, state_off, out)
    so = _state_out(state, state_out, batch, heads, max_state_off)
    if so is None:
        raise Invalid("a prefill writes the state")
    nbytes = 0
    if workspace is not None:
        if not workspace.is_cuda or not workspace.is_contiguous() or workspace.device != state.device:
            raise Invalid("workspace must be a contiguous CUDA tensor on the state's device")
        nbytes = workspace.numel() * workspace.element_size()
    _launched(ffi.glm53f_kda_lin_prefill_varlen(heads, qk_heads, batch, _ptr(cu_rows), rows, max_len, *args, _ptr(state), _ptr(so), _ptr(state_off), kind,
                                                _scale(scale), o, o_stride, _ptr(workspace) if nbytes else None, nbytes, _stream()),
              "glm53f_kda_lin_prefill_varlen")
