"""The projections either side of the KDA core: host side of include/glm53f_proj.h.

Mirror of the reference's `Bf16Mat` and `Gemm::bf16` (crates/glm53f-forward/src/gemm.rs:35-48, 212-235) and of the
three GEMMs a KDA layer issues on its normed input (crates/glm53f-forward/src/forward.rs:3494-3542).  Where the
reference picks its CUDA-core GEMV for up to 8 rows and cuBLAS above, every row count goes to the tcgen05 kernel
here.  Tensors are torch CUDA tensors; there is no CPU path.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import ffi
from .core import CudaError, Invalid

_BF = (torch.bfloat16, torch.int16, torch.uint16)
HIDDEN = 4096
KDA_HEADS, KDA_DIM = 64, 128
KDA_WIDTH = KDA_HEADS * KDA_DIM          # 8192
KDA_QKV = 3 * KDA_WIDTH                  # 24,576
KDA_P_COLS = KDA_QKV + KDA_HEADS         # 24,640: [q | k | v | beta logits] (crates/glm53f-forward/src/shape.rs:23-32)


def _launched(code: int, what: str) -> None:
    if code == 0:
        return
    if code == 1:
        raise Invalid(f"{what}: rejected by the launcher")
    raise CudaError(code, what)


@dataclass
class Bf16Mat:
    """A BF16 weight [groups][n][k] on the device (gemm.rs:35-48): row stride `ld`, group stride `gstride` (elements)."""

    t: torch.Tensor
    n: int
    k: int
    ld: int
    groups: int = 1
    gstride: int = 0

    @classmethod
    def dense(cls, t: torch.Tensor) -> "Bf16Mat":
        if t.dim() == 2:
            return cls(t, t.shape[0], t.shape[1], t.shape[1], 1, 0)
        return cls(t, t.shape[1], t.shape[2], t.shape[2], t.shape[0], t.shape[1] * t.shape[2])

    def bytes(self) -> int:
        return self.groups * self.n * self.k * 2


def bf16(x: torch.Tensor, ldx: int, x_gstride: int, w: Bf16Mat, rows: int, out: torch.Tensor, ldo: int, o_gstride: int,
         out_f32: bool = False, x_offset: int = 0, out_offset: int = 0) -> None:
    """out[g][m][o] = sum_k x[g][m][k] w[g][o][k] (Gemm::bf16, gemm.rs:212-235); offsets in elements of x / out."""
    if rows == 0:
        return
    job = _job(x, ldx, x_gstride, w, rows, out, ldo, o_gstride, out_f32, x_offset, out_offset)
    code = ffi.load().glm53f_kda_proj_bf16(*job, torch.cuda.current_stream().cuda_stream)
    _launched(code, "glm53f_kda_proj_bf16")


ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4, "sigmoid": 5}  # GLM53F_PROJ_*


def fused(x: torch.Tensor, ldx: int, x_gstride: int, w: Bf16Mat, rows: int, out: torch.Tensor, ldo: int, o_gstride: int, out_f32: bool = False,
          x_offset: int = 0, out_offset: int = 0, *, bias: torch.Tensor | None = None, activation: str = "none",
          residual: torch.Tensor | None = None, ldr: int | None = None, r_gstride: int | None = None, residual_offset: int = 0) -> None:
    """`bf16` with an epilogue in the same launch: out = residual + act(x w^T + bias), formed in f32 and rounded once.  bias [groups][n]
    (bf16 or f32); residual of out's type, with out's strides unless others are given, `out` itself or memory of its own."""
    if activation not in ACTIVATIONS:
        raise Invalid(f"activation {activation!r}: one of {', '.join(ACTIVATIONS)}")
    if rows == 0:
        return
    code = ffi.host().proj_fused(x, ldx, x_gstride, w.t, w.n, w.k, w.ld, w.groups, w.gstride, rows, out, ldo, o_gstride, out_f32, x_offset, out_offset, bias,
                                 ACTIVATIONS[activation], residual, ldr, r_gstride, residual_offset)
    if code >= 0:
        return _launched(code, "glm53f_kda_proj_bf16_fused")
    # Not the plain accepted call: the same checks here, with their errors.
    if min(rows, ldx, x_gstride, ldo, o_gstride, x_offset, out_offset) < 0:
        raise Invalid("rows, strides and offsets are not negative")
    job = _job(x, ldx, x_gstride, w, rows, out, ldo, o_gstride, out_f32, x_offset, out_offset)
    e = ffi.ProjEpilogue(activation=ACTIVATIONS[activation])
    if bias is not None:
        if bias.dtype not in (torch.float32, *_BF) or not bias.is_contiguous() or bias.numel() != w.groups * w.n:
            raise Invalid(f"bias must be {w.groups} x {w.n} contiguous values, bf16 or f32")
        e.bias, e.bias_gstride, e.bias_f32 = bias.data_ptr(), w.n, int(bias.dtype == torch.float32)
    if residual is not None:
        ldr, r_gstride = ldo if ldr is None else ldr, o_gstride if r_gstride is None else r_gstride
        if (residual.dtype == torch.float32) != out_f32 or (not out_f32 and residual.dtype not in _BF):
            raise Invalid("the residual has out's type")
        if residual_offset < 0 or ldr < w.n or r_gstride < 0 or residual.numel() < residual_offset + (w.groups - 1) * r_gstride + (rows - 1) * ldr + w.n:
            raise Invalid("the residual is smaller than the shapes named")
        e.residual, e.ldr, e.r_gstride = residual.data_ptr() + residual_offset * residual.element_size(), ldr, r_gstride
    here = torch.cuda.current_device()
    for t in (x, w.t, out, bias, residual):
        if t is not None and (not t.is_cuda or t.device.index != here):
            raise Invalid(f"a tensor on {t.device}, the current device is cuda:{here}")
    code = ffi.load().glm53f_kda_proj_bf16_fused(ffi.ProjJob(*job), e, torch.cuda.current_stream().cuda_stream)
    _launched(code, "glm53f_kda_proj_bf16_fused")


INT4_GROUPS = (32, 64, 128)
INT4_MOST_K = 65536


@dataclass
class Int4Mat:
    """A weight [n][k] of 4-bit codes, laid out for `int4`: w = scale * (code - zero), a scale and a zero point (`zeros`; else 8) for each `group` k."""

    t: torch.Tensor
    n: int
    k: int
    group: int
    zeros: bool

    @classmethod
    def pack(cls, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, *, group: int = 128) -> "Int4Mat":
        """From codes uint8 [n][k / 2] (the even k in the low halves), scales bf16 [n][k / group] and zeros uint8 [n][k / group] of 0 .. 15, on the
        device: one launch, on the current stream."""
        if codes.dim() != 2 or codes.dtype != torch.uint8:
            raise Invalid("codes must be uint8 [n][k / 2]")
        n, k = codes.shape[0], 2 * codes.shape[1]
        if group not in INT4_GROUPS or n < 1 or k < 64 or k % 64 or k % group or k > INT4_MOST_K:
            raise Invalid(f"a weight of {n} x {k} in groups of {group}: k a multiple of 64 and of the group (32, 64 or 128), at most {INT4_MOST_K}")
        for t, name, dtype in ((scales, "scales", torch.bfloat16), (zeros, "zeros", torch.uint8)):
            if t is not None and (t.dtype != dtype or tuple(t.shape) != (n, k // group)):
                raise Invalid(f"{name} must be {dtype} [{n}][{k // group}], got {t.dtype} {tuple(t.shape)}")
        here = torch.cuda.current_device()
        for t in (codes, scales, zeros):
            if t is not None and (not t.is_cuda or t.device.index != here or not t.is_contiguous()):
                raise Invalid(f"codes, scales and zeros are contiguous CUDA tensors on the current device, cuda:{here}")
        packed = torch.empty(ffi.glm53f_kda_int4_bytes(n, k, group, int(zeros is not None)), dtype=torch.uint8, device=codes.device)
        _launched(ffi.glm53f_kda_int4_pack(codes.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(), n, k, group, packed.data_ptr(),
                                           torch.cuda.current_stream().cuda_stream), "glm53f_kda_int4_pack")
        return cls(packed, n, k, group, zeros is not None)

    @classmethod
    def quantise(cls, w: torch.Tensor, *, group: int = 128, zeros: bool = False) -> "Int4Mat":
        """The nearest codes of a weight [n][k]: a group's scale is its largest magnitude / 7, or with `zeros` its span (0 within) / 15, as bf16."""
        if w.dim() != 2 or group not in INT4_GROUPS or w.shape[1] % group or w.shape[1] % 64:
            raise Invalid(f"a weight [n][k], k a multiple of 64 and of the group (32, 64 or 128), got {tuple(w.shape)}")
        n, k = w.shape
        g = w.float().contiguous().view(n, k // group, group)
        if zeros:
            low, high = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
            scales = ((high - low) / 15).bfloat16()
        else:
            scales = (g.abs().amax(-1) / 7).bfloat16()
        step = torch.where(scales == 0, 1.0, scales.float())
        zero = torch.round(-low / step).clamp(0, 15) if zeros else torch.full_like(step, 8.0)
        codes = (torch.round(g / step[..., None]) + zero[..., None]).clamp(0, 15).to(torch.uint8).view(n, k)
        return cls.pack(codes[:, 0::2] | (codes[:, 1::2] << 4), scales, zero.to(torch.uint8) if zeros else None, group=group)

    def bytes(self) -> int:
        return self.n * self.k // 2 + self.n * (self.k // self.group) * (3 if self.zeros else 2)


def int4(x: torch.Tensor, ldx: int, w: Int4Mat, rows: int, out: torch.Tensor, ldo: int, out_f32: bool = False, x_offset: int = 0, out_offset: int = 0) -> None:
    """out[m][o] = sum_k x[m][k] w[o][k] with 4-bit weights (glm53f_kda_proj_int4); strides and offsets in elements, as in `bf16`.  No weight is rounded: group sums
    are multiplied by their scales in f32."""
    if rows == 0:
        return
    code = ffi.host().proj_int4(x, ldx, w.t, w.n, w.k, w.group, w.zeros, rows, out, ldo, out_f32, x_offset, out_offset)
    if code >= 0:
        return _launched(code, "glm53f_kda_proj_int4")
    # Not the plain accepted call: the same checks here, with their errors.
    if min(rows, ldx, ldo, x_offset, out_offset) < 0 or max(rows, ldx, ldo) > 0x7fffffff:
        raise Invalid("rows, strides and offsets are not negative, and rows and strides below 2^31")
    if x.dtype not in _BF:
        raise Invalid("x is bf16")
    if (out.dtype != torch.float32) if out_f32 else (out.dtype not in _BF):
        raise Invalid("out is f32 when out_f32, else bf16")
    if ldx < w.k or ldo < w.n:
        raise Invalid(f"rows of {ldx} and {ldo} for {w.k} inputs and {w.n} outputs")
    if x.numel() < x_offset + (rows - 1) * ldx + w.k or out.numel() < out_offset + (rows - 1) * ldo + w.n or not x.is_contiguous() or not out.is_contiguous():
        raise Invalid("a buffer is not contiguous or smaller than the shapes named")
    here = torch.cuda.current_device()
    for t in (x, w.t, out):
        if not t.is_cuda or t.device.index != here:
            raise Invalid(f"a tensor on {t.device}, the current device is cuda:{here}")
    if w.t.numel() < ffi.glm53f_kda_int4_bytes(w.n, w.k, w.group, int(w.zeros)):
        raise Invalid("the weight is smaller than the shapes named")
    code = ffi.load().glm53f_kda_proj_int4(x.data_ptr() + 2 * x_offset, ldx, w.t.data_ptr(), w.n, w.k, w.group, int(w.zeros), rows,
                                           out.data_ptr() + out_offset * out.element_size(), int(out_f32), ldo, torch.cuda.current_stream().cuda_stream)
    _launched(code, "glm53f_kda_proj_int4")


def _job(x, ldx, x_gstride, w: Bf16Mat, rows, out, ldo, o_gstride, out_f32=False, x_offset=0, out_offset=0) -> tuple:
    """The checked arguments of one GEMM: those of glm53f_kda_proj_bf16 before the stream, the fields of ffi.ProjJob."""
    if x.dtype not in _BF or w.t.dtype not in _BF:
        raise Invalid("x and the weight are bf16")
    if out.dtype != (torch.float32 if out_f32 else x.dtype) and not (not out_f32 and out.element_size() == 2):
        raise Invalid("out is f32 when out_f32, else bf16")
    need_x = x_offset + (w.groups - 1) * x_gstride + (rows - 1) * ldx + w.k
    need_o = out_offset + (w.groups - 1) * o_gstride + (rows - 1) * ldo + w.n
    if x.numel() < need_x or out.numel() < need_o or w.t.numel() < (w.groups - 1) * w.gstride + (w.n - 1) * w.ld + w.k:
        raise Invalid("a buffer is smaller than the shapes named")
    return (x.data_ptr() + 2 * x_offset, ldx, x_gstride, w.t.data_ptr(), w.ld, w.gstride, w.groups, rows, w.n, w.k,
            out.data_ptr() + out_offset * out.element_size(), 1 if out_f32 else 0, ldo, o_gstride)


@dataclass
class KdaProjW:
    """The projection weights of one KDA layer (crates/glm53f-forward/src/weights.rs:145-162): the fused [q|k|v|b]
    weight [24,640][4096], the low-rank gates' first factor [256][4096] (f and g stacked) and second factors
    [2][8192][128]."""

    qkvb: Bf16Mat
    fga: Bf16Mat
    fgb: Bf16Mat


def kda_input_projections(normed: torch.Tensor, rows: int, w: KdaProjW, p: torch.Tensor, fga: torch.Tensor, ag: torch.Tensor) -> None:
    """The three GEMMs of a KDA layer's input (forward.rs:3494-3542): p [rows][24,640] = normed . qkvb^T; fga
    [rows][256] = normed . fga^T; ag [rows][2 x 8192] = per group g, fga[:, 128 g : 128 g + 128] . fgb[g]^T."""
    if rows == 0:
        return
    both = (_job(normed, HIDDEN, 0, w.fga, rows, fga, 2 * KDA_DIM, 0), _job(normed, HIDDEN, 0, w.qkvb, rows, p, KDA_P_COLS, 0))
    apart = _disjoint(p, fga) and _disjoint(p, normed) and _disjoint(fga, normed)
    stream = torch.cuda.current_stream().cuda_stream
    if apart:  # the first gate factor beside the fused projection of the same rows
        _launched(ffi.glm53f_kda_proj_bf16_many((ffi.ProjJob * 2)(*(ffi.ProjJob(*j) for j in both)), 2, stream), "glm53f_kda_proj_bf16_many")
    else:
        bf16(normed, HIDDEN, 0, w.qkvb, rows, p, KDA_P_COLS, 0)
        bf16(normed, HIDDEN, 0, w.fga, rows, fga, 2 * KDA_DIM, 0)
    bf16(fga, 2 * KDA_DIM, KDA_DIM, w.fgb, rows, ag, 2 * KDA_WIDTH, KDA_WIDTH)


def _disjoint(a: torch.Tensor, b: torch.Tensor) -> bool:
    lo, hi = sorted(((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in (a, b)))
    return lo[1] <= hi[0]
