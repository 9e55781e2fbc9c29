"""Verification of drafted tokens against the target's distribution: what stands between a verify and its commit.

The reference keeps a draft while it equals the target's choice (crates/glm53f-coordinator/src/scheduler.rs:765-875); that is
the greedy case here.  With given random numbers the kept tokens and the one behind them are distributed as the target's own.
"""
from __future__ import annotations

import torch

from . import ffi
from .core import Invalid, _launched, _need, _ptr, _stream

PROBABILITIES, LOGITS_F32, LOGITS_BF16 = 0, 1, 2


def _rows(t, what, rows, vocab, dtypes):
    """Row stride of a [rows][vocab] tensor."""
    if not t.is_cuda or t.dim() != 2 or t.dtype not in dtypes:
        raise Invalid(f"{what} must be a 2-D CUDA tensor of {', '.join(str(d) for d in dtypes)}")
    if t.shape[0] < rows or t.shape[1] != vocab or vocab < 1 or (vocab > 1 and t.stride(1) != 1):
        raise Invalid(f"{what} must hold {rows} rows of {vocab} values, each contiguous; got {tuple(t.shape)}, strides {tuple(t.stride())}")
    stride = t.stride(0) if t.shape[0] > 1 else vocab
    if stride < vocab:
        raise Invalid(f"{what}'s rows overlap")
    return stride


def accept_batch(cu_rows, tokens, target, u, keep, next, *, probabilities=False, draft=None, temperature=None):
    """glm53f_kda_accept_batch.  Window b is rows [cu_rows[b], cu_rows[b + 1]) (int32, device): its first row holds the last certain token,
    the others drafted ones.  Row i of `target` [rows][vocab] judges tokens[i + 1]: logits (f32 or bf16, divided by temperature[b], f32;
    0: greedy; None: 1), or f32 probabilities.  `draft` f32 [rows][vocab]: row i is what tokens[i] was drawn from (None: the
    drafter had one choice).  u f32 [rows] in [0, 1): u[i] judges tokens[i], a window's first draws the next token.  Writes
    int32 keep[b], the rows to commit (1 .. the window's), and next[b], the token behind them (-1: the row left nothing)."""
    code = ffi.host().accept(cu_rows, tokens, target, u, keep, next, probabilities, draft, temperature)
    if code >= 0:
        return _launched(code, "glm53f_kda_accept_batch")
    # Not the plain accepted call: the same checks here, with their errors.
    _need(cu_rows, "cu_rows", (torch.int32,), 1)
    batch = cu_rows.numel() - 1
    _need(tokens, "tokens", (torch.int32,), 0)
    rows = tokens.numel()
    _need(u, "u", (torch.float32,), rows)
    _need(keep, "keep", (torch.int32,), batch)
    _need(next, "next", (torch.int32,), batch)
    if target is None or target.dim() != 2:
        raise Invalid("target must be [rows][vocab]")
    vocab = target.shape[1]
    ld = _rows(target, "target", rows, vocab, (torch.float32,) if probabilities else (torch.float32, torch.bfloat16))
    kind = PROBABILITIES if probabilities else LOGITS_F32 if target.dtype == torch.float32 else LOGITS_BF16
    draft_ld = 0 if draft is None else _rows(draft, "draft", rows, vocab, (torch.float32,))
    if temperature is not None:
        if probabilities:
            raise Invalid("probabilities have no temperature")
        _need(temperature, "temperature", (torch.float32,), batch)
    here = torch.cuda.current_device()
    for t in (cu_rows, tokens, target, u, keep, next, draft, temperature):
        if t is not None and t.device.index != here:
            raise Invalid(f"a tensor on {t.device}, the current device is cuda:{here}")
    if rows == 0 and batch > 0:  # only empty windows: their addresses are not used
        keep[:batch].zero_()
        next[:batch].fill_(-1)
        return
    _launched(ffi.glm53f_kda_accept_batch(batch, _ptr(cu_rows), vocab, _ptr(target), kind, ld, _ptr(tokens), _ptr(draft), draft_ld, _ptr(temperature),
                                          _ptr(u), _ptr(keep), _ptr(next), _stream()), "glm53f_kda_accept_batch")
