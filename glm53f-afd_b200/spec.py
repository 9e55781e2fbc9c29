"""Verification of drafted tokens against the target's distribution: what stands between a verify and its commit.  And what is reported of the same
logits: log probabilities, entropy and alternatives (`logprobs`), with their gradients.

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


MOST_TOP, MOST_VOCAB = 32, 2_000_000


def _per_row(t, what, rows, dtype=torch.float32):
    _need(t, what, (dtype,), rows)
    if t.numel() != rows:
        raise Invalid(f"{what} holds {t.numel()} elements for {rows} rows")


def _logits(t, what):
    """(rows, vocab, row stride, kind) of a [rows][vocab] tensor of logits."""
    if t is None or t.dim() != 2:
        raise Invalid(f"{what} must be [rows][vocab]")
    rows, vocab = t.shape
    ld = _rows(t, what, rows, vocab, (torch.float32, torch.bfloat16))
    if vocab > MOST_VOCAB:
        raise Invalid(f"a vocabulary of {vocab}, at most {MOST_VOCAB}")
    return rows, vocab, ld, LOGITS_F32 if t.dtype == torch.float32 else LOGITS_BF16


def logprobs(logits, tokens, logprob, *, temperature=None, entropy=None, lse=None, top=None):
    """glm53f_kda_logprobs.  Of each row of `logits` [rows][vocab] (f32 or bf16), p = softmax(logits / temperature[row]): writes f32 [rows] `logprob`, log p of
    tokens[row] (int32; outside the vocabulary: none, 0), `entropy` and `lse` (for `logprobs_backward`), and in `top` = (int32 ids, f32 values), both
    [rows][up to 32], the largest logits' indices, ties to the lowest, with their log p (-1 and -inf where fewer logits are above -inf).  tokens
    and logprob may be None together, as may the others.  temperature f32 [rows]; 0 or less, and None: 1."""
    code = ffi.host().logprobs(logits, tokens, logprob, temperature, entropy, lse, top)
    if code >= 0:
        return _launched(code, "glm53f_kda_logprobs")
    # Not the plain accepted call: the same checks here, with their errors.
    rows, vocab, ld, kind = _logits(logits, "logits")
    if (tokens is None) != (logprob is None):
        raise Invalid("tokens and logprob come together")
    if tokens is not None:
        _per_row(tokens, "tokens", rows, torch.int32)
    for t, name in ((logprob, "logprob"), (temperature, "temperature"), (entropy, "entropy"), (lse, "lse")):
        if t is not None:
            _per_row(t, name, rows)
    ids, values, n = None, None, 0
    if top is not None:
        ids, values = top
        if ids.dim() != 2 or ids.shape[0] != rows or not 1 <= ids.shape[1] <= MOST_TOP or ids.shape != values.shape:
            raise Invalid(f"top must be two tensors [{rows}][1 to {MOST_TOP}], got {tuple(ids.shape)} and {tuple(values.shape)}")
        n = ids.shape[1]
        _need(ids, "top's indices", (torch.int32,), rows * n)
        _need(values, "top's values", (torch.float32,), rows * n)
    if logprob is None and entropy is None and lse is None and top is None:
        raise Invalid("nothing to write")
    _same_device(logits, tokens, logprob, temperature, entropy, lse, ids, values)
    _launched(ffi.glm53f_kda_logprobs(rows, vocab, _ptr(logits), kind, ld, _ptr(tokens), _ptr(temperature), _ptr(logprob), _ptr(entropy), _ptr(lse), n,
                                      _ptr(ids), _ptr(values), _stream()), "glm53f_kda_logprobs")


def logprobs_backward(logits, tokens, lse, dlogprob, dlogits, *, temperature=None, entropy=None, dentropy=None):
    """glm53f_kda_logprobs_backward: writes `dlogits` (the logits' type; may be the logits themselves) from the gradients of `logprobs`' logprob and entropy (f32
    [rows]; one of them may be None).  lse and, with dentropy, entropy are what `logprobs` gave for the same logits, tokens and temperature."""
    code = ffi.host().logprobs_backward(logits, tokens, lse, dlogprob, dlogits, temperature, entropy, dentropy)
    if code >= 0:
        return _launched(code, "glm53f_kda_logprobs_backward")
    rows, vocab, ld, kind = _logits(logits, "logits")
    if dlogits is None or dlogits.dtype != logits.dtype or dlogits.shape != logits.shape:
        raise Invalid("dlogits has the logits' type and shape")
    _, _, dld, _ = _logits(dlogits, "dlogits")
    _per_row(tokens, "tokens", rows, torch.int32)
    _per_row(lse, "lse", rows)
    for t, name in ((temperature, "temperature"), (entropy, "entropy"), (dlogprob, "dlogprob"), (dentropy, "dentropy")):
        if t is not None:
            _per_row(t, name, rows)
    if dlogprob is None and dentropy is None:
        raise Invalid("no gradient to pass on")
    if dentropy is not None and entropy is None:
        raise Invalid("dentropy needs the entropy")
    if rows and (dlogits.data_ptr() != logits.data_ptr() or dld != ld):
        size = logits.element_size()
        if (dlogits.data_ptr() < logits.data_ptr() + ((rows - 1) * ld + vocab) * size
                and logits.data_ptr() < dlogits.data_ptr() + ((rows - 1) * dld + vocab) * size):
            raise Invalid("dlogits must be the logits or memory of its own")
    _same_device(logits, tokens, lse, dlogprob, dlogits, temperature, entropy, dentropy)
    _launched(ffi.glm53f_kda_logprobs_backward(rows, vocab, _ptr(logits), kind, ld, _ptr(tokens), _ptr(temperature), _ptr(lse), _ptr(entropy), _ptr(dlogprob),
                                               _ptr(dentropy), _ptr(dlogits), dld, _stream()), "glm53f_kda_logprobs_backward")


def _same_device(*tensors):
    here = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.device.index != here:
            raise Invalid(f"a tensor on {t.device}, the current device is cuda:{here}")
