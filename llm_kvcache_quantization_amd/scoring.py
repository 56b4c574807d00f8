"""Log probabilities of what a model answered: of given tokens, with the entropy and the likeliest alternatives.

:func:`token_logprobs` takes rows of logits in one pass.  ``generate_from_ids`` and ``sample_from_ids`` record it for the
tokens they choose.  Devices and streams are as in :mod:`paged`; there is no backward pass.

The reference takes the argmax of its logits and keeps nothing of them (src/engine/generate_loop.py:393).
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import _capi as C
from .paged import _INTEGERS, _call, _no_grad, _packer

MAX_TOP = 32
COLDEST, HOTTEST = 1e-30, 1e30  # temperatures: they, their inverses and the entropy's sums lie in fp32
_TYPES = {torch.float16: C.KVQ_LOGITS_F16, torch.bfloat16: C.KVQ_LOGITS_BF16, torch.float32: C.KVQ_LOGITS_F32}
_LOGPROBS = _packer(C.TokenLogprobsParams)


class TokenLogprobs(NamedTuple):
    """What :func:`token_logprobs` returns; ``logprobs`` is None without tokens, the last two without ``top``."""

    logprobs: Optional[Tensor]
    entropy: Tensor
    top_logprobs: Optional[Tensor]
    top_tokens: Optional[Tensor]


@functools.lru_cache(maxsize=256)
def _scratch(rows: int, vocab: int, top: int, kind: int) -> int:
    """Bytes of scratch of a call: a matter of its sizes alone."""
    p = C.TokenLogprobsParams()
    p.rows, p.vocab, p.top, p.logits_type, p.inv_temperature = rows, vocab, top, kind, 1.0
    return C.lib().kvq_token_logprobs_workspace_bytes(ctypes.byref(p))


def token_logprobs(logits: Tensor, tokens: Optional[Tensor] = None, top: int = 0, *, temperature: float = 1.0) -> TokenLogprobs:
    """Of each row of ``logits`` [..., V] (fp16, bf16 or fp32), with p = softmax(row / temperature):

    * ``logprobs`` fp32 [...]: log p of the row's token in ``tokens`` [...] (integers; NaN for one outside [0, V));
    * ``entropy`` fp32 [...]: -sum p log p, in nats;
    * ``top_tokens`` int64 and ``top_logprobs`` fp32 [..., top]: the ``top`` likeliest tokens (at most 32) and their log
      p, the lower token first among equal logits, NaN logits below all others.

    Sums are fp32; ``temperature`` is 1e-30 to 1e30.  -Inf logits, and those further below the row's largest than fp32
    goes, have probability 0; a row whose softmax is none (a NaN, a +Inf, nothing but -Inf) has NaN for its log
    probabilities and entropy.
    """
    if logits.ndim < 1 or not logits.is_cuda or logits.dtype not in _TYPES:
        raise ValueError(f"logits must be fp16, bf16 or fp32 [..., V] on a GPU, got {logits.dtype} {tuple(logits.shape)} on {logits.device}")
    shape, vocab, device = logits.shape[:-1], logits.shape[-1], logits.device
    if vocab < 1:
        raise ValueError("logits must have at least one token")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be 0 to {min(MAX_TOP, vocab)}, got {top}")
    if not COLDEST <= temperature <= HOTTEST:
        raise ValueError(f"temperature must be {COLDEST} to {HOTTEST}, got {temperature}")
    if tokens is not None:
        if tokens.shape != shape or tokens.dtype not in _INTEGERS:
            raise ValueError(f"tokens must be integers {tuple(shape)}, one for each row of logits, got {tokens.dtype} {tuple(tokens.shape)}")
        if tokens.dtype not in (torch.int32, torch.int64):
            tokens = tokens.to(torch.int64)
        if tokens.device != device:
            tokens = tokens.to(device)
        tokens = tokens.contiguous()
    _no_grad(logits)
    x = logits if logits.ndim == 2 else logits.reshape(-1, vocab)
    rows, (step, inner) = x.shape[0], x.stride()
    if vocab > 1 and inner != 1:
        x = x.contiguous()
        step = vocab
    if tokens is None:
        logprobs, entropy = None, x.new_empty(shape, dtype=torch.float32)
    else:
        logprobs, entropy = torch.empty_like(tokens, dtype=torch.float32), torch.empty_like(tokens, dtype=torch.float32)
    best = entropy.new_empty((*shape, top)) if top else None
    ids = x.new_empty((*shape, top), dtype=torch.int64) if top else None
    out = TokenLogprobs(logprobs, entropy, best, ids)
    if rows == 0:
        return out
    nbytes = _scratch(rows, vocab, top, _TYPES[x.dtype])
    scratch = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _call(C.lib().kvq_token_logprobs, _LOGPROBS.pack(
        x.data_ptr(), step, 0 if tokens is None else tokens.data_ptr(), 0 if tokens is None else logprobs.data_ptr(),
        entropy.data_ptr(), best.data_ptr() if top else 0, ids.data_ptr() if top else 0,
        0 if scratch is None else scratch.data_ptr(), nbytes, rows, vocab, top, _TYPES[x.dtype],
        tokens is not None and tokens.dtype == torch.int64, 1.0 / temperature, 0), device)
    return out
