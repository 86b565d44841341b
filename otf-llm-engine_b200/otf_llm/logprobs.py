"""Log probabilities of what a model answers with, on the native kernels.

``token_logprobs`` gives the log probability and the rank of one token per row of logits, the row's entropy and its
likeliest tokens, in one pass over the logits: what a server reports beside its tokens, and what scoring a text
needs.  The reference's runner leaves this to HF (otf_llm/run_symmetric_2bit.py:188-215); the greedy pick of a row is
``_native.i8_head_argmax``.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native
from .paged import _call
from .speculative import _rows

MAX_TOP = 32
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor        # fp32 [n]
    entropy: torch.Tensor         # fp32 [n]
    ranks: torch.Tensor           # int32 [n], 0: the likeliest
    top_tokens: torch.Tensor      # int64 [n, top]
    top_logprobs: torch.Tensor    # fp32 [n, top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0) -> TokenLogprobs:
    """Log probabilities of one token per row (otf_token_logprobs).

    logits: fp32, fp16 or bf16 [n, vocab] with a unit inner stride; tokens: int64 [n], a negative one asks for
    nothing (log probability 0, rank -1).  ``top``: how many of the likeliest tokens to list, 32 at most, equal ones
    by the lower index; where fewer have a logit above -inf, -1 and -inf follow.  NaN counts as -inf, +inf as the
    largest finite number.  A token outside the vocabulary gets a NaN and raises the ``_native.device_error`` flag."""
    key = (logits.device, logits.dtype, logits.shape, logits.stride(), tokens.shape, top)
    plan = _plans.get(key)
    if plan is None:
        plan = _plan(logits, tokens, top)
        if len(_plans) >= 256:
            _plans.clear()
        _plans[key] = plan
    dev, n, vocab, ld, dtype, top = plan
    if tokens.dtype is not torch.int64 or tokens.device != dev or not tokens.is_contiguous():
        raise ValueError(f"tokens must be contiguous int64 on {dev}, got {tokens.dtype} on {tokens.device}")
    # the three numbers of a row in one piece of memory
    values = torch.empty((3, n), dtype=torch.float32, device=dev)
    logprobs, entropy, ranks = values.unbind()
    ranks = ranks.view(torch.int32)
    top_tokens = tokens.new_empty((n, top))
    top_logprobs = values.new_empty((n, top))
    if n:
        at = values.data_ptr()
        _call(_native.lib().otf_token_logprobs, dev, logits.data_ptr(), ld, dtype, tokens.data_ptr(), n, vocab, top, at, at + 4 * n,
              at + 8 * n, top_tokens.data_ptr() if top else None, top_logprobs.data_ptr() if top else None)
    return TokenLogprobs(logprobs, entropy, ranks, top_tokens, top_logprobs)


# shapes and strides of earlier calls' arguments, with what their checks found
_plans: dict = {}


def _plan(logits: torch.Tensor, tokens: torch.Tensor, top: int) -> tuple:
    _native._need_cuda(logits, "logits")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits must be fp32, fp16 or bf16, got {logits.dtype}")
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must be [n, vocab], got {list(logits.shape)}")
    n, vocab = logits.shape
    if int(top) != top or not 0 <= top <= MAX_TOP:
        raise ValueError(f"top must be 0 to {MAX_TOP}, got {top}")
    ld, = _rows(logits, "logits", (n, vocab))
    if ld < vocab:
        raise ValueError(f"logits needs rows that do not overlap, got strides {logits.stride()}")
    if tokens.shape != (n,):
        raise ValueError(f"tokens must be a contiguous [{n}] vector, got {list(tokens.shape)}")
    return logits.device, n, vocab, ld, _DTYPES[logits.dtype], int(top)
