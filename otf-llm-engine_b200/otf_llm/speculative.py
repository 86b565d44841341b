"""Verification of drafted tokens against the target model's logits, on the native kernels.

A draft (a smaller model, or tokens looked up in the prompt) proposes a few tokens per sequence,
the target model scores them all in one pass, and ``verify_drafts`` keeps the tokens that the
target's distribution allows, so that what is produced is distributed as if the target had
produced it token by token.  The reference decodes one token per pass with HF's generate
(otf_llm/run_symmetric_2bit.py:188-215); the greedy pick of one row is ``_native.i8_head_argmax``.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _native
from .paged import _on, _stream

MAX_DRAFTS = 32


def _rows3(t: torch.Tensor, name: str, shape, dev) -> Tuple[int, int]:
    """Check fp32 [batch, rows, vocab] values with a unit inner stride; (sequence stride, row stride)."""
    if t.device != dev or t.dtype != torch.float32 or tuple(t.shape) != shape or (t.stride(2) != 1 and shape[2] > 1):
        raise ValueError(f"{name} must be fp32 {list(shape)} with a unit inner stride on {dev}, got {t.dtype} "
                         f"{list(t.shape)} with strides {t.stride()} on {t.device}")
    return (t.stride(0) if shape[0] > 1 else 0), (t.stride(1) if shape[1] > 1 else shape[2])


def _rows2(t: torch.Tensor, name: str, dtype, shape, dev) -> int:
    if t.device != dev or t.dtype != dtype or tuple(t.shape) != shape or (t.stride(1) != 1 and shape[1] > 1):
        raise ValueError(f"{name} must be {dtype} {list(shape)} with a unit inner stride on {dev}, got {t.dtype} "
                         f"{list(t.shape)} with strides {t.stride()} on {t.device}")
    return t.stride(0) if shape[0] > 1 else shape[1]


def verify_drafts(target_logits: torch.Tensor, draft_tokens: torch.Tensor, *,
                  draft_logits: Optional[torch.Tensor] = None, uniforms: Optional[torch.Tensor] = None,
                  noise: Optional[torch.Tensor] = None, temperature: Union[float, torch.Tensor] = 1.0,
                  counts: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Take or refuse drafted tokens (otf_verify_drafts).

    target_logits: fp32 [batch, drafts + 1, vocab], row j the target's logits behind j drafted
    tokens; draft_tokens: int64 [batch, drafts], 0 to 32 of them; draft_logits: fp32
    [batch, drafts, vocab], the logits that they were drawn from, or None where the draft was
    certain of them.  uniforms (fp32 [batch, drafts], in [0, 1)) decide which are taken, noise
    (fp32 [batch, vocab], exponentially distributed, e.g. ``torch.empty(...).exponential_()``)
    which token follows; a temperature of 0 needs neither and takes what the target would have
    picked greedily.  temperature: a number, or fp32 [batch] on the device.  counts: int32
    [batch], how many drafted tokens each sequence has, where not all.

    Returns (tokens int64 [batch, drafts + 1]: the taken ones, the one that follows, then -1;
    accepted int32 [batch])."""
    _native._need_cuda(target_logits, "target_logits")
    dev = target_logits.device
    if target_logits.dim() != 3 or target_logits.shape[0] == 0 or target_logits.shape[2] == 0:
        raise ValueError(f"target_logits must be [batch, drafts + 1, vocab], got {list(target_logits.shape)}")
    batch, drafts, vocab = target_logits.shape[0], target_logits.shape[1] - 1, target_logits.shape[2]
    if not 0 <= drafts <= MAX_DRAFTS:
        raise ValueError(f"0 to {MAX_DRAFTS} drafted tokens, got {drafts}")
    seq_t, ld_t = _rows3(target_logits, "target_logits", (batch, drafts + 1, vocab), dev)
    ld_tok = _rows2(draft_tokens, "draft_tokens", torch.int64, (batch, drafts), dev)
    seq_d = ld_d = ld_u = ld_n = 0
    if draft_logits is not None:
        seq_d, ld_d = _rows3(draft_logits, "draft_logits", (batch, drafts, vocab), dev)
    if uniforms is not None:
        ld_u = _rows2(uniforms, "uniforms", torch.float32, (batch, drafts), dev)
    if noise is not None:
        ld_n = _rows2(noise, "noise", torch.float32, (batch, vocab), dev)
    each, one = None, 0.0
    if isinstance(temperature, torch.Tensor):
        _rows2(temperature.view(1, -1), "temperature", torch.float32, (1, batch), dev)
        each = temperature.data_ptr()
        if noise is None or (drafts and uniforms is None):
            raise ValueError("temperatures of each sequence need uniforms and noise")
    else:
        one = float(temperature)
        if not (one == 0.0 or 1e-20 <= one <= 1e20):
            raise ValueError(f"temperature must be 0, or positive and finite, got {one}")
        if one > 0 and (noise is None or (drafts and uniforms is None)):
            raise ValueError("a temperature above 0 needs uniforms and noise")
    if counts is not None:
        _rows2(counts.view(1, -1), "counts", torch.int32, (1, batch), dev)
    tokens = torch.empty((batch, drafts + 1), dtype=torch.int64, device=dev)
    accepted = torch.empty(batch, dtype=torch.int32, device=dev)
    L = _native.lib()
    n = L.otf_verify_workspace_bytes(batch, drafts, vocab)
    if n < 0:
        raise ValueError("shape not supported by otf_verify_drafts")
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    with _on(dev):
        st = L.otf_verify_drafts(target_logits.data_ptr(), seq_t, ld_t,
                                 None if draft_logits is None else draft_logits.data_ptr(), seq_d, ld_d,
                                 draft_tokens.data_ptr(), ld_tok, None if uniforms is None else uniforms.data_ptr(),
                                 ld_u, None if noise is None else noise.data_ptr(), ld_n, each, one,
                                 None if counts is None else counts.data_ptr(), tokens.data_ptr(), accepted.data_ptr(),
                                 batch, drafts, vocab, ws.data_ptr(), n, _stream(dev))
    _native._check(st, "otf_verify_drafts")
    return tokens, accepted
