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
from .paged import MAX_NODES, _call

MAX_DRAFTS = 32


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
    which token follows; a temperature of 0 takes what the target would have picked greedily, and
    needs neither where it is given as a number.  temperature: a number, or fp32 [batch] on the
    device, which is not looked at beforehand: it needs both.  counts: int32
    [batch], how many drafted tokens each sequence has, where not all.

    Returns (tokens int64 [batch, drafts + 1]: the taken ones, the one that follows, then -1;
    accepted int32 [batch])."""
    key = (target_logits.device, target_logits.shape, target_logits.stride(), draft_tokens.shape, draft_tokens.stride(),
           None if draft_logits is None else (draft_logits.shape, draft_logits.stride()),
           None if uniforms is None else (uniforms.shape, uniforms.stride()),
           None if noise is None else (noise.shape, noise.stride()))
    plan = _plans.get(key)
    if plan is None:
        plan = _plan(target_logits, draft_tokens, draft_logits, uniforms, noise)
        if len(_plans) >= 256:
            _plans.clear()
        _plans[key] = plan
    dev, batch, drafts, vocab, seq_t, ld_t, ld_tok, seq_d, ld_d, ld_u, ld_n, bytes_ = plan
    pt, ptok = _address(target_logits, "target_logits", _F32, dev), _address(draft_tokens, "draft_tokens", torch.int64, dev)
    pd = pu = pn = each = pc = None
    one = 0.0
    if draft_logits is not None:
        pd = _address(draft_logits, "draft_logits", _F32, dev)
    if uniforms is not None:
        pu = _address(uniforms, "uniforms", _F32, dev)
    if noise is not None:
        pn = _address(noise, "noise", _F32, dev)
    if isinstance(temperature, torch.Tensor):
        each = _vector(temperature, "temperature", _F32, batch, dev)
    else:
        one = float(temperature)
        if not (one == 0.0 or 1e-20 <= one <= 1e20):
            raise ValueError(f"temperature must be 0, or positive and finite, got {one}")
    if (pn is None or (drafts and pu is None)) and (each is not None or one > 0):
        raise ValueError("a temperature above 0 needs uniforms and noise")
    if counts is not None:
        pc = _vector(counts, "counts", torch.int32, batch, dev)
    tokens = torch.empty((batch, drafts + 1), dtype=torch.int64, device=dev)
    accepted = torch.empty(batch, dtype=torch.int32, device=dev)
    # a large call's scratch, for this call alone and on its stream
    ws = torch.empty(bytes_, dtype=torch.uint8, device=dev) if bytes_ else None
    _call(_native.lib().otf_verify_drafts, dev, pt, seq_t, ld_t, pd, seq_d, ld_d, ptok, ld_tok, pu, ld_u, pn, ld_n, each, one, pc,
          tokens.data_ptr(), accepted.data_ptr(), batch, drafts, vocab, ws.data_ptr() if bytes_ else None, bytes_)
    return tokens, accepted


def verify_tree(target_logits: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, *,
                starts: Optional[torch.Tensor] = None, batch: Optional[int] = None, depth: Optional[int] = None,
                noise: Optional[torch.Tensor] = None, temperature: Union[float, torch.Tensor] = 1.0
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Choose a way through trees of drafted tokens (otf_verify_tree).

    target_logits: fp32 [n, vocab], the target's logits behind every node; tokens (int64 [n]) and parents (int32
    [n]) of the nodes, sequence b's from starts[b] on (int32 [batch + 1] on the device), or n / ``batch`` each (one
    sequence by default), 64 at most, as ``PagedKVCache.attend_tree`` takes them: node 0 is the root, the last token
    that is certain, and a node's parent comes before it.  At each node, from the root on, the target draws the token
    that follows, with noise (fp32 [batch, depth + 1, vocab], exponentially distributed) at a temperature above 0,
    else its first largest logit; the walk goes on at a child that holds the token, the first of several, until
    there is none or ``depth`` (noise.shape[1] - 1, or 63) are taken.  Every token is so distributed as the target
    alone draws it, whatever was drafted.  temperature: a number, or fp32 [batch] on the device.

    Returns (tokens int64 [batch, depth + 1]: the taken ones, the one that follows, then -1; path int32 [batch,
    depth]: the taken nodes, then -1, for ``PagedKVCache.keep``; accepted int32 [batch])."""
    key = (target_logits.device, target_logits.shape, target_logits.stride(), tokens.shape, parents.shape,
           None if starts is None else starts.shape, batch, depth, None if noise is None else (noise.shape, noise.stride()))
    plan = _tree_plans.get(key)
    if plan is None:
        plan = _plan_tree(target_logits, tokens, parents, starts, batch, depth, noise)
        if len(_tree_plans) >= 256:
            _tree_plans.clear()
        _tree_plans[key] = plan
    dev, n, vocab, ld, batch, depth, seq_n, ld_n, bytes_ = plan
    pt = _address(target_logits, "target_logits", _F32, dev)
    ptok, pp = _address(tokens, "tokens", torch.int64, dev), _address(parents, "parents", torch.int32, dev)
    ps = None if starts is None else _vector(starts, "starts", torch.int32, batch + 1, dev)
    if not (tokens.is_contiguous() and parents.is_contiguous()):
        raise ValueError("tokens and parents must be contiguous")
    pn = each = None
    if noise is not None:
        pn = _address(noise, "noise", _F32, dev)
    one = 0.0
    if isinstance(temperature, torch.Tensor):
        each = _vector(temperature, "temperature", _F32, batch, dev)
    else:
        one = float(temperature)
        if not (one == 0.0 or 1e-20 <= one <= 1e20):
            raise ValueError(f"temperature must be 0, or positive and finite, got {one}")
    if pn is None and (each is not None or one > 0):
        raise ValueError("a temperature above 0 needs noise")
    out, path, accepted = tokens.new_empty((batch, depth + 1)), parents.new_empty((batch, depth)), parents.new_empty(batch)
    # a small call's scratch, for this call alone and on its stream
    ws = tokens.new_empty(bytes_ // 8) if bytes_ else None
    _call(_native.lib().otf_verify_tree, dev, pt, ld, ptok, pp, ps, n, pn, seq_n, ld_n, each, one, out.data_ptr(),
          path.data_ptr() if depth else None, accepted.data_ptr(), batch, depth, vocab, ws.data_ptr() if bytes_ else None, bytes_)
    return out, path, accepted


def _plan_tree(target: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, starts: Optional[torch.Tensor],
               batch: Optional[int], depth: Optional[int], noise: Optional[torch.Tensor]) -> tuple:
    _native._need_cuda(target, "target_logits")
    if target.dim() != 2 or target.shape[0] == 0 or target.shape[1] == 0:
        raise ValueError(f"target_logits must be [n, vocab], got {list(target.shape)}")
    n, vocab = target.shape
    ld, = _rows(target, "target_logits", (n, vocab))
    if ld < vocab:
        raise ValueError(f"target_logits needs rows that do not overlap, got strides {target.stride()}")
    for name, t in (("tokens", tokens), ("parents", parents)):
        if t.shape != (n,):
            raise ValueError(f"{name} must be a contiguous [{n}] vector, got {list(t.shape)}")
    if starts is not None:
        if starts.dim() != 1 or starts.shape[0] < 2 or (batch is not None and batch != starts.shape[0] - 1):
            raise ValueError(f"starts must be a [batch + 1] vector, got {list(starts.shape)}")
        batch = starts.shape[0] - 1
    else:
        batch = 1 if batch is None else int(batch)
        if batch < 1 or n % batch or n // batch > MAX_NODES:
            raise ValueError(f"{n} nodes do not divide among {batch} sequences of {MAX_NODES} at most; give starts")
    if depth is None:
        depth = MAX_NODES - 1 if noise is None or noise.dim() != 3 else noise.shape[1] - 1
    if int(depth) != depth or not 0 <= depth < MAX_NODES:
        raise ValueError(f"depth must be 0 to {MAX_NODES - 1}, got {depth}")
    depth, seq_n, ld_n = int(depth), 0, 0
    if noise is not None:
        seq_n, ld_n = _rows(noise, "noise", (batch, depth + 1, vocab))
        if seq_n < 0 or ld_n < vocab:
            raise ValueError(f"noise needs rows that do not overlap, got strides {noise.stride()}")
    size = _native.lib().otf_verify_tree_workspace_bytes(n, vocab)
    if size < 0:
        raise ValueError("shape not supported by otf_verify_tree")
    return target.device, n, vocab, ld, batch, depth, seq_n, ld_n, size


_F32 = torch.float32
# shapes and strides of earlier calls' arguments, with what their checks found
_plans: dict = {}
_tree_plans: dict = {}


def _address(t: torch.Tensor, name: str, dtype: torch.dtype, dev: torch.device) -> int:
    if t.dtype is not dtype or t.device != dev:
        raise ValueError(f"{name} must be {dtype} on {dev}, got {t.dtype} on {t.device}")
    return t.data_ptr()


def _vector(t: torch.Tensor, name: str, dtype: torch.dtype, n: int, dev: torch.device) -> int:
    if t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{n}] vector, got {list(t.shape)} with strides {t.stride()}")
    return _address(t, name, dtype, dev)


def _rows(t: torch.Tensor, name: str, shape: Tuple[int, ...]) -> Tuple[int, ...]:
    """The strides of all dimensions but the last, whose values lie next to one another."""
    if tuple(t.shape) != shape or (t.stride(-1) != 1 and shape[-1] > 1):
        raise ValueError(f"{name} must be {list(shape)} with a unit inner stride, got {list(t.shape)} with strides "
                         f"{t.stride()}")
    if len(shape) == 2:
        return (t.stride(0) if shape[0] > 1 else shape[1],)
    return (t.stride(0) if shape[0] > 1 else 0), (t.stride(1) if shape[1] > 1 else shape[2])


def _plan(target: torch.Tensor, tokens: torch.Tensor, draft: Optional[torch.Tensor], uniforms: Optional[torch.Tensor],
          noise: Optional[torch.Tensor]) -> tuple:
    _native._need_cuda(target, "target_logits")
    if target.dim() != 3 or target.shape[0] == 0 or target.shape[1] == 0 or target.shape[2] == 0:
        raise ValueError(f"target_logits must be [batch, drafts + 1, vocab], got {list(target.shape)}")
    batch, drafts, vocab = target.shape[0], target.shape[1] - 1, target.shape[2]
    if drafts > MAX_DRAFTS:
        raise ValueError(f"0 to {MAX_DRAFTS} drafted tokens, got {drafts}")
    seq_t, ld_t = _rows(target, "target_logits", (batch, drafts + 1, vocab))
    ld_tok, = _rows(tokens, "draft_tokens", (batch, drafts))
    seq_d = ld_d = ld_u = ld_n = 0
    if draft is not None:
        seq_d, ld_d = _rows(draft, "draft_logits", (batch, drafts, vocab))
    if uniforms is not None:
        ld_u, = _rows(uniforms, "uniforms", (batch, drafts))
    if noise is not None:
        ld_n, = _rows(noise, "noise", (batch, vocab))
    n = _native.lib().otf_verify_workspace_bytes(batch, drafts, vocab, 0 if draft is None or drafts == 0 else 1)
    if n < 0:
        raise ValueError("shape not supported by otf_verify_drafts")
    return target.device, batch, drafts, vocab, seq_t, ld_t, ld_tok, seq_d, ld_d, ld_u, ld_n, n
