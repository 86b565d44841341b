"""A key/value cache in pages for sequences of different lengths, on the native kernels.

``PagedKVCache`` holds one layer's pages: ``append`` turns new queries and keys by their rotary
positions and writes keys and values into the pages, ``attend`` is the attention of one or a few
new tokens per sequence over them, ``evict`` cuts long sequences to a budget by accumulated
attention weight.  ``Rotary`` holds the frequencies (whole heads or a part of them, half or
interleaved layout, plain or scaled for long contexts).

The contiguous caches of ``decode_model`` keep one fixed length per sequence; the reference keeps
HF's cache of one sequence (otf_llm/run_symmetric_2bit.py:150-187).
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple, Union

import torch

from . import _native

_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
MAX_NEW_TOKENS = 16

_SCALING_KEYS = {
    "default": (),
    "linear": ("factor",),
    "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"),
    "yarn": ("factor", "original_max_position_embeddings"),
}
_SCALING_OPTIONAL = {"yarn": ("attention_factor", "beta_fast", "beta_slow")}


def rope_frequencies(rot_dim: int, theta: float = 10000.0, scaling: Optional[dict] = None
                     ) -> Tuple[torch.Tensor, float]:
    """Rotary frequencies in radians per position (float64 [rot_dim / 2], on the CPU) and the factor
    on the turned values.  ``scaling``: None, or a dict as HF configurations hold it in
    ``rope_scaling``, with ``rope_type`` "default", "linear", "llama3" or "yarn" and its numbers."""
    if rot_dim < 0 or rot_dim % 2:
        raise ValueError(f"rot_dim must be even and not negative, got {rot_dim}")
    if not theta > 0:
        raise ValueError(f"theta must be positive, got {theta}")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    f = float(theta) ** (-i / max(rot_dim, 1))
    if scaling is None:
        return f, 1.0
    kind = scaling.get("rope_type", scaling.get("type"))
    if kind not in _SCALING_KEYS:
        raise ValueError(f"rope_type must be one of {sorted(_SCALING_KEYS)}, got {kind!r}")
    need, may = _SCALING_KEYS[kind], _SCALING_OPTIONAL.get(kind, ())
    missing = [k for k in need if scaling.get(k) is None]
    unknown = [k for k in scaling if k not in need + may + ("rope_type", "type", "rope_theta")]
    if missing or unknown:
        raise ValueError(f"rope_type {kind!r}: missing {missing}, not supported {unknown}")
    if scaling.get("rope_theta") not in (None, theta):
        raise ValueError(f"scaling's rope_theta is {scaling['rope_theta']}, theta {theta}")
    if kind == "default":
        return f, 1.0
    factor = float(scaling["factor"])
    if not factor > 0:
        raise ValueError(f"factor must be positive, got {factor}")
    if kind == "linear":
        return f / factor, 1.0
    context = float(scaling["original_max_position_embeddings"])
    if kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not 0 < low < high:
            raise ValueError("low_freq_factor must be positive and below high_freq_factor")
        turns = context * f / (2 * math.pi)                 # over the original context
        mix = ((turns - low) / (high - low)).clamp(0, 1)
        return f * mix + f / factor * (1 - mix), 1.0
    attention = scaling.get("attention_factor")
    if attention is None:
        attention = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0

    def place(turns: float) -> float:                       # the pair that turns so often over the context
        return rot_dim * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(theta))

    if not theta > 1 or not context > 0:
        raise ValueError("yarn needs a theta above 1 and a positive original_max_position_embeddings")
    low = max(math.floor(place(float(scaling.get("beta_fast") or 32.0))), 0)
    high = min(math.ceil(place(float(scaling.get("beta_slow") or 1.0))), rot_dim - 1)
    ramp = ((i / 2 - low) / ((high - low) if high != low else 0.001)).clamp(0, 1)
    return f * (1 - ramp) + f / factor * ramp, float(attention)


class Rotary:
    """Rotary positions of the first ``rot_dim`` values of every head (all of them by default):
    pairs (i, i + rot_dim / 2), or (2i, 2i + 1) if ``interleaved``.  See ``rope_frequencies``."""

    def __init__(self, head_dim: int, *, rot_dim: Optional[int] = None, theta: float = 10000.0,
                 scaling: Optional[dict] = None, interleaved: bool = False, device="cuda"):
        rot_dim = head_dim if rot_dim is None else int(rot_dim)
        if not 0 <= rot_dim <= head_dim:
            raise ValueError(f"rot_dim {rot_dim} outside 0..{head_dim}")
        self.head_dim, self.rot_dim, self.interleaved = int(head_dim), rot_dim, bool(interleaved)
        self.frequencies, self.factor = rope_frequencies(rot_dim, theta, scaling)
        self.turns = (self.frequencies / (2 * math.pi)).to(device)
        self.device = self.turns.device
        a = _native.RotaryArgs()
        a.turns, a.rot_dim = self.turns.data_ptr() if rot_dim else None, rot_dim
        a.factor, a.interleaved = self.factor, int(self.interleaved)
        self._args = a
        self._ref = ctypes.byref(a)


class PagedKVCache:
    """One layer's keys and values in pages.

    k_pages, v_pages: fp16 or bf16 [n_pages, page_size, kv_heads, head_dim] with the same strides
    and unit inner stride (a transposed view of [n_pages, kv_heads, page_size, head_dim] will do);
    page_table: int32 [batch, max_pages], whose row b names the pages of sequence b in order;
    lengths: int32 [batch], the tokens that each sequence has cached, negative for a place
    without a sequence (left as it is by every call).  The tensors stay the caller's and are
    changed in place: pages are handed out by writing the table, and ``advance`` counts a step's
    tokens, a prompt's too, once every layer has appended and attended them (layers may share
    table and lengths).

    Tokens and sequences that do not fit, and pages outside the pool, are left out on the device
    and raise the ``_native.device_error`` flag (see include/otf_b200.h)."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor):
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages), ("page_table", page_table), ("lengths", lengths)):
            _native._need_cuda(t, name)
            if t.device != k_pages.device:
                raise ValueError(f"{name} is on {t.device}, k_pages on {k_pages.device}")
        if k_pages.dtype not in _DTYPES or v_pages.dtype != k_pages.dtype:
            raise TypeError(f"pages must be fp16 or bf16 both, got {k_pages.dtype} and {v_pages.dtype}")
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.stride() != v_pages.stride():
            raise ValueError("k_pages and v_pages must be [n_pages, page_size, kv_heads, head_dim] with equal strides")
        n, page, heads, dim = k_pages.shape
        if dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {dim}")
        if n == 0 or page == 0 or heads == 0:
            raise ValueError(f"empty pages {tuple(k_pages.shape)}")
        stride = [s if e > 1 else dim for e, s in zip(k_pages.shape[:3], k_pages.stride()[:3])]
        if k_pages.stride(3) != 1 or any(s % 8 or s < 0 for s in stride) or k_pages.data_ptr() % 16 or \
                v_pages.data_ptr() % 16 or any(s < dim for s in stride[1:]):
            raise ValueError(f"pages need 16-byte aligned rows and a unit inner stride, got strides {k_pages.stride()}")
        if page_table.dtype != torch.int32 or lengths.dtype != torch.int32:
            raise TypeError("page_table and lengths must be int32")
        if page_table.dim() != 2 or page_table.shape[1] == 0 or page_table.stride(1) != 1:
            raise ValueError("page_table must be a row-major [batch, max_pages] tensor")
        if lengths.shape != page_table.shape[:1] or lengths.shape[0] == 0 or not lengths.is_contiguous():
            raise ValueError(f"lengths must be a contiguous [{page_table.shape[0]}] vector")
        self._k_pages, self._v_pages, self._page_table, self._lengths = k_pages, v_pages, page_table, lengths
        self.device, self.dtype = k_pages.device, k_pages.dtype
        self.page_size, self.kv_heads, self.head_dim = page, heads, dim
        self.batch, self.max_pages = page_table.shape
        self.capacity = self.max_pages * page
        self._scale = dim ** -0.5
        c = _native.PagedCache()
        c.k_pages, c.v_pages = k_pages.data_ptr(), v_pages.data_ptr()
        c.page_stride, c.token_stride, c.head_stride = stride
        c.n_pages, c.page_size, c.kv_heads, c.head_dim = n, page, heads, dim
        c.page_table, c.max_pages = page_table.data_ptr(), self.max_pages
        c.ld_table = page_table.stride(0) if self.batch > 1 else max(page_table.stride(0), self.max_pages)
        c.lengths, c.batch, c.dtype = lengths.data_ptr(), self.batch, _DTYPES[self.dtype]
        self._args = c
        self._ref = ctypes.byref(c)
        # shapes and strides of earlier calls' arguments, with what their checks found: a decode
        # loop's calls differ in addresses alone
        self._append_plans: dict = {}
        self._attend_plans: dict = {}

    # the tensors are changed in place, never replaced: the native side holds their addresses
    @property
    def k_pages(self) -> torch.Tensor:
        return self._k_pages

    @property
    def v_pages(self) -> torch.Tensor:
        return self._v_pages

    @property
    def page_table(self) -> torch.Tensor:
        return self._page_table

    @property
    def lengths(self) -> torch.Tensor:
        return self._lengths

    @classmethod
    def allocate(cls, n_pages: int, page_size: int, kv_heads: int, head_dim: int, page_table: torch.Tensor,
                 lengths: torch.Tensor, dtype: torch.dtype = torch.float16) -> "PagedKVCache":
        """A cache of new zeroed pages [n_pages, page_size, kv_heads, head_dim] under the given table."""
        k, v = (torch.zeros(n_pages, page_size, kv_heads, head_dim, dtype=dtype, device=page_table.device)
                for _ in range(2))
        return cls(k, v, page_table, lengths)

    def _heads(self, t: torch.Tensor, name: str, heads: Optional[int] = None) -> int:
        """Check the shape and strides of [rows, heads, head_dim] values whose heads lie next to one
        another; the row stride."""
        d = self.head_dim
        if t.dim() != 3 or t.shape[2] != d or (heads is not None and t.shape[1] != heads) or t.shape[1] == 0:
            raise ValueError(f"{name} must be [rows, {heads or 'heads'}, {d}], got {tuple(t.shape)}")
        row, head, one = t.stride()
        if one != 1 or (head != d and t.shape[1] > 1):
            raise ValueError(f"{name} needs its heads next to one another, got strides {t.stride()}")
        if t.shape[0] <= 1:
            row = t.shape[1] * d
        if row % 8 or row < t.shape[1] * d:
            raise ValueError(f"{name} needs 16-byte aligned rows that do not overlap, got strides {t.stride()}")
        return row

    def _refuse(self, **given: torch.Tensor) -> None:
        for name, t in given.items():
            if t.dtype is not self.dtype or t.device != self.device or t.data_ptr() & 15:
                raise ValueError(f"{name} must be 16-byte aligned {self.dtype} on {self.device}, got {t.dtype} on "
                                 f"{t.device}")

    def _output(self, out: torch.Tensor, name: str, like: torch.Tensor) -> Tuple[int, int]:
        """The row stride and address of an output of like's shape."""
        if out.shape != like.shape:
            raise ValueError(f"{name} must have q's shape {tuple(like.shape)}, got {tuple(out.shape)}")
        self._refuse(**{name: out})
        rows = self._flat(out, name)
        return self._heads(rows, name, rows.shape[1]), out.data_ptr()

    def _vector(self, t: torch.Tensor, name: str, n: int) -> int:
        if t.device != self.device or t.dtype != torch.int32 or t.shape != (n,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 [{n}] vector on {self.device}")
        return t.data_ptr()

    def append(self, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, rotary: Optional[Rotary] = None, *,
               starts: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None
               ) -> Optional[torch.Tensor]:
        """New tokens enter the cache (otf_paged_append).

        q [n, heads, head_dim] (or None), k and v [n, kv_heads, head_dim]: rows of new tokens, e.g.
        parts of a fused projection's output.  Sequence b has the rows starts[b] .. starts[b + 1] - 1
        (int32 [batch + 1] on the device), or n / batch each; its t-th becomes token lengths[b] + t,
        and turns by that position, or by positions[row] (int32 [n]) where places and positions
        differ (after ``evict``).  Returns the turned queries, in ``q_out`` (which may be q, and else shares no
        memory with q, k and v) or a new tensor.  Rows behind the last sequence are left as they were, as are those of a negative
        length.  ``lengths`` is not advanced.

        ``weights``, as ``attend`` adds them up: the new tokens' entries are set to 0.  Give them wherever
        earlier tokens may have held these places: drafted ones that were refused, or those of the
        sequence before in this place of the batch."""
        key = (None if q is None else (q.shape, q.stride()), k.shape, k.stride(), v.shape, v.stride())
        plan = self._append_plans.get(key)
        if plan is None:
            plan = self._remember(self._append_plans, key, self._plan_append(q, k, v))
        n, heads, ldq, ldk, ldv = plan
        dtype, dev = self.dtype, self.device
        pk, pv = k.data_ptr(), v.data_ptr()
        if k.dtype is not dtype or v.dtype is not dtype or k.device != dev or v.device != dev or (pk | pv) & 15:
            self._refuse(k=k, v=v)
        pq = po = ps = pp = None
        ldo = 0
        if q is not None:
            pq = q.data_ptr()
            if q.dtype is not dtype or q.device != dev or pq & 15:
                self._refuse(q=q)
            if q_out is None:
                q_out = torch.empty_like(q)         # heads next to one another, rows without gaps
                ldo, po = heads * self.head_dim, q_out.data_ptr()
            else:
                ldo, po = self._output(q_out, "q_out", q)
        elif q_out is not None:
            raise ValueError("q_out without q")
        if starts is not None:
            ps = self._vector(starts, "starts", self.batch + 1)
        elif n % self.batch:
            raise ValueError(f"{n} rows do not divide among {self.batch} sequences; give starts")
        if positions is not None:
            pp = self._vector(positions, "positions", n)
        if rotary is not None and (rotary.head_dim != self.head_dim or rotary.device != self.device):
            raise ValueError(f"rotary is for heads of {rotary.head_dim} on {rotary.device}")
        if weights is not None:
            ldw = self._weights(weights, "weights", self.capacity)
            if n:
                _call(_native.lib().otf_paged_append_weights, dev, self._ref, None if rotary is None else rotary._ref, pq, ldq,
                      po, ldo, heads, pk, ldk, pv, ldv, ps, pp, n, weights.data_ptr(), ldw)
        elif n:
            _call(_native.lib().otf_paged_append, dev, self._ref, None if rotary is None else rotary._ref, pq, ldq, po,
                  ldo, heads, pk, ldk, pv, ldv, ps, pp, n)
        return q_out

    def _plan_append(self, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor) -> tuple:
        ldk, ldv = self._heads(k, "k", self.kv_heads), self._heads(v, "v", self.kv_heads)
        n, heads, ldq = k.shape[0], 0, 0
        if q is not None:
            ldq, heads = self._heads(q, "q"), q.shape[1]
        for name, t in (("v", v), ("q", q)):
            if t is not None and t.shape[0] != n:
                raise ValueError(f"{name} has {t.shape[0]} rows, k {n}")
        return n, heads, ldq, ldk, ldv

    @staticmethod
    def _remember(plans: dict, key: tuple, plan: tuple) -> tuple:
        if len(plans) >= 256:                               # prompts come in many lengths
            plans.clear()
        plans[key] = plan
        return plan

    def attend(self, q: torch.Tensor, *, scale: Optional[float] = None, weights: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of the newest tokens over the cache (otf_paged_attn).

        q: [batch, heads, head_dim], or [batch, tokens, heads, head_dim] with the 1 to 16 newest
        tokens of every sequence (all of them appended, ``lengths`` not yet advanced): row t of
        sequence b sees the tokens 0 .. lengths[b] + t.  ``scale`` defaults to head_dim ** -0.5.
        ``weights`` (fp32 [batch, kv_heads, at least capacity], contiguous): to every token's entry
        is added the softmax weight that it received from the rows and the query heads of that KV
        head (rows of drafted tokens that are refused afterwards have added theirs).  Scratch for them grows with the table's room, not the lengths: 4 bytes x batch x heads x
        tokens x capacity, at most 2 GiB at a time (the call then takes several passes).  A cache made
        over fewer columns of a large table, ``page_table[:, :n]``, needs and walks less.  Returns ``out``,
        of q's shape, which shares no memory with q (rows of negative lengths are left as they were)."""
        key = (q.shape, q.stride(), weights is None)
        plan = self._attend_plans.get(key)
        if plan is None:
            plan = self._remember(self._attend_plans, key, self._plan_attend(q, weights))
        tokens, heads, ldq, bytes_ = plan
        pq, dev = q.data_ptr(), self.device
        if q.dtype is not self.dtype or q.device != dev or pq & 15:
            self._refuse(q=q)
        if out is None:
            out = torch.empty_like(q)
            ldo, po = heads * self.head_dim, out.data_ptr()
        else:
            ldo, po = self._output(out, "out", q)
            if po == pq:
                raise ValueError("out must not be q")
        pw, ldw = None, 0
        if weights is not None:
            ldw = self._weights(weights, "weights", self.capacity)
            pw = weights.data_ptr()
        # from the caching allocator, for this call alone: calls on two streams, or in two captured
        # graphs, share nothing
        ws = torch.empty(bytes_, dtype=torch.uint8, device=dev)
        _call(_native.lib().otf_paged_attn, dev, self._ref, pq, ldq, heads, tokens,
              self._scale if scale is None else float(scale), po, ldo, pw, ldw, ws.data_ptr(), bytes_)
        return out

    def _plan_attend(self, q: torch.Tensor, weights: Optional[torch.Tensor]) -> tuple:
        if q.dim() not in (3, 4):
            raise ValueError(f"q must have 3 or 4 dimensions, got {tuple(q.shape)}")
        tokens = q.shape[1] if q.dim() == 4 else 1
        if q.shape[0] != self.batch or not 1 <= tokens <= MAX_NEW_TOKENS:
            raise ValueError(f"q must hold 1 to {MAX_NEW_TOKENS} tokens of {self.batch} sequences, got {tuple(q.shape)}")
        rows = self._flat(q, "q")
        ldq, heads = self._heads(rows, "q"), rows.shape[1]
        if heads % self.kv_heads:
            raise ValueError(f"{heads} query heads over {self.kv_heads} KV heads")
        n = _native.lib().otf_paged_attn_workspace_bytes(self.batch, heads, self.kv_heads, self.head_dim, tokens,
                                                         self.capacity, 0 if weights is None else 1)
        if n < 0:
            raise ValueError("shape not supported by otf_paged_attn")
        return tokens, heads, ldq, n

    def evict(self, weights: torch.Tensor, budget: int, recent: int, *, to: Optional["PagedKVCache"] = None,
              weights_out: Optional[torch.Tensor] = None, lengths_out: Optional[torch.Tensor] = None
              ) -> torch.Tensor:
        """Cut every sequence longer than ``budget`` tokens to it (otf_paged_evict), for each KV head
        by itself: the ``recent`` last tokens stay, and of the others those of the largest
        ``weights`` (as ``attend`` adds them up; ties: the earlier token), in their order.

        In place by default: pages (of one sequence each), ``weights`` and ``lengths`` of this cache are
        cut, and a sequence's pages behind its first budget / page_size (rounded up) may be handed on.  With
        ``to``, a cache of the same geometry whose table names other pages, the kept tokens go there
        (its ``lengths`` are set, and ``weights_out``, fp32 [batch, kv_heads, at least budget], is
        written), and this one stays as it is.

        ``lengths_out`` (int32 [batch]) takes the new lengths instead of the cut cache's ``lengths``:
        layers that share one lengths vector give another one for all but the last.  Returns int32
        [batch, kv_heads, budget]: the places that were kept, then -1."""
        ldw = self._weights(weights, "weights", self.capacity)
        budget, recent = int(budget), int(recent)
        if to is None:
            if weights_out is not None:
                raise ValueError("weights_out without to: in place, weights are cut themselves")
            to, weights_out = self, weights
        elif weights_out is None:
            raise ValueError("weights_out is needed with to")
        elif weights_out.data_ptr() == weights.data_ptr() or to.lengths.data_ptr() == self.lengths.data_ptr() or \
                to.page_table.data_ptr() == self.page_table.data_ptr():
            raise ValueError("to's table, lengths and weights must not be this cache's (leave to out to cut in place)")
        if (to.batch, to.kv_heads, to.head_dim, to.page_size, to.dtype, to.device) != \
                (self.batch, self.kv_heads, self.head_dim, self.page_size, self.dtype, self.device):
            raise ValueError("to must have this cache's batch, heads, page size, type and device")
        if not 0 < budget <= to.capacity or not 0 <= recent <= budget:
            raise ValueError(f"budget {budget} (of {to.capacity}) and recent {recent} do not fit")
        ldo = self._weights(weights_out, "weights_out", budget)
        if lengths_out is None:
            lengths_out = to.lengths
        elif to is not self and lengths_out.data_ptr() == self.lengths.data_ptr():
            raise ValueError("lengths_out must not be the source's lengths with to")
        kept = torch.empty((self.batch, self.kv_heads, budget), dtype=torch.int32, device=self.device)
        _call(_native.lib().otf_paged_evict, self.device, self._ref, to._ref, weights.data_ptr(), ldw, weights_out.data_ptr(), ldo,
              budget, recent, kept.data_ptr(), self._vector(lengths_out, "lengths_out", self.batch))
        return kept

    def advance(self, tokens: Union[int, torch.Tensor] = 1) -> None:
        """lengths += tokens, where there is a sequence: a number, or int32 [batch] on the device where the
        sequences differ (``starts.diff()`` after prompts, ``accepted + 1`` after a pass over drafts)."""
        there = self.lengths.ge(0).to(torch.int32)
        if isinstance(tokens, torch.Tensor):
            self._vector(tokens, "tokens", self.batch)
            self.lengths.add_(there.mul_(tokens))
        else:
            self.lengths.add_(there, alpha=int(tokens))

    def _weights(self, t: torch.Tensor, name: str, least: int) -> int:
        if t.device != self.device or t.dtype != torch.float32 or t.dim() != 3 or not t.is_contiguous() or \
                t.shape[:2] != (self.batch, self.kv_heads) or t.shape[2] < least:
            raise ValueError(f"{name} must be contiguous fp32 [{self.batch}, {self.kv_heads}, at least {least}] on "
                             f"{self.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
        return t.shape[2]

    @staticmethod
    def _flat(t: torch.Tensor, name: str) -> torch.Tensor:
        """[batch, tokens, heads, dim] as rows, without a copy."""
        if t.dim() == 3:
            return t
        if t.shape[0] > 1 and t.shape[1] > 1 and t.stride(0) != t.shape[1] * t.stride(1):
            raise ValueError(f"{name} needs evenly strided rows, got strides {t.stride()}")
        row = t.stride(1) if t.shape[1] > 1 else t.stride(0)
        return t.as_strided((t.shape[0] * t.shape[1], t.shape[2], t.shape[3]), (row, t.stride(2), t.stride(3)))


def _call(fn, dev: torch.device, *args) -> None:
    """An entry point of the library with the device current and its current stream as the last
    argument (the raw handle: torch.cuda.current_stream would make a Stream object)."""
    index = dev.index
    if torch.cuda.current_device() == index:
        st = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            st = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if st:
        _native._check(st, fn.__name__)
