"""The paged key/value cache's operators, as they are measured.

Four operators, each as a user's program calls it and in a plain form of elementary torch operations:

* append: rotary positions on new queries and keys, keys and values written into the cache's pages;
* attend: one or a few new tokens per sequence attend over the pages (optionally adding up the
  attention weight that every cached token receives);
* evict: the cache shortened to a budget, by recency and accumulated attention weight;
* verify: drafted tokens accepted or refused against the target model's distribution.

Sizes: Llama-shaped heads of this framework's configurations (32 and 64 query heads over 8 KV heads
of 128, 32 over 32), small ones of the tests (heads of 64), vocabularies of 32000 and 128256.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the cache write of one decoded token, a single user's session: latency
        {"name": "append one token", "op": "append", "batch": 1, "tokens": 1, "ragged": False, "len": 1023, "heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "scaling": "none", "type": "fp16", "page": 16,
         "order": "token"},
        # a decode step of a full serving batch, rotary on half of each head, interleaved, YaRN-scaled
        {"name": "append a batch's step", "op": "append", "batch": 64, "tokens": 1, "ragged": False, "len": 6000,
         "heads": 64, "kv_heads": 8, "dim": 128, "rot": 64, "interleaved": True, "scaling": "yarn", "type": "bf16",
         "page": 32, "order": "head"},
        # prompts of different lengths entering the cache together, frequencies scaled for long contexts
        {"name": "append prompts", "op": "append", "batch": 11, "tokens": 2500, "ragged": True, "len": 3000, "heads": 64,
         "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "scaling": "llama3", "type": "fp16", "page": 16,
         "order": "token"},
        # one decoded token of a short conversation: latency
        {"name": "attend one short", "op": "attend", "batch": 1, "len": 700, "tokens": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "type": "fp16", "page": 16, "order": "token", "weights": False},
        # one decoded token over a very long document: the split over the cache's length decides
        {"name": "attend one long", "op": "attend", "batch": 1, "len": 131071, "tokens": 1, "heads": 64, "kv_heads": 8,
         "dim": 128, "type": "fp16", "page": 64, "order": "head", "weights": False},
        # a decode step of a full serving batch with very different lengths
        {"name": "attend a ragged batch", "op": "attend", "batch": 64, "len": 8190, "tokens": 1, "heads": 64,
         "kv_heads": 8, "dim": 128, "type": "bf16", "page": 16, "order": "token", "weights": False},
        # the target model's pass over four drafted tokens and the one before them, weights kept for eviction
        {"name": "attend drafts, weights", "op": "attend", "batch": 16, "len": 4001, "tokens": 5, "heads": 32,
         "kv_heads": 8, "dim": 128, "type": "fp16", "page": 20, "order": "token", "weights": True},
        # a batch of long conversations cut to a budget
        {"name": "evict a batch", "op": "evict", "batch": 16, "len": 8191, "budget": 2048, "recent": 256, "kv_heads": 8,
         "dim": 128, "type": "fp16", "page": 16, "order": "token"},
        # one very long document cut to a sixteenth
        {"name": "evict one long", "op": "evict", "batch": 1, "len": 65536, "budget": 4096, "recent": 1024, "kv_heads": 8,
         "dim": 128, "type": "bf16", "page": 64, "order": "head"},
        # drafts looked up from the prompt (no draft model): one sequence, a small vocabulary
        {"name": "verify looked-up drafts", "op": "verify", "batch": 1, "drafts": 4, "vocab": 32000, "drafted": False,
         "temperature": 1.0, "ragged": False},
        # a serving batch's drafts from a draft model
        {"name": "verify a batch", "op": "verify", "batch": 64, "drafts": 5, "vocab": 128256, "drafted": True,
         "temperature": 0.8, "ragged": True},
        # greedy decoding's drafts
        {"name": "verify greedily", "op": "verify", "batch": 16, "drafts": 7, "vocab": 128256, "drafted": False,
         "temperature": 0.0, "ragged": False},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("append", "attend", "evict", "verify"))
    if op == "verify":
        batch, drafts, vocab = _log(rng, 1, 64), rng.randint(0, 8), _log(rng, 1000, 131072)
        while batch * (drafts + 1) * vocab > 64 * 6 * 128256:
            batch = max(1, batch // 2)
        return {"op": op, "batch": batch, "drafts": drafts, "vocab": vocab, "drafted": rng.random() < 0.6,
                "temperature": rng.choice((0.0, 0.6, 0.8, 1.0, 1.3)), "ragged": rng.random() < 0.5}
    kv_heads, group = rng.choice(((8, 4), (8, 8), (32, 1), (1, 8), (2, 7), (4, 5), (8, 2)))
    dim = rng.choice((64, 128, 128))
    case = {"op": op, "batch": _log(rng, 1, 64), "kv_heads": kv_heads, "dim": dim, "type": rng.choice(("fp16", "bf16")),
            "page": rng.choice((8, 16, 16, 20, 32, 64, 128)), "order": rng.choice(("token", "head"))}
    row = kv_heads * dim
    if op == "append":
        tokens = rng.choice((1, rng.randint(2, 8), _log(rng, 9, 4000)))
        case.update(tokens=tokens, ragged=tokens > 1 and rng.random() < 0.7, len=_log(rng, 1, 8000), heads=kv_heads * group,
                    rot=rng.choice((dim, dim, dim // 2, 24)), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(("none", "linear", "llama3", "yarn")))
        while case["batch"] * tokens * (case["heads"] + 2 * kv_heads) * dim > 13000 * 80 * 128 or \
                case["batch"] * (case["len"] + tokens) * row > 11 * 5500 * 1024:
            case["batch"], case["len"] = max(1, case["batch"] // 2), max(1, case["len"] * 3 // 4)
        return case
    case["len"] = _log(rng, 1, 131072) if op == "attend" else _log(rng, 64, 65536)
    while case["batch"] * case["len"] * row > 64 * 4096 * 1024 // (1 if op == "attend" else 2):
        case["batch"], case["len"] = max(1, case["batch"] // 2), max(64, case["len"] * 3 // 4)
    if op == "attend":
        case.update(tokens=rng.choice((1, 1, 1, rng.randint(2, 8))), heads=kv_heads * group, weights=rng.random() < 0.3)
        case["len"] = max(case["len"], case["tokens"])
    else:
        case["budget"] = rng.randint(max(2, case["len"] // 16), max(3, case["len"] * 3 // 4))
        case["recent"] = rng.randint(0, case["budget"] // 2)
    return case


# ---- shapes that a case fixes (the seed only permutes them) -------------------------------------


def _spread(n, low, high):
    """n whole numbers from high down to low, evenly."""
    return [high - (high - low) * i // max(1, n - 1) for i in range(n)]


def _totals(case):
    """How many tokens each sequence's cache holds in the end (append: before the new ones)."""
    low = case.get("tokens", 1) if case["op"] == "attend" else 1 if case["op"] == "evict" else 0
    return _spread(case["batch"], max(low, case["len"] // 64), case["len"])


def _new(case):
    return _spread(case["batch"], max(1, case["tokens"] // 10), case["tokens"]) if case["ragged"] else \
        [case["tokens"]] * case["batch"]


def _shuffled(values, gen):
    order = torch.randperm(len(values), generator=gen).tolist()
    return [values[i] for i in order]


def _frequencies(case):
    """Rotary frequencies per position, in 64 bits, and the factor on the rotated values."""
    n, theta, factor, original = case["rot"], 500000.0, 8.0, 8192.0
    i = torch.arange(0, n // 2, dtype=torch.float64)
    f = theta ** (-2 * i / n)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "llama3":
        wave = 2 * math.pi / f
        smooth = (original / wave - 1.0) / (4.0 - 1.0)
        mixed = (1 - smooth) * f / factor + smooth * f
        return torch.where(wave > original / 1.0, f / factor, torch.where(wave < original / 4.0, f, mixed)), 1.0
    if case["scaling"] == "yarn":
        at = [n * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), n - 1)
        ramp = ((i - low) / ((high - low) or 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


SCALING = {
    "none": None,
    "linear": {"rope_type": "linear", "factor": 8.0},
    "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position_embeddings": 8192},
    "yarn": {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 8192},
}


# ---- what a program has in hand -----------------------------------------------------------------


def _pool(case, batch, room, gen, fill):
    """Pages for `batch` sequences of up to `room` tokens, handed out in a random order."""
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    each = -(-room // page)
    n = batch * each + 3
    shape = (n, page, heads, dim) if case["order"] == "token" else (n, heads, page, dim)
    pages = []
    for _ in range(2):
        t = torch.empty(shape, dtype=TYPES[case["type"]], device=DEVICE)
        t.normal_(generator=gen) if fill else t.zero_()
        pages.append(t if case["order"] == "token" else t.transpose(1, 2))
    table = torch.randperm(n, generator=gen, device=DEVICE)[:batch * each].to(torch.int32).view(batch, each)
    return pages[0], pages[1], table.contiguous()


def _cache(k, v, table, lengths):
    where = os.path.join(ROOT, "otf-llm-engine_b200")
    if where not in sys.path:
        sys.path.insert(0, where)
    from otf_llm.paged import PagedKVCache
    return PagedKVCache(k, v, table, lengths)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    cpu = torch.Generator().manual_seed(int(seed))
    st = {"case": case}
    if case["op"] == "verify":
        return _prepare_verify(case, st, gen, cpu)
    dtype, batch = TYPES[case["type"]], case["batch"]
    totals = _shuffled(_totals(case), cpu)
    if case["op"] == "append":
        new = _shuffled(_new(case), cpu)
        st["n"] = n = sum(new)
        st["starts"] = torch.tensor([0] + new, device=DEVICE).cumsum(0).to(torch.int32)
        qkv = torch.randn(n, (case["heads"] + 2 * case["kv_heads"]) * case["dim"], generator=gen, device=DEVICE).to(dtype)
        # the three parts of one fused projection's rows
        q, k, v = qkv.view(n, -1, case["dim"]).split([case["heads"], case["kv_heads"], case["kv_heads"]], dim=1)
        st.update(q=q, k=k, v=v)
        st["f"], st["factor"] = _frequencies(case)
        st["f"] = st["f"].to(DEVICE)
        room = max(totals) + max(new)
        st["kp"], st["vp"], st["table"] = _pool(case, batch, room, gen, True)
        st["lengths"] = torch.tensor(totals, dtype=torch.int32, device=DEVICE)
    elif case["op"] == "attend":
        st["kp"], st["vp"], st["table"] = _pool(case, batch, case["len"], gen, True)
        st["lengths"] = torch.tensor([t - case["tokens"] for t in totals], dtype=torch.int32, device=DEVICE)
        st["q"] = torch.randn(batch, case["tokens"], case["heads"], case["dim"], generator=gen, device=DEVICE).to(dtype)
        if case["weights"]:
            st["weights"] = torch.rand(batch, case["kv_heads"], st["table"].shape[1] * case["page"], generator=gen,
                                       device=DEVICE)
    else:
        st["kp"], st["vp"], st["table"] = _pool(case, batch, case["len"], gen, True)
        st["lengths"] = torch.tensor(totals, dtype=torch.int32, device=DEVICE)
        w = torch.rand(batch, case["kv_heads"], st["table"].shape[1] * case["page"], generator=gen, device=DEVICE)
        st["weights"] = torch.where(w < 0.1, 0.0, w ** 6 * 20)       # a few heavy tokens, some never looked at
        st["kp_to"], st["vp_to"], st["table_to"] = _pool(case, batch, case["budget"] + 64, gen, False)
        st["lengths_to"] = torch.zeros(batch, dtype=torch.int32, device=DEVICE)
        st["weights_to"] = torch.zeros(batch, case["kv_heads"], st["table_to"].shape[1] * case["page"], device=DEVICE)
    if own:
        st["cache"] = _cache(st["kp"], st["vp"], st["table"], st["lengths"])
        if case["op"] == "append":
            from otf_llm.paged import Rotary
            st["rotary"] = Rotary(case["dim"], rot_dim=case["rot"], theta=500000.0, scaling=SCALING[case["scaling"]],
                                  interleaved=case["interleaved"], device=DEVICE)
        if case["op"] == "evict":
            st["to"] = _cache(st["kp_to"], st["vp_to"], st["table_to"], st["lengths_to"])
    return st


def _prepare_verify(case, st, gen, cpu):
    batch, drafts, vocab = case["batch"], case["drafts"], case["vocab"]
    target = torch.randn(batch, drafts + 1, vocab, generator=gen, device=DEVICE) * 2.5
    # a few likely continuations in every place, as a language model has them
    heads = torch.randint(0, vocab, (batch, drafts + 1, 8), generator=gen, device=DEVICE)
    target.scatter_add_(2, heads, torch.rand(batch, drafts + 1, 8, generator=gen, device=DEVICE) * 6 + 6)
    st["target"] = target
    if case["drafted"]:
        st["draft"] = target[:, :drafts] + 0.7 * torch.randn(batch, drafts, vocab, generator=gen, device=DEVICE)
        race = torch.empty_like(st["draft"]).exponential_(generator=gen).log_().neg_()
        st["tokens"] = (st["draft"] / max(case["temperature"], 0.05) + race).argmax(2)
        del race
    else:
        other = torch.randint(0, vocab, (batch, drafts), generator=gen, device=DEVICE)
        keep = torch.rand(batch, drafts, generator=gen, device=DEVICE) < 0.8
        st["tokens"] = torch.where(keep, target[:, :drafts].argmax(2), other)
    st["uniforms"] = torch.rand(batch, drafts, generator=gen, device=DEVICE)
    st["noise"] = torch.empty(batch, vocab, device=DEVICE).exponential_(generator=gen)
    if case["ragged"]:
        counts = _shuffled(_spread(batch, 0, drafts), cpu)
        st["counts"] = torch.tensor(counts, dtype=torch.int32, device=DEVICE)
    if own:
        where = os.path.join(ROOT, "otf-llm-engine_b200")
        if where not in sys.path:
            sys.path.insert(0, where)
    return st


# ---- one pass -----------------------------------------------------------------------------------


def run(st):
    return {"append": _append, "attend": _attend, "evict": _evict, "verify": _verify}[st["case"]["op"]](st)


def _append(st):
    case = st["case"]
    if own:
        q = st["cache"].append(st["q"], st["k"], st["v"], st["rotary"], starts=st["starts"])
        return [q, st["kp"], st["vp"]]
    row = torch.arange(st["n"], device=DEVICE)
    seq = torch.bucketize(row, st["starts"][1:].long(), right=True)
    slot = st["lengths"].long()[seq] + row - st["starts"].long()[seq]
    angle = slot.double()[:, None] * st["f"]
    cos, sin = (angle.cos() * st["factor"]).float()[:, None], (angle.sin() * st["factor"]).float()[:, None]
    turned, half = [], case["rot"] // 2
    for x in (st["q"], st["k"]):
        x = x.float()
        lead = x[..., :case["rot"]]
        a, b = (lead[..., 0::2], lead[..., 1::2]) if case["interleaved"] else (lead[..., :half], lead[..., half:])
        parts = a * cos - b * sin, b * cos + a * sin
        lead = torch.stack(parts, -1).flatten(-2) if case["interleaved"] else torch.cat(parts, -1)
        turned.append(torch.cat([lead, x[..., case["rot"]:]], -1).to(st["q"].dtype))
    page, at = st["table"].long()[seq, slot // case["page"]], slot % case["page"]
    st["kp"][page, at] = turned[1]
    st["vp"][page, at] = st["v"]
    return [turned[0], st["kp"], st["vp"]]


def _attend(st):
    case = st["case"]
    if own:
        out = st["cache"].attend(st["q"], weights=st.get("weights"))
        return [out, st["weights"]] if case["weights"] else [out]
    batch, new, kv, dim = case["batch"], case["tokens"], case["kv_heads"], case["dim"]
    table = st["table"].long()
    k = st["kp"][table].float().reshape(batch, -1, kv, dim).permute(0, 2, 3, 1)          # [batch, kv, dim, place]
    group = case["heads"] // kv
    q = st["q"].float().view(batch, new, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, kv, new * group, dim)
    s = torch.matmul(q, k).view(batch, kv, new, group, -1) / math.sqrt(dim)
    del k
    place = torch.arange(s.shape[-1], device=DEVICE)
    seen = place <= st["lengths"].long()[:, None, None] + torch.arange(new, device=DEVICE)[:, None]
    s = s.masked_fill(~seen[:, None, :, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    v = st["vp"][table].float().reshape(batch, -1, kv, dim).transpose(1, 2)
    out = torch.matmul(p.view(batch, kv, new * group, -1), v).view(batch, kv, new, group, dim)
    out = out.permute(0, 2, 1, 3, 4).reshape(batch, new, case["heads"], dim).to(st["q"].dtype)
    if not case["weights"]:
        return [out]
    st["weights"] += p.sum((2, 3))
    return [out, st["weights"]]


def _evict(st):
    case = st["case"]
    budget, recent, kv = case["budget"], case["recent"], case["kv_heads"]
    if own:
        kept = st["cache"].evict(st["weights"], budget, recent, to=st["to"], weights_out=st["weights_to"])
        return [kept, st["kp_to"], st["vp_to"], st["weights_to"], st["lengths_to"]]
    w, length = st["weights"], st["lengths"].long()[:, None, None]
    place = torch.arange(w.shape[2], device=DEVICE)
    key = torch.where(place >= length - recent, math.inf, w)
    key = torch.where(place >= length, -math.inf, key)
    order = key.sort(dim=2, descending=True, stable=True).indices[..., :budget]
    if order.shape[2] < budget:
        order = torch.nn.functional.pad(order, (0, budget - order.shape[2]), value=w.shape[2])
    left = length.clamp(max=budget)
    rank = torch.arange(budget, device=DEVICE)
    there = rank < left
    kept = torch.where(there, order, w.shape[2]).sort(dim=2).values
    safe = torch.where(there, kept, 0)
    row, head = torch.arange(case["batch"], device=DEVICE)[:, None, None], torch.arange(kv, device=DEVICE)[:, None]
    page_to, at_to = st["table_to"].long()[row, rank // case["page"]], (rank % case["page"]).expand_as(safe)
    page, at = st["table"].long()[row, safe // case["page"]], safe % case["page"]
    page_to, head = page_to.expand_as(safe), head.expand_as(safe)
    for src, dst in ((st["kp"], st["kp_to"]), (st["vp"], st["vp_to"])):
        dst[page_to, at_to, head] = torch.where(there[..., None], src[page, at, head], dst[page_to, at_to, head])
    st["weights_to"].zero_()
    st["weights_to"][..., :budget] = torch.where(there, w.gather(2, safe), 0.0)
    st["lengths_to"].copy_(left.view(-1))
    return [torch.where(there, kept, -1).to(torch.int32), st["kp_to"], st["vp_to"], st["weights_to"], st["lengths_to"]]


def _softmax64(x, temperature):
    x = x.double()
    e = ((x - x.amax(-1, keepdim=True)) / temperature).exp()
    return e / e.sum(-1, keepdim=True)


def _verify(st):
    case = st["case"]
    if own:
        from otf_llm.speculative import verify_drafts
        return list(verify_drafts(st["target"], st["tokens"], draft_logits=st.get("draft"), uniforms=st["uniforms"],
                                  noise=st["noise"], temperature=case["temperature"], counts=st.get("counts")))
    batch, drafts = case["batch"], case["drafts"]
    counts = st["counts"].long() if case["ragged"] else torch.full((batch,), drafts, device=DEVICE)
    step, row = torch.arange(drafts, device=DEVICE), torch.arange(batch, device=DEVICE)
    if case["temperature"] == 0.0:
        best = st["target"].argmax(2)
        took = st["tokens"] == best[:, :drafts]
    else:
        p = _softmax64(st["target"], case["temperature"])
        p_at = p[:, :drafts].gather(2, st["tokens"][..., None])[..., 0]
        if case["drafted"]:
            q_at = _softmax64(st["draft"], case["temperature"]).gather(2, st["tokens"][..., None])[..., 0]
        else:
            q_at = torch.ones_like(p_at)
        took = st["uniforms"].double() * q_at < p_at
    took = took & (step < counts[:, None])
    accepted = took.long().cumprod(1).sum(1)
    if case["temperature"] == 0.0:
        last = best[row, accepted]
    else:
        p = p[row, accepted]
        w = p
        if drafts:
            at = accepted.clamp(max=drafts - 1)
            refused = (accepted < counts)[:, None]
            if case["drafted"]:
                q = _softmax64(st["draft"][row, at], case["temperature"])
            else:
                q = torch.arange(case["vocab"], device=DEVICE) == st["tokens"][row, at][:, None]
                q = q.double() * 2
            left = torch.where(refused, (p - q).clamp(min=0), p)
            w = torch.where(left.sum(1, keepdim=True) > 0, left, p)
        last = (w / st["noise"].double()).argmax(1)
    place = torch.arange(drafts + 1, device=DEVICE)
    tokens = torch.cat([st["tokens"], last[:, None]], 1)
    tokens = torch.where(place < accepted[:, None], tokens, torch.where(place == accepted[:, None], last[:, None], -1))
    return [tokens, accepted.to(torch.int32)]


# ---- what a pass cannot do without ---------------------------------------------------------------


def work(case):
    if case["op"] == "verify":
        counts = _spread(case["batch"], 0, case["drafts"]) if case["ragged"] else [case["drafts"]] * case["batch"]
        rows = sum(counts) + case["batch"]
        flops = rows * case["vocab"] * 2
        if case["temperature"] > 0:
            rows += case["batch"] + (sum(counts) if case["drafted"] else 0)      # the noise, and the draft's logits
            flops = rows * case["vocab"] * 4
        return {"bytes": rows * case["vocab"] * 4 + case["batch"] * (2 * case["drafts"] + 1) * 8, "flops": flops}
    row = case["kv_heads"] * case["dim"]
    if case["op"] == "append":
        values = sum(_new(case)) * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": values * 4, "flops": values * 3}
    totals = _totals(case)
    if case["op"] == "attend":
        cached, queries = sum(totals), case["batch"] * case["tokens"] * case["heads"] * case["dim"]
        read = cached * row * 4 + queries * 4 + (cached * case["kv_heads"] * 8 if case["weights"] else 0)
        return {"bytes": read, "flops": 4 * cached * case["heads"] * case["tokens"] * case["dim"]}
    left = sum(min(t, case["budget"]) for t in totals)
    return {"bytes": sum(totals) * case["kv_heads"] * 4 + left * (row * 8 + case["kv_heads"] * 8),
            "flops": sum(totals) * case["kv_heads"] * 4}


# ---- the definitions in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    if case["op"] == "verify":
        return None                                     # whole numbers alone
    st = _inputs_alone(case, seed)
    page, lengths = case["page"], st["lengths"].tolist()
    if case["op"] == "append":
        return _exact_append(case, st, lengths)
    if case["op"] == "attend":
        out, weights = [], st["weights"].double() if case["weights"] else None
        group = case["heads"] // case["kv_heads"]
        for b, old in enumerate(lengths):
            n = old + case["tokens"]
            pages = st["table"][b, :-(-n // page)].long()
            k = st["kp"].index_select(0, pages).reshape(-1, case["kv_heads"], case["dim"])[:n].double()
            v = st["vp"].index_select(0, pages).reshape(-1, case["kv_heads"], case["dim"])[:n].double()
            rows = []
            for t in range(case["tokens"]):
                m = old + t + 1
                q = st["q"][b, t].double().view(case["kv_heads"], group, case["dim"])
                p = torch.softmax(torch.einsum("kgd,nkd->kgn", q, k[:m]) * case["dim"] ** -0.5, -1)
                rows.append(torch.einsum("kgn,nkd->kgd", p, v[:m]).reshape(case["heads"], case["dim"]))
                if case["weights"]:
                    weights[b, :, :m] += p.sum(1)
            out.append(torch.stack(rows))
        return [torch.stack(out), weights] if case["weights"] else [torch.stack(out)]
    k_to, v_to, w_to = st["kp_to"].double(), st["vp_to"].double(), st["weights_to"].double()
    for b, n in enumerate(lengths):
        for h in range(case["kv_heads"]):
            keep = torch.arange(n, device=DEVICE)
            if n > case["budget"]:
                old = n - case["recent"]
                # by weight, the lower index first where weights are equal
                order = (-st["weights"][b, h, :old].double()).argsort(stable=True)[:case["budget"] - case["recent"]]
                keep = torch.cat([order.sort().values, keep[old:]])
            to = torch.arange(keep.numel(), device=DEVICE)
            page_to, page_from = st["table_to"][b].long()[to // page], st["table"][b].long()[keep // page]
            k_to[page_to, to % page, h] = st["kp"][page_from, keep % page, h].double()
            v_to[page_to, to % page, h] = st["vp"][page_from, keep % page, h].double()
            w_to[b, h, :keep.numel()] = st["weights"][b, h][keep].double()
    return [None, k_to, v_to, w_to, None]


def _inputs_alone(case, seed):
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was


def _exact_append(case, st, lengths):
    f, factor = [], 1.0
    for i in range(case["rot"] // 2):
        x = 500000.0 ** (-2.0 * i / case["rot"])
        if case["scaling"] == "linear":
            x /= 8.0
        elif case["scaling"] == "llama3":
            turns = 8192.0 * x / (2 * math.pi)          # over the original context
            mix = min(1.0, max(0.0, (turns - 1.0) / 3.0))
            x = mix * x + (1 - mix) * x / 8.0
        elif case["scaling"] == "yarn":
            def place(turns):
                return case["rot"] * math.log(8192.0 / (turns * 2 * math.pi)) / (2 * math.log(500000.0))
            low, high = max(math.floor(place(32.0)), 0), min(math.ceil(place(1.0)), case["rot"] - 1)
            mix = min(1.0, max(0.0, (i - low) / ((high - low) or 0.001)))
            x, factor = x * (1 - mix) + x / 8.0 * mix, 0.1 * math.log(8.0) + 1.0
        f.append(x)
    f = torch.tensor(f, dtype=torch.float64, device=DEVICE)
    k_pages, v_pages = st["kp"].double(), st["vp"].double()
    starts, q_out = st["starts"].tolist(), st["q"].double()
    for b, old in enumerate(lengths):
        rows = torch.arange(starts[b], starts[b + 1], device=DEVICE)
        slots = old + torch.arange(rows.numel(), device=DEVICE)
        pages = st["table"][b].long()[slots // case["page"]]
        turn = torch.polar(torch.full((rows.numel(), f.numel()), factor, dtype=torch.float64, device=DEVICE),
                           slots.double()[:, None] * f)[:, None]
        for name in ("q", "k"):
            x = st[name][rows].double()
            lead = x[..., :case["rot"]].unflatten(-1, (-1, 2) if case["interleaved"] else (2, -1))
            dim = -1 if case["interleaved"] else -2
            z = torch.complex(*(t.contiguous() for t in lead.unbind(dim))) * turn
            x[..., :case["rot"]] = torch.stack([z.real, z.imag], dim).flatten(-2)
            if name == "q":
                q_out[rows] = x
            else:
                k_pages[pages, slots % case["page"]] = x
        v_pages[pages, slots % case["page"]] = st["v"][rows].double()
    return [q_out, k_pages, v_pages]
