"""Attention of many rows over the paged cache, drafts in a tree and log probabilities, as they are measured.

Five operators, each as a user's program calls it and in a plain form of elementary torch operations:

* window: rows of any number per sequence (one decoded token, prompts) attend over the pages, each to the
  last `window` tokens and the first `sinks` ones, or to all before it;
* tree: the nodes of a tree of drafted tokens attend over the pages and the nodes on their way up;
* walk: the tree's tokens taken or refused by what the target model draws behind each of them;
* keep: the taken nodes' keys and values moved behind the cached tokens;
* logprobs: log probability and rank of given tokens, entropy and the most likely tokens.

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
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ROWS = 65536            # rows x heads whose scores a plain pass over prompts holds at a time


def listed():
    return [
        # one decoded token of a model with a sliding window, a single user's session: latency
        {"name": "window one token", "op": "window", "batch": 1, "tokens": 1, "ragged": False, "len": 5000, "window": 1024,
         "sinks": 4, "heads": 32, "kv_heads": 8, "dim": 128, "type": "fp16", "page": 16, "order": "token"},
        # a decode step of a full serving batch of long conversations, each held to its window and sinks
        {"name": "window a batch's step", "op": "window", "batch": 64, "tokens": 1, "ragged": False, "len": 12001,
         "window": 4096, "sinks": 4, "heads": 64, "kv_heads": 8, "dim": 128, "type": "bf16", "page": 16, "order": "token"},
        # prompts of different lengths, some behind cached tokens, through a windowed layer: the products decide
        {"name": "window prompts", "op": "window", "batch": 4, "tokens": 8191, "ragged": True, "len": 4000, "window": 4096,
         "sinks": 16, "heads": 64, "kv_heads": 8, "dim": 128, "type": "fp16", "page": 16, "order": "token"},
        # a small tree of one sequence, as extra decoding heads propose it: latency
        {"name": "tree of one sequence", "op": "tree", "batch": 1, "nodes": 26, "ragged": False, "len": 4097, "window": 0,
         "sinks": 0, "heads": 32, "kv_heads": 8, "dim": 128, "type": "fp16", "page": 16, "order": "token"},
        # large trees of a serving batch's sequences
        {"name": "trees of a batch", "op": "tree", "batch": 32, "nodes": 64, "ragged": True, "len": 8190, "window": 0,
         "sinks": 0, "heads": 64, "kv_heads": 8, "dim": 128, "type": "bf16", "page": 20, "order": "head"},
        # the greedy walk through one sequence's tree: latency
        {"name": "walk greedily", "op": "walk", "batch": 1, "nodes": 26, "ragged": False, "depth": 5, "vocab": 32000,
         "temperature": 0.0},
        # sampled walks through a batch's trees
        {"name": "walk a batch", "op": "walk", "batch": 64, "nodes": 40, "ragged": True, "depth": 6, "vocab": 128256,
         "temperature": 0.8},
        # one sequence's taken nodes: latency
        {"name": "keep one path", "op": "keep", "batch": 1, "nodes": 26, "depth": 5, "len": 4097, "kv_heads": 8, "dim": 128,
         "type": "fp16", "page": 16, "order": "token"},
        # a batch's taken nodes
        {"name": "keep a batch's paths", "op": "keep", "batch": 64, "nodes": 64, "depth": 8, "len": 2000, "kv_heads": 32,
         "dim": 128, "type": "bf16", "page": 32, "order": "head"},
        # the tokens of one decode step, with the alternatives that an answer lists
        {"name": "logprobs of a step", "op": "logprobs", "rows": 4, "vocab": 32000, "top": 5, "type": "fp32"},
        # a long prompt scored token by token
        {"name": "logprobs of a prompt", "op": "logprobs", "rows": 2047, "vocab": 128256, "top": 0, "type": "fp32"},
        # half-precision logits of a large batch, twenty alternatives each
        {"name": "logprobs, twenty alternatives", "op": "logprobs", "rows": 1024, "vocab": 128256, "top": 20, "type": "bf16"},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("window", "window", "tree", "tree", "walk", "keep", "logprobs", "logprobs"))
    if op == "logprobs":
        rows, vocab = _log(rng, 1, 4096), _log(rng, 1000, 160000)
        case = {"op": op, "rows": rows, "vocab": vocab, "top": rng.choice((0, 1, 5, 20, rng.randint(0, 32))),
                "type": rng.choice(("fp32", "fp32", "fp16", "bf16"))}
        while case["rows"] * vocab > 2047 * 128256 // (1 if case["top"] == 0 and case["type"] == "fp32" else 2):
            case["rows"] = max(1, case["rows"] // 2)
        return case
    if op == "walk":
        case = {"op": op, "batch": _log(rng, 1, 64), "nodes": rng.choice((rng.randint(1, 64), rng.randint(8, 64))),
                "ragged": rng.random() < 0.5, "depth": rng.randint(1, 8), "vocab": _log(rng, 1000, 131072),
                "temperature": rng.choice((0.0, 0.6, 0.8, 1.0, 1.3))}
        while case["batch"] * case["nodes"] * case["vocab"] > 64 * 22 * 128256:
            case["batch"] = max(1, case["batch"] // 2)
        return case
    kv_heads, group = rng.choice(((8, 4), (8, 8), (32, 1), (1, 8), (2, 7), (4, 5), (8, 2)))
    case = {"op": op, "batch": _log(rng, 1, 64), "kv_heads": kv_heads, "dim": rng.choice((64, 128, 128)),
            "type": rng.choice(("fp16", "bf16")), "page": rng.choice((8, 16, 16, 20, 32, 64, 128)),
            "order": rng.choice(("token", "head"))}
    row = kv_heads * case["dim"]
    if op == "keep":
        case.update(nodes=rng.randint(2, 64), depth=rng.randint(1, 10), len=_log(rng, 1, 4000))
        while case["batch"] * (case["len"] + 64) * row > 64 * 2064 * 4096:
            case["len"] = max(1, case["len"] // 2)
        return case
    case.update(heads=kv_heads * group, len=_log(rng, 1, 100000), window=rng.choice((0, 0, _log(rng, 64, 8192))))
    case["sinks"] = rng.choice((0, 4, 16, rng.randint(1, 300))) if case["window"] else 0
    if op == "tree":
        case.update(nodes=rng.choice((rng.randint(1, 64), rng.randint(17, 64))), ragged=rng.random() < 0.5)
        while case["batch"] * (case["len"] + 64) * row > 32 * 4200 * 1024:
            case["batch"], case["len"] = max(1, case["batch"] // 2), max(1, case["len"] * 3 // 4)
        return case
    tokens = rng.choice((1, 1, rng.randint(2, 16), _log(rng, 17, 8000)))
    case.update(tokens=tokens, ragged=tokens > 1 and rng.random() < 0.7)
    while case["batch"] * (case["len"] + tokens) * row > 64 * 6100 * 1024:
        case["batch"], case["len"] = max(1, case["batch"] // 2), max(1, case["len"] * 3 // 4)
    while work(case)["flops"] > 3e12:
        case["batch"], case["len"], case["tokens"] = max(1, case["batch"] // 2), max(1, case["len"] // 2), max(2, case["tokens"] * 3 // 4)
    return case


# ---- shapes that a case fixes (the seed only permutes them) -------------------------------------


def _spread(n, low, high):
    """n whole numbers from high down to low, evenly."""
    return [high - (high - low) * i // max(1, n - 1) for i in range(n)]


def _rows_of(case):
    """How many new rows each sequence has."""
    most = case["nodes"] if case["op"] in ("tree", "walk") else case["tokens"]
    return _spread(case["batch"], max(1, most // 8), most) if case["ragged"] else [most] * case["batch"]


def _lengths_of(case):
    """How many tokens each sequence's cache holds before them."""
    low = 0 if case["op"] == "window" and case["tokens"] > 1 else 1
    return _spread(case["batch"], max(low, case["len"] // 64 * low), case["len"])


def _shuffled(values, gen):
    order = torch.randperm(len(values), generator=gen).tolist()
    return [values[i] for i in order]


def _tree(nodes, depth, gen):
    """Parents of a tree's nodes, every one before its children: node 0 is the root, the first `depth` nodes
    behind it a line, the others hang anywhere above the last level, first children more often."""
    parents, level = [-1], [0]
    for i in range(1, nodes):
        if i <= depth:
            p = i - 1
        else:
            open_ = [j for j in range(i) if level[j] < depth]
            u = float(torch.rand((), generator=gen))
            p = open_[min(len(open_) - 1, int(u * u * len(open_)))]
        parents.append(p)
        level.append(level[p] + 1)
    return parents, level


# ---- what a program has in hand -----------------------------------------------------------------


def _pool(case, batch, room, gen):
    """Pages for `batch` sequences of up to `room` tokens, handed out in a random order."""
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    each = -(-room // page)
    n = batch * each + 3
    shape = (n, page, heads, dim) if case["order"] == "token" else (n, heads, page, dim)
    pages = []
    for _ in range(2):
        t = torch.empty(shape, dtype=TYPES[case["type"]], device=DEVICE)
        t.normal_(generator=gen)
        pages.append(t if case["order"] == "token" else t.transpose(1, 2))
    table = torch.randperm(n, generator=gen, device=DEVICE)[:batch * each].to(torch.int32).view(batch, each)
    return pages[0], pages[1], table.contiguous()


def _framework():
    where = os.path.join(ROOT, "otf-llm-engine_b200")
    if where not in sys.path:
        sys.path.insert(0, where)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    cpu = torch.Generator().manual_seed(int(seed))
    st = {"case": case}
    if own:
        _framework()
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn(rows, vocab, generator=gen, device=DEVICE) * 2.5
        # a few likely continuations in every place, as a language model has them
        at = torch.randint(0, vocab, (rows, 8), generator=gen, device=DEVICE)
        x.scatter_add_(1, at, torch.rand(rows, 8, generator=gen, device=DEVICE) * 6 + 6)
        other = torch.randint(0, vocab, (rows,), generator=gen, device=DEVICE)
        likely = torch.rand(rows, generator=gen, device=DEVICE) < 0.7
        st.update(x=x.to(TYPES[case["type"]]), tokens=torch.where(likely, at[:, 0], other))
        return st
    batch = case["batch"]
    if case["op"] == "walk":
        return _prepare_walk(case, st, gen, cpu)
    lengths = _shuffled(_lengths_of({**case, "tokens": case.get("tokens", 2)}), cpu)
    st["lens"] = lengths
    st["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
    if case["op"] == "keep":
        st["kp"], st["vp"], st["table"] = _pool(case, batch, max(lengths) + case["nodes"], gen)
        # the taken nodes of each sequence: a way down through places in rising order
        taken = _shuffled(_spread(batch, 0 if batch > 1 else min(case["depth"], case["nodes"] - 1),
                                  min(case["depth"], case["nodes"] - 1)), cpu)
        path = torch.full((batch, case["depth"]), -1, dtype=torch.int32)
        for b, n in enumerate(taken):
            path[b, :n] = (torch.randperm(case["nodes"] - 1, generator=cpu)[:n].sort().values + 1).to(torch.int32)
        st["path"], st["accepted"] = path.to(DEVICE), torch.tensor(taken, dtype=torch.int32, device=DEVICE)
    else:
        new = _shuffled(_rows_of(case), cpu)
        st["new"], st["n"] = new, sum(new)
        st["starts"] = torch.tensor([0] + new, device=DEVICE).cumsum(0).to(torch.int32)
        st["kp"], st["vp"], st["table"] = _pool(case, batch, max(a + b for a, b in zip(lengths, new)), gen)
        st["q"] = torch.randn(st["n"], case["heads"], case["dim"], generator=gen, device=DEVICE).to(TYPES[case["type"]])
        if case["op"] == "tree":
            parents = [p for n in new for p in _tree(n, 6, cpu)[0]]
            st["parents"] = torch.tensor(parents, dtype=torch.int32, device=DEVICE)
    if own:
        from otf_llm.paged import PagedKVCache
        st["cache"] = PagedKVCache(st["kp"], st["vp"], st["table"], st["lengths"])
    return st


def _prepare_walk(case, st, gen, cpu):
    vocab = case["vocab"]
    new = _shuffled(_rows_of(case), cpu)
    n = sum(new)
    target = torch.randn(n, vocab, generator=gen, device=DEVICE) * 2.5
    spikes = torch.randint(0, vocab, (n, 8), generator=gen, device=DEVICE)
    target.scatter_add_(1, spikes, torch.rand(n, 8, generator=gen, device=DEVICE) * 6 + 6)
    st["target"], st["new"] = target, new
    st["starts"] = torch.tensor([0] + new, device=DEVICE).cumsum(0).to(torch.int32)
    best = target.topk(64 if vocab >= 64 else vocab, dim=1).indices.cpu()
    parents, tokens, at = [], [], 0
    for m in new:
        up, _ = _tree(m, case["depth"], cpu)
        children = [0] * m
        for i, p in enumerate(up):
            # the k-th child of a node is its k-th likeliest token
            tokens.append(int(best[at + p, children[p] % best.shape[1]]) if p >= 0 else 0)
            if p >= 0:
                children[p] += 1
        parents += up
        at += m
    st["parents"] = torch.tensor(parents, dtype=torch.int32, device=DEVICE)
    st["tokens"] = torch.tensor(tokens, dtype=torch.int64, device=DEVICE)
    if case["temperature"] > 0:
        st["noise"] = torch.empty(case["batch"], case["depth"] + 1, vocab, device=DEVICE).exponential_(generator=gen)
    return st


# ---- one pass -----------------------------------------------------------------------------------


def run(st):
    return {"window": _window, "tree": _tree_attention, "walk": _walk, "keep": _keep, "logprobs": _logprobs}[st["case"]["op"]](st)


def _attend(q, k, v, seen):
    """q [rows, heads, dim], k and v [keys, kv_heads, dim], seen [rows, keys]: softmax(q k / sqrt(dim)) v in 32 bits."""
    rows, heads, dim = q.shape
    kv = k.shape[1]
    x = q.float().view(rows, kv, heads // kv, dim).permute(1, 2, 0, 3).reshape(kv, -1, dim) / math.sqrt(dim)
    s = torch.matmul(x, k.float().permute(1, 2, 0)).view(kv, heads // kv, rows, -1)
    s = s.masked_fill(~seen, -math.inf)
    p = s.sub_(s.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).view(kv, -1, k.shape[0])
    out = torch.matmul(p, v.float().permute(1, 0, 2))
    return out.view(kv, heads // kv, rows, dim).permute(2, 0, 1, 3).reshape(rows, heads, dim).to(q.dtype)


def _window(st):
    case = st["case"]
    window, sinks = case["window"] or None, case["sinks"]
    if own:
        return [st["cache"].attend_rows(st["q"], starts=st["starts"], window=window, sinks=sinks)]
    if case["tokens"] == 1:
        return [_step(st)]
    # all sequences' scores do not fit: as many rows of one sequence at a time as may
    page, outs, row = case["page"], [], 0
    most = max(1, ROWS // case["heads"])
    blocks = [(b, t, min(t + most, n)) for b, n in enumerate(st["new"]) for t in range(0, n, most)]
    for b, t0, t1 in blocks:
        start = st["lens"][b]
        first = 0 if window is None else max(0, start + t0 - window + 1)
        place = torch.arange(first, start + t1, device=DEVICE)
        if first and sinks:
            place = torch.cat([torch.arange(min(sinks, first), device=DEVICE), place])
        at = st["table"][b].long()[place // page], place % page
        here = torch.arange(start + t0, start + t1, device=DEVICE)[:, None]
        seen = place <= here
        if window is not None:
            seen &= (place > here - window) | (place < sinks)
        outs.append(_attend(st["q"][row:row + t1 - t0], st["kp"][at], st["vp"][at], seen))
        row += t1 - t0
    return [torch.cat(outs)]


def _step(st):
    """One token of every sequence, all of them at once: the last `window` places and the first `sinks`."""
    case = st["case"]
    batch, kv, dim, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    here = st["lengths"].long()[:, None]
    if case["window"]:
        last = here - torch.arange(min(case["window"], case["len"] + 1) - 1, -1, -1, device=DEVICE)
        first = torch.arange(case["sinks"], device=DEVICE).expand(batch, -1)
        place = torch.cat([first, last], 1)
        # a sink inside the window is seen there
        seen = torch.cat([first < last[:, :1], last >= 0], 1)
    else:
        place = torch.arange(case["len"] + 1, device=DEVICE).expand(batch, -1)
        seen = place <= here
    place = torch.where(seen, place, 0)
    pages = st["table"].long().gather(1, place // page)
    k = st["kp"][pages, place % page].float().permute(0, 2, 3, 1)
    q = st["q"].float().view(batch, kv, -1, dim) / math.sqrt(dim)
    s = torch.matmul(q, k).masked_fill(~seen[:, None, None], -math.inf)
    del k
    p = (s - s.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    v = st["vp"][pages, place % page].float().transpose(1, 2)
    return torch.matmul(p, v).reshape(batch, case["heads"], dim).to(st["q"].dtype)


def _above(parents, of, node, batch, nodes):
    """[rows, nodes] of truth: whether the j-th node of a row's sequence is the row's own or above it."""
    reach = torch.eye(nodes, device=DEVICE).repeat(batch, 1, 1)
    up = parents.long()
    reach[of, node, torch.where(up < 0, node, up)] = 1.0
    for _ in range(6):                                  # ways of up to 64 steps
        reach = torch.matmul(reach, reach).clamp(max=1.0)
    return reach[of, node] > 0


def _tree_attention(st):
    case = st["case"]
    if own:
        return [st["cache"].attend_tree(st["q"], st["parents"], starts=st["starts"], window=case["window"] or None,
                                        sinks=case["sinks"])]
    batch, kv, dim, page, nodes = case["batch"], case["kv_heads"], case["dim"], case["page"], case["nodes"]
    group = case["heads"] // kv
    row = torch.arange(st["n"], device=DEVICE)
    of = torch.bucketize(row, st["starts"][1:].long(), right=True)
    node = row - st["starts"].long()[of]
    above = _above(st["parents"], of, node, batch, nodes)
    depth = above.sum(1) - 1
    # rows of every sequence side by side, padded to the most nodes
    q = torch.zeros(batch, nodes, case["heads"], dim, device=DEVICE)
    q[of, node] = st["q"].float() / math.sqrt(dim)
    table = st["table"].long()
    place = torch.arange(table.shape[1] * page, device=DEVICE)
    start = st["lengths"].long()[of][:, None]
    seen = place < start
    if case["window"]:
        seen = seen & ((place > start + depth[:, None] - case["window"]) | (place < case["sinks"]))
    drafted = place - start
    seen = seen | ((drafted >= 0) & (drafted < nodes) & above.gather(1, drafted.clamp(0, nodes - 1)))
    mask = torch.ones(batch, nodes, place.shape[0], dtype=torch.bool, device=DEVICE)
    mask[of, node] = seen
    k = st["kp"][table].reshape(batch, -1, kv, dim).permute(0, 2, 3, 1).float()
    x = q.view(batch, nodes, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv, group * nodes, dim)
    s = torch.matmul(x, k).view(batch, kv, group, nodes, -1)
    del k
    s = s.masked_fill_(~mask[:, None, None], -math.inf)
    p = s.sub_(s.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).view(batch, kv, group * nodes, -1)
    v = st["vp"][table].reshape(batch, -1, kv, dim).transpose(1, 2).float()
    out = torch.matmul(p, v).view(batch, kv, group, nodes, dim).permute(0, 3, 1, 2, 4).reshape(batch, nodes, case["heads"], dim)
    return [out[of, node].to(st["q"].dtype)]


def _walk(st):
    case = st["case"]
    if own:
        from otf_llm.speculative import verify_tree
        return list(verify_tree(st["target"], st["tokens"], st["parents"], starts=st["starts"], depth=case["depth"],
                                noise=st.get("noise"), temperature=case["temperature"]))
    batch, depth, T = case["batch"], case["depth"], case["temperature"]
    starts = st["starts"].long()
    n = st["tokens"].shape[0]
    row = torch.arange(n, device=DEVICE)
    of = torch.bucketize(row, starts[1:], right=True)
    up = torch.where(st["parents"] < 0, -1, st["parents"].long() + starts[of])
    at, going = starts[:-1].clone(), torch.ones(batch, dtype=torch.bool, device=DEVICE)
    tokens = torch.full((batch, depth + 1), -1, dtype=torch.int64, device=DEVICE)
    path = torch.full((batch, depth), -1, dtype=torch.int32, device=DEVICE)
    accepted = torch.zeros(batch, dtype=torch.int32, device=DEVICE)
    for j in range(depth + 1):
        x = st["target"][at]
        if T == 0:
            drawn = x.argmax(1)
        else:
            x = x.double()
            p = ((x - x.amax(1, keepdim=True)) / T).exp()
            drawn = (p / p.sum(1, keepdim=True) / st["noise"][:, j].double()).argmax(1)
        tokens[:, j] = torch.where(going, drawn, -1)
        if j == depth:
            break
        hit = (up == at[of]) & (st["tokens"] == drawn[of])
        child = torch.full((batch,), n, dtype=torch.int64, device=DEVICE).scatter_reduce_(
            0, of, torch.where(hit, row, n), "amin")
        going = going & (child < n)
        at = torch.where(going, child, at)
        path[:, j] = torch.where(going, child - starts[:-1], -1)
        accepted += going
    return [tokens, path, accepted]


def _keep(st):
    case = st["case"]
    if own:
        st["cache"].keep(st["path"], st["accepted"])
        return [st["kp"], st["vp"]]
    page, depth = case["page"], case["depth"]
    j = torch.arange(depth, device=DEVICE)
    start = st["lengths"].long()[:, None]
    stays = j < st["accepted"].long()[:, None]
    src = start + torch.where(stays, st["path"].long(), 0)
    to = start + torch.where(stays, j + 1, 0)           # the others: the root to itself
    table = st["table"].long()
    page_from, page_to = table.gather(1, src // page), table.gather(1, to // page)
    for pool in (st["kp"], st["vp"]):
        pool[page_to, to % page] = pool[page_from, src % page]
    return [st["kp"], st["vp"]]


def _logprobs(st):
    case = st["case"]
    if own:
        from otf_llm.logprobs import token_logprobs
        got = token_logprobs(st["x"], st["tokens"], top=case["top"])
        return [got.logprobs, got.entropy, got.ranks] + ([got.top_tokens, got.top_logprobs] if case["top"] else [])
    x = st["x"].float()
    m = x.amax(1, keepdim=True)
    d = x - m
    e = d.exp()
    total = e.sum(1, dtype=torch.float64)
    entropy = total.log() - e.mul_(d).sum(1, dtype=torch.float64) / total
    del e
    mine = x.gather(1, st["tokens"][:, None])
    place = torch.arange(case["vocab"], device=DEVICE)
    ranks = ((x > mine) | ((x == mine) & (place < st["tokens"][:, None]))).sum(1).to(torch.int32)
    lse = m[:, 0].double() + total.log()
    out = [(mine[:, 0].double() - lse).float(), entropy.float(), ranks]
    if case["top"]:
        del d
        best = x.sort(dim=1, descending=True, stable=True)
        out += [best.indices[:, :case["top"]].contiguous(), (best.values[:, :case["top"]].double() - lse[:, None]).float()]
    return out


# ---- what a pass cannot do without ---------------------------------------------------------------


def _sum(n):
    return n * (n + 1) // 2


def _capped(n, most):
    """1 + 2 + ... + n, each no more than `most`."""
    return _sum(min(n, most)) + max(0, n - most) * most


def _seen(case):
    """Of all sequences together: the cached or new tokens that some row sees, and the sum over rows of what each sees."""
    keys = pairs = 0
    window, sinks = case["window"] or 1 << 40, case["sinks"]
    for n, new in zip(_lengths_of(case), _rows_of(case)):
        if case["op"] == "tree":
            cached = min(n, window + min(sinks, max(0, n - window)))
            keys += cached + new
            pairs += (cached + min(new, 5)) * new
            continue
        first = max(0, n - window + 1)
        keys += n + new - first + min(sinks, first)
        # the row at place p sees p + 1 tokens up to a window's, then a window and what sinks lie before it
        pairs += _sum(min(n + new, window)) - _sum(min(n, window))
        low, high = max(n, window) - window, max(n + new, window) - window
        pairs += (high - low) * window + _capped(high, sinks) - _capped(low, sinks)
    return keys, pairs


def work(case):
    if case["op"] == "logprobs":
        size = 4 if case["type"] == "fp32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 20 + 12 * case["top"]), "flops": case["rows"] * case["vocab"] * 5}
    if case["op"] == "walk":
        # a sequence looks at as many rows as tokens that it produces: three of four levels, as trees like these go
        steps = case["batch"] * (1 + min(case["depth"], case["nodes"] - 1) * 3 // 4)
        rows = steps * (2 if case["temperature"] > 0 else 1)
        return {"bytes": rows * case["vocab"] * 4 + sum(_rows_of(case)) * 12, "flops": rows * case["vocab"] * 2}
    row = case["kv_heads"] * case["dim"]
    if case["op"] == "keep":
        most = min(case["depth"], case["nodes"] - 1)
        moved = sum(_spread(case["batch"], 0 if case["batch"] > 1 else most, most))
        return {"bytes": moved * row * 8 + case["batch"] * (case["depth"] + 2) * 4, "flops": moved}
    keys, pairs = _seen(case)
    return {"bytes": keys * row * 4 + sum(_rows_of(case)) * case["heads"] * case["dim"] * 4,
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---- the definitions in 64 bits -------------------------------------------------------------------


def _inputs_alone(case, seed):
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was


def exact(case, seed):
    if case["op"] == "walk":
        return None                                     # whole numbers alone
    st = _inputs_alone(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(case, st)
    page = case["page"]
    if case["op"] == "keep":
        k, v = st["kp"].double(), st["vp"].double()
        for b, (n, taken) in enumerate(zip(st["lens"], st["accepted"].tolist())):
            for j in range(taken):
                a, z = n + int(st["path"][b, j]), n + 1 + j
                for new, old in ((k, st["kp"]), (v, st["vp"])):
                    new[st["table"][b, z // page], z % page] = old[st["table"][b, a // page], a % page].double()
        return [k, v]
    outs, row = [], 0
    window, sinks, group = case["window"] or 1 << 40, case["sinks"], case["heads"] // case["kv_heads"]
    for n, new in zip(st["lens"], st["new"]):
        b = len(outs)
        pages = st["table"][b, :-(-(n + new) // page)].long()
        k = st["kp"].index_select(0, pages).flatten(0, 1)[:n + new].double().transpose(0, 1)
        v = st["vp"].index_select(0, pages).flatten(0, 1)[:n + new].double().transpose(0, 1)
        place = torch.arange(n + new, device=DEVICE)
        if case["op"] == "tree":
            parents = st["parents"][row:row + new].tolist()
            seen = torch.zeros(new, n + new, dtype=torch.bool, device=DEVICE)
            depths = []
            for i, p in enumerate(parents):
                depths.append(0 if p < 0 else depths[p] + 1)
                if p >= 0:
                    seen[i, n:] = seen[p, n:]
                seen[i, n + i] = True
            here = n + torch.tensor(depths, device=DEVICE)[:, None]
            seen[:, :n] = ((here - place[:n] < window) | (place[:n] < sinks))
        part = []
        for t in range(0, new, 256):
            q = st["q"][row + t:row + min(t + 256, new)].double()
            q = q.view(-1, case["kv_heads"], group, case["dim"]).permute(1, 2, 0, 3)
            if case["op"] == "tree":
                mine = seen[t:t + 256]
            else:
                here = n + torch.arange(t, min(t + 256, new), device=DEVICE)[:, None]
                mine = (place <= here) & ((here - place < window) | (place < sinks))
            low, high = 0, n + new
            if window < n and not sinks:
                low = max(0, n + (t if case["op"] == "window" else 0) - window)
            if case["op"] == "window":
                high = min(high, n + t + 256)
            s = torch.einsum("kgtd,knd->kgtn", q, k[:, low:high]) * case["dim"] ** -0.5
            p = torch.softmax(torch.where(mine[:, low:high], s, -math.inf), -1)
            part.append(torch.einsum("kgtn,knd->tkgd", p, v[:, low:high]).reshape(-1, case["heads"], case["dim"]))
        outs.append(torch.cat(part))
        row += new
    return [torch.cat(outs)]


def _exact_logprobs(case, st):
    parts = []
    for r in range(0, case["rows"], 128):
        x = st["x"][r:r + 128].double()
        lp = torch.log_softmax(x, 1)
        part = [lp.gather(1, st["tokens"][r:r + 128, None])[:, 0], -(lp.exp() * lp).sum(1)]
        if case["top"]:
            part.append(lp.topk(case["top"], dim=1).values)
        parts.append(part)
    out = [torch.cat(p) for p in zip(*parts)]
    return out[:2] + [None] + ([None, out[2]] if case["top"] else [])
