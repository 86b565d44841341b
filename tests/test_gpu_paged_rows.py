"""Attention of rows of any number per sequence over the paged cache, in a line or in a tree, through windows with
sinks, against its definition in 64 bits."""
import pytest
import torch

import paged_oracle as ref
import rows_oracle as rows
from test_gpu_paged import TYPES, flag, make, same

pytestmark = pytest.mark.gpu


def tree(n, g, wide=3):
    return [-1] + [int(torch.randint(max(0, i - wide * 2), i, (), generator=g)) for i in range(1, n)]


def check(dev, lengths, new, page, heads, kv, dim, dtype, order="token", window=None, sinks=0, trees=False, scale=None,
          extra=0, uniform=False, seed=1, poison=False):
    """Every row against 64 bits; rows of no sequence keep what they held."""
    cache, pools, table, g = make(dev, [n + t if n >= 0 else n for n, t in zip(lengths, new)], page, kv, dim, dtype, order,
                                  room=[max(n, 0) + t + 1 for n, t in zip(lengths, new)], seed=seed)
    cache.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    n = sum(new)
    q = torch.randn(n + extra, heads, dim, generator=g).to(dtype)
    starts = None if uniform else torch.tensor([0] + new).cumsum(0).to(torch.int32).to(dev)
    parents = [tree(t, g) for t in new] if trees else [None] * len(new)
    out = torch.full((n + extra, heads, dim), 7.0, dtype=dtype, device=dev)
    if trees:
        flat = torch.tensor([p for up in parents for p in up] + [5] * extra, dtype=torch.int32, device=dev)
        got = cache.attend_tree(q.to(dev), flat, starts=starts, window=window, sinks=sinks, scale=scale, out=out)
    else:
        got = cache.attend_rows(q.to(dev), starts=starts, window=window, sinks=sinks, scale=scale, out=out)
    assert got is out and flag() == 0
    got = got.cpu()
    rep = heads // kv
    row = 0
    for b, t in enumerate(new):
        if lengths[b] < 0:
            assert bool((got[row:row + t] == 7.0).all())
        else:
            want = rows.attend(pools, table, lengths[b], q[row:row + t], b, window, sinks,
                               dim ** -0.5 if scale is None else scale, parents[b])
            for j, w in enumerate(want):
                far = (got[row + j].double() - w[0]).abs()
                # a block of 256 rows (tokens x query heads of a KV head) with more than 128 rounds probabilities once
                once = any(min(256, t * rep - r // 256 * 256) > 128 for r in (j * rep, j * rep + rep - 1))
                most = rows.tolerance(w, dim, dtype, once)
                assert bool((far <= most).all()), (b, j, float((far / most).max()))
        row += t
    assert bool((got[n:] == 7.0).all())


ROWS = [
    # lengths, new rows, page, heads, kv, dim, window, sinks
    ([0], [1], 16, 1, 1, 64, None, 0),
    ([5, 0, -1, 33], [1, 1, 1, 1], 16, 8, 2, 128, None, 0),
    ([300], [1], 16, 8, 2, 128, 70, 4),
    ([700, 129, 127, 128], [1, 1, 1, 1], 20, 4, 1, 128, 128, 3),
    ([10, 0, 200], [3, 140, 17], 8, 4, 2, 64, None, 0),
    ([0, 250], [130, 300], 1, 4, 2, 128, None, 0),
    ([400], [70], 16, 7, 1, 128, 50, 5),
    ([0, 600], [260, 40], 128, 5, 5, 64, 1, 0),
    ([450, 3], [33, 129], 64, 8, 1, 128, 130, 150),
    ([900], [5], 3, 28, 4, 64, 200, 300),
    ([0, 0, 7], [0, 300, 1], 16, 8, 2, 64, 64, 1),
    ([1030], [1], 16, 32, 1, 128, 1 << 33, 7),
]


@pytest.mark.parametrize("dtype,order", [("fp16", "token"), ("bf16", "head")])
@pytest.mark.parametrize("lengths,new,page,heads,kv,dim,window,sinks", ROWS)
def test_rows_match_definition(lengths, new, page, heads, kv, dim, window, sinks, dtype, order, cuda_dev):
    check(cuda_dev, lengths, new, page, heads, kv, dim, TYPES[dtype], order, window, sinks, extra=2)


TREES = [
    ([0], [1], 16, 1, 1, 64, None, 0),
    ([200], [26], 16, 4, 1, 128, None, 0),
    ([130, -2, 1, 64], [64, 5, 33, 12], 20, 8, 2, 64, None, 0),
    ([500, 0], [64, 64], 8, 8, 2, 128, 64, 3),
    ([260], [64], 16, 16, 2, 128, 100, 140),
    ([127, 128, 100], [1, 2, 60], 7, 3, 3, 64, None, 0),
]


@pytest.mark.parametrize("dtype,order", [("fp16", "head"), ("bf16", "token")])
@pytest.mark.parametrize("lengths,new,page,heads,kv,dim,window,sinks", TREES)
def test_trees_match_definition(lengths, new, page, heads, kv, dim, window, sinks, dtype, order, cuda_dev):
    check(cuda_dev, lengths, new, page, heads, kv, dim, TYPES[dtype], order, window, sinks, trees=True, extra=1)


def test_long_lengths_split_over_many_parts(cuda_dev):
    """One sequence's keys over all CTAs: parts of one item from more than 32 of them, joined; 8, 60 and 128 rows."""
    check(cuda_dev, [6000], [1], 16, 8, 1, 128, torch.float16)
    check(cuda_dev, [5000], [15], 16, 4, 1, 64, torch.bfloat16, trees=True)
    check(cuda_dev, [5003], [32], 20, 4, 1, 128, torch.float16)
    check(cuda_dev, [4000], [70], 16, 4, 1, 64, torch.float16, window=3000, sinks=700)


def test_many_sequences_and_uniform_rows(cuda_dev):
    check(cuda_dev, [(37 * b) % 90 for b in range(70)], [1] * 70, 8, 4, 2, 64, torch.float16, uniform=True)
    check(cuda_dev, [(31 * b) % 150 for b in range(40)], [b % 4 for b in range(40)], 16, 2, 1, 64, torch.bfloat16, extra=3)
    check(cuda_dev, [9, 40, 70], [12, 12, 12], 16, 8, 2, 128, torch.float16, trees=True, uniform=True)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30, 3.0])
def test_scales(scale, cuda_dev):
    check(cuda_dev, [140, 3], [5, 130], 16, 4, 2, 64, torch.float16, scale=scale, window=90, sinks=2)
    check(cuda_dev, [140], [9], 16, 8, 2, 128, torch.bfloat16, scale=scale, trees=True)


def far_seen(lengths, new, window, sinks, parents):
    return [[rows.seen(n, t, window, sinks, parents[b]) for t in range(new[b])] for b, n in enumerate(lengths)]


@pytest.mark.parametrize("lengths,new,heads,kv,dim,window,sinks,trees", [
    ([200], [6], 4, 1, 128, 100, 3, False), ([150], [40], 4, 2, 64, None, 0, True), ([60], [180], 2, 1, 128, 70, 5, False),
    ([0], [130], 3, 1, 64, None, 0, False), ([300], [26], 4, 1, 128, None, 0, True)])
def test_what_a_row_does_not_see_does_not_reach_it(lengths, new, heads, kv, dim, window, sinks, trees, cuda_dev):
    """Infinities and NaN among keys and values: rows that see them are odd, all others are as if they were not there."""
    n = lengths[0]
    cache, pools, table, g = make(cuda_dev, [n + new[0]], 16, kv, dim, torch.float16, room=[n + new[0] + 1], seed=3)
    q = torch.randn(new[0], heads, dim, generator=g).half()
    parents = tree(new[0], g) if trees else None
    cache.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))

    def run():
        if trees:
            return cache.attend_tree(q.to(cuda_dev), torch.tensor(parents, dtype=torch.int32, device=cuda_dev), window=window,
                                     sinks=sinks).cpu()
        return cache.attend_rows(q.to(cuda_dev), window=window, sinks=sinks).cpu()
    plain = run()
    for place, pool, value, dims in ((n + new[0] // 2, 1, float("inf"), [dim - 1]), (n + 1, 1, float("nan"), [0, 33]),
                                     (max(0, n - 60), 1, float("-inf"), [5]), (n + new[0] - 1, 0, float("nan"), [2])):
        at = ref.place(table, 16, 0, place)
        page = (cache.k_pages, cache.v_pages)[pool]
        kept = page[at].clone()
        page[at][:, dims] = value
        got = run()
        page[at] = kept
        for t in range(new[0]):
            if place in rows.seen(n, t, window, sinks, parents):
                assert bool((~got[t][:, dims if pool else slice(None)].isfinite()).all()), (place, t)
                if pool:
                    clean = [d for d in range(dim) if d not in dims]
                    assert same(got[t][:, clean], plain[t][:, clean]), (place, t)
            else:
                assert same(got[t], plain[t]), (place, t)
    assert flag() == 0


def test_results_do_not_depend_on_what_lies_around(cuda_dev):
    """The same call twice gives the same bits, whatever ran in between (rows that are not there hold stale values)."""
    def call():
        cache, _, _, g = make(cuda_dev, [700, 90], 16, 1, 128, torch.bfloat16, room=[720, 300], seed=5)
        cache.lengths.copy_(torch.tensor([690, 80], dtype=torch.int32))
        q = torch.randn(10 + 150, 3, 128, generator=g).bfloat16().to(cuda_dev)
        return cache.attend_rows(q, starts=torch.tensor([0, 10, 160], dtype=torch.int32, device=cuda_dev), window=333, sinks=1)
    one = call()
    check(cuda_dev, [300], [200], 16, 4, 1, 128, torch.float16, scale=5.0)
    assert same(one, call())


def test_strides_views_and_other_places(cuda_dev):
    """Queries as part of a fused projection's rows, outputs as columns of a wider buffer."""
    cache, _, _, g = make(cuda_dev, [40, 7], 16, 2, 64, torch.float16, room=[60, 60])
    cache.lengths.copy_(torch.tensor([30, 5], dtype=torch.int32))
    wide = torch.randn(12, 9, 64, generator=g).half().to(cuda_dev)
    q = wide[:, 1:5]
    plain = cache.attend_rows(q.contiguous())
    buffer = torch.zeros(12, 11, 64, dtype=torch.float16, device=cuda_dev)
    out = cache.attend_rows(q, out=buffer[:, 3:7])
    assert out.data_ptr() == buffer[:, 3:7].data_ptr() and same(out, plain)
    assert not buffer[:, :3].any() and not buffer[:, 7:].any()
    # beside the queries themselves
    before = wide[:, :5].clone()
    assert same(cache.attend_rows(q, out=wide[:, 5:]), plain) and same(wide[:, :5], before)
    parents = torch.tensor([-1, 0, 1, 1, 0, 2] * 2, dtype=torch.int32, device=cuda_dev)
    assert same(cache.attend_tree(q, parents), cache.attend_tree(q.contiguous(), parents))
    assert flag() == 0


def test_pages_outside_sequences_that_do_not_fit_and_bad_parents(cuda_dev):
    cache, pools, table, g = make(cuda_dev, [40, 30], 16, 1, 64, torch.float16, room=[47, 47])
    cache.lengths.copy_(torch.tensor([35, 28], dtype=torch.int32))
    q = torch.randn(8, 2, 64, generator=g).half().to(cuda_dev)
    plain = cache.attend_rows(q[:7], starts=torch.tensor([0, 5, 7], dtype=torch.int32, device=cuda_dev))
    assert flag() == 0
    # more rows than the table has room for, and starts that run backwards or past the rows
    seven = torch.full((8, 2, 64), 7.0, dtype=torch.float16, device=cuda_dev)
    cache.lengths.copy_(torch.tensor([62, 28], dtype=torch.int32))
    got = cache.attend_rows(q, starts=torch.tensor([0, 5, 7], dtype=torch.int32, device=cuda_dev), out=seven.clone())
    assert flag() == 1 and bool((got[:5] == 7).all()) and same(got[5:7], plain[5:]) and bool((got[7] == 7).all())
    cache.lengths.copy_(torch.tensor([35, 28], dtype=torch.int32))
    got = cache.attend_rows(q, starts=torch.tensor([0, 5, 9], dtype=torch.int32, device=cuda_dev), out=seven.clone())
    assert flag() == 1 and same(got[:5], plain[:5]) and bool((got[5:] == 7).all())
    got = cache.attend_rows(q, starts=torch.tensor([4, 2, 4], dtype=torch.int32, device=cuda_dev), out=seven.clone())
    assert flag() == 1 and bool((got[:2] == 7).all()) and bool((got[4:] == 7).all())
    # a page outside the pool reads as zeros
    kept = cache.page_table[0, 1].clone()
    cache.page_table[0, 1] = 10 ** 6
    got = cache.attend_rows(q[:5], starts=torch.tensor([0, 5, 5], dtype=torch.int32, device=cuda_dev))
    assert flag() == 1
    cache.page_table[0, 1] = kept
    at = int(kept)
    saved = cache.k_pages[at].clone(), cache.v_pages[at].clone()
    cache.k_pages[at], cache.v_pages[at] = 0, 0
    assert same(got, cache.attend_rows(q[:5], starts=torch.tensor([0, 5, 5], dtype=torch.int32, device=cuda_dev)))
    cache.k_pages[at], cache.v_pages[at] = saved
    # parents out of range count as -1; 65 nodes are left out
    bad = cache.attend_tree(q[:4], torch.tensor([-1, 1, -7, 0], dtype=torch.int32, device=cuda_dev))
    assert flag() == 1
    good = cache.attend_tree(q[:4], torch.tensor([-1, -1, -1, 0], dtype=torch.int32, device=cuda_dev))
    assert flag() == 0 and same(bad, good)
    big, _, _, g = make(cuda_dev, [5, 5], 16, 1, 64, torch.float16, room=[90, 90], fill=0.0)
    q = torch.randn(66, 1, 64, generator=g).half().to(cuda_dev)
    got = big.attend_tree(q, torch.full((66,), -1, dtype=torch.int32, device=cuda_dev),
                          starts=torch.tensor([0, 65, 66], dtype=torch.int32, device=cuda_dev),
                          out=torch.full_like(q, 7.0))
    assert flag() == 1 and bool((got[:65] == 7).all()) and not bool((got[65] == 7).any())


def test_captured_replayed_and_on_two_streams(cuda_dev):
    """Two captured calls on streams of their own, replayed at the same time with other lengths and rows."""
    made = []
    for i in range(2):
        cache, pools, table, g = make(cuda_dev, [400 + i, 77], 16, 2, 128, torch.float16, room=[500, 300], seed=20 + i)
        q = torch.randn(60, 8, 128, generator=g).half().to(cuda_dev)
        starts = torch.tensor([0, 20, 60], dtype=torch.int32, device=cuda_dev)
        cache.lengths.copy_(torch.tensor([380, 30], dtype=torch.int32))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            cache.attend_rows(q, starts=starts, window=200, sinks=3)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = cache.attend_rows(q, starts=starts, window=200, sinks=3)
        made.append((cache, q, starts, side, graph, out))
    torch.cuda.synchronize()
    for cache, q, starts, *_ in made:
        cache.lengths.copy_(torch.tensor([350, 37], dtype=torch.int32))
        starts.copy_(torch.tensor([0, 50, 60], dtype=torch.int32))
    torch.cuda.synchronize()
    for _ in range(10):
        for *_, side, graph, out in made:
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    for cache, q, starts, _, _, out in made:
        assert same(out, cache.attend_rows(q, starts=starts, window=200, sinks=3))
    assert flag() == 0


def test_as_prefill_and_decode_attention(cuda_dev):
    """Beside attend: the same newest tokens of every sequence, within both calls' roundings; and a prompt's rows are what
    its tokens would have got one by one."""
    cache, pools, table, g = make(cuda_dev, [333, 20, 64], 16, 2, 128, torch.float16, room=[350, 40, 80])
    cache.lengths.copy_(torch.tensor([330, 17, 61], dtype=torch.int32))
    q = torch.randn(3, 3, 8, 128, generator=g).half()
    a, b = cache.attend(q.to(cuda_dev)).cpu(), cache.attend_rows(q.view(9, 8, 128).to(cuda_dev)).cpu().view(3, 3, 8, 128)
    for s, n in enumerate((330, 17, 61)):
        for w, x, y in zip(rows.attend(pools, table, n, q[s], s, None, 0, 128 ** -0.5), a[s], b[s]):
            most = rows.tolerance(w, 128, torch.float16, False)
            assert bool(((x.double() - y.double()).abs() <= 2 * most).all())


def test_a_tree_as_it_is_used(cuda_dev):
    """Prompts through append and attend_rows, then drafts in trees: append with the nodes' positions, attend_tree,
    verify_tree, keep and advance; after it the cache holds what the taken tokens alone would have written, and the
    answer's log probabilities are the target's."""
    from otf_llm.logprobs import token_logprobs
    from otf_llm.paged import PagedKVCache, Rotary
    from otf_llm.speculative import verify_tree
    g = torch.Generator().manual_seed(7)
    batch, heads, kv, dim, vocab, dev = 3, 4, 2, 64, 50, cuda_dev
    table = torch.randperm(30, generator=g)[:24].view(3, 8).to(torch.int32).to(dev)
    lengths = torch.tensor([0, 0, -1], dtype=torch.int32, device=dev)
    cache = PagedKVCache.allocate(30, 16, kv, dim, table, lengths)
    rotary = Rotary(dim, theta=10000.0, device=dev)
    embed = torch.randn(vocab, (heads + 2 * kv) * dim, generator=g).half().to(dev)
    head = (torch.randn(heads * dim, vocab, generator=g) * 0.4).half().to(dev)

    def qkv(ids):
        return embed[ids].view(-1, heads + 2 * kv, dim).split([heads, kv, kv], dim=1)

    prompts = [torch.randint(0, vocab, (n,), generator=g) for n in (20, 45)]
    starts = torch.tensor([0, 20, 65, 65], dtype=torch.int32, device=dev)
    q = cache.append(*qkv(torch.cat(prompts).to(dev)), rotary, starts=starts)
    out = cache.attend_rows(q, starts=starts, window=32, sinks=2)
    cache.advance(starts.diff())
    logits = out.reshape(65, -1).float() @ head.float()
    certain = logits[[19, 64]].argmax(1)
    answers = [[int(t)] for t in certain]
    for step in range(3):
        parents = [[-1, 0, 0, 1, 1, 2, 3], [-1, 0, 1, 2]]
        # children: what the token alone would lead to, and others
        trees = [[answers[b][-1]] + [int(torch.randint(0, vocab, (), generator=g)) for _ in up[1:]] for b, up in enumerate(parents)]
        flat = torch.tensor([t for tr in trees for t in tr], device=dev)
        ups = torch.tensor([p for up in parents for p in up], dtype=torch.int32, device=dev)
        starts = torch.tensor([0, 7, 11, 11], dtype=torch.int32, device=dev)
        depth = torch.tensor([d for up in parents for d in rows.levels(up)], dtype=torch.int32, device=dev)
        of = torch.tensor([0] * 7 + [1] * 4, device=dev)
        before = lengths.clone()
        q = cache.append(*qkv(flat), rotary, starts=starts, positions=lengths[of] + depth)
        out = cache.attend_tree(q, ups, starts=starts, window=64, sinks=1)
        logits = out.reshape(11, -1).float() @ head.float()
        # so that some are taken: the first child of each root holds the root's likeliest token
        for b, at in ((0, 1), (1, 8)):
            flat[at] = logits[0 if b == 0 else 7].argmax()
        tokens, path, accepted = verify_tree(logits, flat, ups, starts=starts, depth=3, temperature=0.0)
        assert accepted.tolist()[2] == 0 and accepted[:2].ge(1).all()
        cache.keep(path, accepted)
        cache.advance(accepted + 1)
        assert lengths.tolist() == [int(before[0] + accepted[0] + 1), int(before[1] + accepted[1] + 1), -1]
        for b in range(2):
            answers[b] += [t for t in tokens[b].tolist() if t >= 0]
            first = 0 if b == 0 else 7
            way = [first] + [first + i for i in path[b].tolist() if i >= 0]
            got = token_logprobs(logits[way], tokens[b, :len(way)].contiguous(), top=2)
            want = torch.log_softmax(logits[way].double(), 1)
            assert torch.allclose(got.logprobs.double(), want.gather(1, tokens[b, :len(way), None])[:, 0], atol=1e-6, rtol=1e-6)
            assert got.ranks.eq(0).all() and got.top_tokens[:, 0].tolist() == tokens[b, :len(way)].tolist()
            # the taken nodes lie one behind another (their drafted keys: those of the tokens they were appended with)
            for j, row in enumerate(way):
                at = ref.place(table.cpu(), 16, b, int(before[b]) + j)
                x = embed[torch.tensor([trees[b][row - first]], device=dev)].view(1, heads + 2 * kv, dim)
                assert same(cache.v_pages[at].cpu(), x[0, heads + kv:].cpu())
    assert flag() == 0


@pytest.mark.parametrize("dim,dtype", [(128, "fp16"), (64, "bf16")])
def test_large_and_small_blocks_in_one_run(dim, dtype, cuda_dev):
    """Blocks of 256 rows, of more and fewer than 128 and of a few, several of each on every SM one after another: what
    one leaves behind must not reach the next one's queries."""
    new = [130, 5, 200, 64, 33, 129, 1]
    check(cuda_dev, [20, 150, 0, 33, 260, 7, 300], new, 16, 192, 96, dim, TYPES[dtype], window=140, sinks=1)


def test_a_block_of_one_node_does_not_see_its_siblings(cuda_dev):
    """33 nodes of 8 query heads: the last block has one node's rows alone, and the others' values are odd."""
    cache, _, table, g = make(cuda_dev, [100 + 33], 16, 1, 128, torch.float16, room=[140], seed=9)
    cache.lengths.fill_(100)
    q = torch.randn(33, 8, 128, generator=g).half().to(cuda_dev)
    parents = torch.full((33,), -1, dtype=torch.int32, device=cuda_dev)
    plain = cache.attend_tree(q, parents)
    for place in (100, 131):
        at = ref.place(table, 16, 0, place)
        kept = cache.v_pages[at].clone()
        cache.v_pages[at][:] = float("nan")
        got = cache.attend_tree(q, parents)
        cache.v_pages[at] = kept
        others = [t for t in range(33) if t != place - 100]
        assert same(got[others], plain[others]) and bool(got[place - 100].isnan().all())
    assert flag() == 0


@pytest.mark.parametrize("page", [2, 4, 6, 12, 24, 40, 48, 96, 136, 200, 256, 1000])
def test_page_sizes(page, cuda_dev):
    """Chunks that cut pages into groups of 4, 8, 16 and more, of fewer, and pages longer than chunks."""
    check(cuda_dev, [700, 13], [3, 140], page, 4, 2, 64, torch.float16, window=400, sinks=5)
    check(cuda_dev, [530], [7], page, 4, 1, 128, torch.bfloat16, order="head", trees=True)


def test_offsets_beyond_32_bits(cuda_dev):
    """Pools of more than 2^31 values: the same bits as from a small pool."""
    from otf_llm.paged import PagedKVCache
    small, _, table, g = make(cuda_dev, [700], 16, 8, 128, torch.float16, room=[720], fill=0.0)
    small.lengths.fill_(690)
    n = 140000
    big = [torch.empty(n, 16, 8, 128, dtype=torch.float16, device=cuda_dev) for _ in range(2)]
    far = torch.arange(n - 1, n - 1 - 2 * table.shape[1], -2, dtype=torch.int32, device=cuda_dev)[None].contiguous()
    for pool, of in zip(big, (small.k_pages, small.v_pages)):
        for j in range(-(-720 // 16)):
            pool[int(far[0, j])] = of[int(table[0, j])]
    cache = PagedKVCache(big[0], big[1], far, torch.full((1,), 690, dtype=torch.int32, device=cuda_dev))
    q = torch.randn(10, 16, 128, generator=g).half().to(cuda_dev)
    assert same(cache.attend_rows(q, window=500, sinks=20), small.attend_rows(q, window=500, sinks=20))
    parents = torch.tensor([-1, 0, 1, 0, 3, 3, 2, 0, 1, 8], dtype=torch.int32, device=cuda_dev)
    assert same(cache.attend_tree(q, parents), small.attend_tree(q, parents))
    path, accepted = torch.tensor([[1, 8, 9]], dtype=torch.int32, device=cuda_dev), torch.tensor([3], dtype=torch.int32, device=cuda_dev)
    for c in (cache, small):
        c.keep(path, accepted)
        c.lengths.fill_(684)
    assert same(cache.attend_rows(q), small.attend_rows(q)) and flag() == 0


@pytest.mark.parametrize("heads,kv", [(40, 1), (300, 1), (9, 3), (64, 2)])
def test_head_layouts(heads, kv, cuda_dev):
    """Ratios of query to KV heads that no tensor copy of queries takes, and more rows of one token than a block."""
    check(cuda_dev, [150, 3], [2, 9], 16, heads, kv, 64, torch.float16, window=100, sinks=2)
    check(cuda_dev, [90], [5], 16, heads, kv, 64, torch.bfloat16, trees=True)


NAN_KEYS = [
    # cached tokens, new rows, heads, kv, dim, window, sinks, the odd key's place; 32 keys of a chunk at a time for 32 rows
    # and fewer, 64 for 64, one CTA or many
    (96, 1, 4, 1, 128, None, 0, 96), (95, 1, 4, 1, 128, None, 0, 95), (0, 1, 8, 1, 64, None, 0, 0), (32, 1, 1, 1, 64, None, 0, 32),
    (128, 1, 4, 1, 128, None, 0, 128), (256, 1, 4, 2, 64, None, 0, 256), (64, 9, 4, 1, 128, None, 0, 64), (5888, 1, 8, 1, 128, None, 0, 5888),
    (5888, 20, 4, 1, 64, None, 0, 5888), (640, 30, 4, 1, 128, None, 0, 640), (384, 60, 4, 1, 64, None, 0, 384),
    (900, 3, 8, 2, 128, 100, 1, 0), (2000, 9, 8, 1, 64, 33, 1, 0), (700, 40, 4, 1, 128, 64, 1, 0)]


@pytest.mark.parametrize("faint", [False, True])
@pytest.mark.parametrize("length,new,heads,kv,dim,window,sinks,place", NAN_KEYS)
def test_a_nan_key_reaches_every_row_that_sees_it(length, new, heads, kv, dim, window, sinks, place, faint, cuda_dev):
    """Also where it is the only key that a row sees of those that are looked at together, or (faint) where the others
    among them weigh nothing beside the rest."""
    cache, _, table, g = make(cuda_dev, [length + new], 16, kv, dim, torch.float16, room=[length + new + 1], seed=4)
    cache.lengths.fill_(length)
    q = torch.rand(new, heads, dim, generator=g).half() + 1
    q = q.to(cuda_dev)
    if faint:
        for s in range(place // 32 * 32, min(place // 32 * 32 + 32, length + new)):
            cache.k_pages[ref.place(table, 16, 0, s)] = -120.0
    plain = cache.attend_rows(q, window=window, sinks=sinks)
    cache.k_pages[ref.place(table, 16, 0, place)][:, dim // 2] = float("nan")
    got = cache.attend_rows(q, window=window, sinks=sinks)
    assert flag() == 0
    for t in range(new):
        if place in rows.seen(length, t, window, sinks):
            assert bool(got[t].isnan().all()), t
        else:
            assert same(got[t], plain[t]), t


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("lengths,new,heads,kv,dim,window,sinks", [
    ([(61 * b) % 200 + 60 for b in range(48)], [3] * 48, 8, 4, 128, 40, 0),          # whose first keys no row sees, one chunk or two
    ([(61 * b) % 300 for b in range(40)], [1 + 7 * b % 40 for b in range(40)], 16, 8, 64, 70, 3),
    ([(47 * b) % 500 for b in range(30)], [(30, 60, 150, 9)[b % 4] for b in range(30)], 32, 16, 128, 130, 1)])
def test_odd_values_of_one_sequence_leave_all_others(lengths, new, heads, kv, dim, window, sinks, dtype, cuda_dev):
    """Many items on every SM, some of them with infinities among values that not all of their rows see."""
    cache, _, table, g = make(cuda_dev, [n + t for n, t in zip(lengths, new)], 16, kv, dim, TYPES[dtype],
                              room=[n + t + 1 for n, t in zip(lengths, new)], seed=6)
    cache.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    q = torch.randn(sum(new), heads, dim, generator=g).to(TYPES[dtype]).to(cuda_dev)
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(cuda_dev)
    plain = cache.attend_rows(q, starts=starts, window=window, sinks=sinks)
    places = {b: lengths[b] + new[b] // 2 for b in range(0, len(new), 3)}
    at = {b: ref.place(table, 16, b, s) for b, s in places.items()}
    for b, (page, place) in at.items():
        cache.v_pages[page, place, b % kv, b % dim] = float("inf")
    calls = [cache.attend_rows(q, starts=starts, window=window, sinks=sinks) for _ in range(4)]
    assert flag() == 0
    want_odd = torch.zeros_like(plain, dtype=torch.bool)
    rep = heads // kv
    for b, s in places.items():
        for t in range(new[b]):
            if s in rows.seen(lengths[b], t, window, sinks):
                want_odd[int(starts[b]) + t, b % kv * rep:(b % kv + 1) * rep, b % dim] = True
    for got in calls:
        assert torch.equal(~got.isfinite(), want_odd)
        assert same(torch.where(want_odd, 0, got), torch.where(want_odd, 0, plain))


def test_a_live_sequence_without_nodes_in_a_step(cuda_dev):
    """As many places as tokens came out are counted: a sequence that has no nodes in a step, or nothing to draw from, keeps
    its length, and what it attends afterwards."""
    from otf_llm.speculative import verify_tree
    cache, _, table, g = make(cuda_dev, [40, 33, 50], 16, 2, 64, torch.float16, room=[60, 60, 60], seed=12)
    cache.lengths.copy_(torch.tensor([36, 32, 45], dtype=torch.int32))
    q = torch.randn(3, 4, 64, generator=g).half().to(cuda_dev)
    before = cache.attend_rows(q)
    starts = torch.tensor([0, 3, 3, 7], dtype=torch.int32, device=cuda_dev)
    parents = torch.tensor([-1, 0, 1, -1, 0, 0, 1], dtype=torch.int32, device=cuda_dev)
    target = torch.zeros(7, 9, device=cuda_dev)
    target[0, 4] = target[1, 5] = 1.0
    target[3] = -float("inf")
    ids = torch.tensor([0, 4, 7, 0, 1, 2, 3], device=cuda_dev)
    tokens, path, accepted = verify_tree(target, ids, parents, starts=starts, depth=2, temperature=0.0)
    assert flag() == 1                                  # the last sequence has nothing to draw from
    assert tokens.tolist() == [[4, 5, -1], [-1] * 3, [-1] * 3] and accepted.tolist() == [1, 0, 0]
    cache.keep(path, accepted)
    cache.advance((tokens >= 0).sum(1, dtype=torch.int32))
    assert cache.lengths.tolist() == [38, 32, 45] and flag() == 0
    after = cache.attend_rows(q)
    assert same(after[1:], before[1:]) and not same(after[0], before[0])
