"""The walk through trees of drafted tokens and the moving of the taken nodes, against 64 bits."""
import math

import pytest
import torch

import rows_oracle as ref
from test_gpu_paged import TYPES, flag, make, same

pytestmark = pytest.mark.gpu


def trees(new, vocab, depth, seed, likely=True):
    """Trees whose children hold the likeliest tokens behind their parents, and noise."""
    g = torch.Generator().manual_seed(seed)
    n = sum(new)
    target = torch.randn(n, vocab, generator=g) * 2
    target.scatter_add_(1, torch.randint(0, vocab, (n, 3), generator=g), torch.rand(n, 3, generator=g) * 4 + 5)
    order = target.argsort(dim=1, descending=True)
    parents, tokens, at = [], [], 0
    for m in new:
        up = [-1] + [int(torch.randint(max(0, i - 4), i, (), generator=g)) for i in range(1, m)]
        count = [0] * m
        for i, p in enumerate(up):
            tokens.append(int(order[at + p, count[p] % vocab]) if p >= 0 else 0)
            if p >= 0:
                count[p] += 1
        parents.append(up)
        at += m
    noise = torch.empty(len(new), depth + 1, vocab).exponential_(generator=g)
    return target, torch.tensor(tokens), parents, noise


def run(dev, target, tokens, parents, new, depth, noise, temperature, uniform=False, **other):
    from otf_llm.speculative import verify_tree
    flat = torch.tensor([p for up in parents for p in up], dtype=torch.int32, device=dev)
    starts = None if uniform else torch.tensor([0] + new).cumsum(0).to(torch.int32).to(dev)
    t = temperature if isinstance(temperature, float) else torch.tensor(temperature, device=dev)
    return verify_tree(target.to(dev), tokens.to(dev), flat, starts=starts, batch=len(new) if uniform else None, depth=depth,
                       noise=None if noise is None else noise.to(dev), temperature=t, **other)


def check(dev, new, vocab, depth, temperature, seed=1, uniform=False):
    target, tokens, parents, noise = trees(new, vocab, depth, seed)
    out, path, accepted = run(dev, target, tokens, parents, new, depth, noise, temperature, uniform)
    assert flag() == 0
    at = 0
    for b, m in enumerate(new):
        T = temperature if isinstance(temperature, float) else float(torch.tensor(temperature[b]))
        drawn, way, taken = ref.walk(target[at:at + m], tokens[at:at + m], parents[b], noise[b], T, depth)
        assert out[b].tolist() == drawn + [-1] * (depth + 1 - len(drawn)), b
        assert path[b].tolist() == way + [-1] * (depth - taken) and int(accepted[b]) == taken, b
        at += m
    return accepted


@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0])
@pytest.mark.parametrize("new,vocab,depth", [([1], 1, 0), ([1, 5], 7, 3), ([26], 1003, 5), ([64, 1, 33], 5000, 8),
                                             ([40] * 5, 32000, 6), ([64], 130, 63)])
def test_walk_matches_definition(new, vocab, depth, temperature, cuda_dev):
    check(cuda_dev, new, vocab, depth, temperature)


def test_walks_of_many_sequences_go_down(cuda_dev):
    """Several CTAs a sequence, one a sequence; uniform trees; and the greedy walks take their likeliest children."""
    taken = check(cuda_dev, [20] * 40, 900, 5, 0.0, seed=3, uniform=True)
    assert int(taken.max()) >= 3
    check(cuda_dev, [(7 * b) % 20 + 1 for b in range(600)], 64, 4, 0.8, seed=4)
    check(cuda_dev, [9, 12, 3], 2000, 4, [0.0, 0.9, 1.4], seed=5)
    # more logits than are looked at at once: clusters of several sizes, unaligned rows
    check(cuda_dev, [40, 3, 64], 140001, 4, 0.9, seed=6)
    check(cuda_dev, [30] * 90, 6003, 3, [0.0, 1.1, 0.7] * 30, seed=7)
    check(cuda_dev, [25] * 700, 1001, 2, 0.8, seed=8)


def test_the_first_of_equal_children_and_of_equal_logits(cuda_dev):
    target = torch.zeros(5, 40)
    target[0, 9] = target[0, 30] = 4.0
    target[2, 5] = 1.0
    out, path, accepted = run(cuda_dev, target, torch.tensor([0, 30, 9, 9, 5]), [[-1, 0, 0, 0, 2]], [5], 4, None, 0.0)
    assert out.tolist() == [[9, 5, 0, -1, -1]] and path.tolist() == [[2, 4, -1, -1]] and accepted.tolist() == [2]


def test_odd_logits_and_noise(cuda_dev):
    """Masked entries are never drawn, however small their noise; NaN as -inf; noise of 0 wins, the first of several."""
    inf, nan = math.inf, math.nan
    target, tokens, parents, noise = trees([4, 4, 4, 4], 600, 2, 8)
    target[0, 10:] = -inf
    noise[0, 0, 300] = 0.0
    target[4, :500] = nan
    target[8, 7] = target[8, 400] = inf
    noise[3, 0, 123] = noise[3, 0, 77] = 0.0
    out, _, _ = run(cuda_dev, target, tokens, parents, [4] * 4, 2, noise, 0.8)
    assert flag() == 0
    first = out[:, 0].tolist()
    assert first[0] < 10 and first[1] >= 500 and first[3] == 77
    assert first[2] == (7 if float(noise[2, 0, 7]) < float(noise[2, 0, 400]) else 400) or first[2] == 7
    low = torch.full((1, 300), torch.finfo(torch.float32).min)
    low[0, 200] = 0.0
    for T in (1e-20, 1e-3, 1e20):
        n = torch.ones(1, 1, 300)
        out, _, _ = run(cuda_dev, low, torch.zeros(1, dtype=torch.int64), [[-1]], [1], 0, n, T)
        assert out.tolist() == [[200]]
    assert flag() == 0


def test_close_races_are_decided_in_64_bits(cuda_dev):
    """Scores that fp32 cannot tell apart: the larger one by 2^-40 wins, wherever it lies."""
    vocab = 4000
    for seed in range(6):
        g = torch.Generator().manual_seed(seed)
        target = torch.full((1, vocab), 20.0)
        noise = torch.full((1, 1, vocab), 1.0) + torch.rand(1, 1, vocab, generator=g) * 2.0 ** -18
        want = int((20.0 - noise.double().log())[0, 0].argmax())
        out, _, _ = run(cuda_dev, target, torch.zeros(1, dtype=torch.int64), [[-1]], [1], 0, noise, 1.0)
        assert int(out[0, 0]) == want


def test_sequences_that_cannot_be_walked(cuda_dev):
    target, tokens, parents, noise = trees([3, 3, 3], 50, 2, 2)
    target[3] = -math.inf
    out, path, accepted = run(cuda_dev, target, tokens, parents, [3] * 3, 2, noise, [0.5, 0.5, -1.0])
    assert flag() == 1
    assert int(out[0, 0]) >= 0 and out[1:].eq(-1).all() and path[1:].eq(-1).all() and accepted[1:].eq(0).all()
    bad = [[-1, 1, 0], [-1, 0, -5], [-1, 0, 2]]
    run(cuda_dev, target.clamp(min=-5), tokens, bad, [3] * 3, 2, noise, 0.5)
    assert flag() == 1
    # none is no mistake: a place of the batch without a sequence
    out, path, accepted = run(cuda_dev, target.clamp(min=-5)[:6], tokens[:6], [[-1, 0, 1], [], [-1, 0, 0]], [3, 0, 3], 2, noise, 0.5)
    assert flag() == 0 and out[1].eq(-1).all() and path[1].eq(-1).all() and int(accepted[1]) == 0 and out[::2, 0].ge(0).all()
    # 65 nodes, and rows that lie outside
    target, tokens, parents, noise = trees([65, 1], 50, 2, 2)
    out, _, accepted = run(cuda_dev, target, tokens, parents, [65, 1], 2, noise, 0.0)
    assert flag() == 1 and out[0].eq(-1).all() and int(out[1, 0]) == int(target[65].argmax())
    out, _, _ = run(cuda_dev, target, tokens, parents, [2, 65], 2, noise, 0.0)
    assert flag() == 1 and out[1].eq(-1).all()


# ---- keep -------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,order", [("fp16", "token"), ("bf16", "head")])
@pytest.mark.parametrize("lengths,page,kv,dim,paths", [
    ([0], 16, 1, 64, [[3]]), ([5, 0, -1, 33], 16, 2, 128, [[1, 2, 9], [], [4], [2, 3, 4, 40]]),
    ([15, 14], 16, 3, 64, [[2, 17, 18], [5, 1, 3]]), ([7], 1, 8, 128, [list(range(1, 64))]),
    ([100, 3], 20, 2, 64, [list(range(63, 0, -1)), [10]])])
def test_keep_moves_the_taken_nodes(lengths, page, kv, dim, paths, dtype, order, cuda_dev):
    cache, pools, table, _ = make(cuda_dev, [n + 64 if n >= 0 else n for n in lengths], page, kv, dim, TYPES[dtype], order)
    cache.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    depth = max(len(p) for p in paths)
    path = torch.tensor([p + [-1] * (depth - len(p)) for p in paths], dtype=torch.int32)
    want = [p.clone() for p in pools]
    for b, (n, way) in enumerate(zip(lengths, paths)):
        if n >= 0:
            for j, i in enumerate(way):
                a, z = (n + i) // page, (n + 1 + j) // page
                for w, pool in zip(want, pools):
                    w[int(table[b, z]), (n + 1 + j) % page] = pool[int(table[b, a]), (n + i) % page]
    cache.keep(path.to(cuda_dev), torch.tensor([len(p) for p in paths], dtype=torch.int32, device=cuda_dev))
    assert flag() == 0
    assert same(cache.k_pages.cpu(), want[0]) and same(cache.v_pages.cpu(), want[1])
    assert cache.lengths.tolist() == lengths


def test_keep_leaves_out_what_does_not_fit(cuda_dev):
    cache, pools, table, _ = make(cuda_dev, [20, 20], 16, 1, 64, torch.float16, room=[20, 20])
    before = [cache.k_pages.clone(), cache.v_pages.clone()]
    for way, count in (([[-1], [2]], [1, 0]), ([[70], [1]], [1, 2]), ([[1], [1]], [-1, -4])):
        cache.lengths.copy_(torch.tensor([10, 10], dtype=torch.int32))
        cache.keep(torch.tensor(way, dtype=torch.int32, device=cuda_dev), torch.tensor(count, dtype=torch.int32, device=cuda_dev))
        assert flag() == 1
        assert same(cache.k_pages, before[0]) and same(cache.v_pages, before[1])


@pytest.mark.parametrize("temperature", [0.0, 0.8])
@pytest.mark.parametrize("vocab", [700, 200000])
def test_a_sequence_beside_starts_that_fall(vocab, temperature, cuda_dev):
    """A sequence whose rows are in order gets its tokens whatever the starts beside it are, few logits or many; also where
    two sequences have the same rows."""
    from otf_llm.speculative import verify_tree
    depth = 3
    target, tokens, parents, _ = trees([7, 6, 64], vocab, depth, 5)
    flat = torch.tensor([p for up in parents for p in up], dtype=torch.int32)
    noise = torch.empty(5, depth + 1, vocab).exponential_(generator=torch.Generator().manual_seed(6))

    def want(b, r0, r1):
        up = [int(p) for p in flat[r0:r1]]
        drawn, way, taken = ref.walk(target[r0:r1], tokens[r0:r1], up, noise[b], temperature, depth)
        return drawn + [-1] * (depth + 1 - len(drawn)), way + [-1] * (depth - taken), taken
    dev = [t.to(cuda_dev) for t in (target, tokens, flat, noise)]
    for starts, good in (([0, 7, 3, 3, 3, 3], {0: (0, 7)}), ([7, 13, 7, 13, 13, 13], {0: (7, 13), 2: (7, 13)}),
                         ([0, 7, 0, 7, 13, 77], {0: (0, 7), 2: (0, 7), 3: (7, 13), 4: (13, 77)}),
                         ([90, 0, 7, -5, 7, 13], {1: (0, 7), 4: (7, 13)})):
        for _ in range(2):                              # the second time over what the first one left in the scratch
            out, path, accepted = verify_tree(dev[0], dev[1], dev[2], starts=torch.tensor(starts, dtype=torch.int32, device=cuda_dev),
                                              depth=depth, noise=dev[3], temperature=temperature)
        assert flag() == 1
        for b in range(5):
            expect = want(b, *good[b]) if b in good else ([-1] * (depth + 1), [-1] * depth, 0)
            assert (out[b].tolist(), path[b].tolist(), int(accepted[b])) == expect, (starts, b)
    # the first sequence with the rows has no temperature to be walked at
    temps = torch.tensor([-1.0, 1.0, temperature, 1.0, 1.0], device=cuda_dev)
    for _ in range(2):
        out, _, accepted = verify_tree(dev[0], dev[1], dev[2], starts=torch.tensor([7, 13, 7, 13, 13, 13], dtype=torch.int32, device=cuda_dev),
                                       depth=depth, noise=dev[3], temperature=temps)
        assert flag() == 1 and out[:2].eq(-1).all() and (out[2].tolist(), int(accepted[2])) == (want(2, 7, 13)[0], want(2, 7, 13)[2])
