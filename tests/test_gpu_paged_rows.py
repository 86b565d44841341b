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
