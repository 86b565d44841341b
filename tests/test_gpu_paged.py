"""The paged key/value cache against its definitions in 64 bits: append with rotary positions,
attention of one or a few new tokens, eviction, and all of them together."""
import math

import pytest
import torch

import paged_oracle as ref

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def make(dev, lengths, page, kv, dim, dtype, order="token", room=None, seed=0, spare=2, fill=float("nan")):
    """A cache whose pages hold `fill` but for the tokens there are, under a shuffled table with
    entries that name no page behind each sequence's room."""
    from otf_llm.paged import PagedKVCache
    g = torch.Generator().manual_seed(seed)
    room = room or [max(n, 1) for n in lengths]
    need = [-(-r // page) for r in room]
    n_pages, most = sum(need) + spare, max(need) + 1
    shape = (n_pages, page, kv, dim) if order == "token" else (n_pages, kv, page, dim)
    pools = [torch.full(shape, fill, dtype=dtype) for _ in range(2)]
    if order == "head":
        pools = [p.transpose(1, 2) for p in pools]
    ids = torch.randperm(n_pages, generator=g).tolist()
    table = torch.full((len(lengths), most), -7, dtype=torch.int32)
    for b, n in enumerate(need):
        for j in range(n):
            table[b, j] = ids.pop()
    for b, n in enumerate(lengths):
        for s in range(max(n, 0)):
            for pool in pools:
                pool[ref.place(table, page, b, s)] = torch.randn(kv, dim, generator=g).to(dtype)
    on = [p.to(dev) if order == "token" else p.transpose(1, 2).contiguous().to(dev).transpose(1, 2) for p in pools]
    cache = PagedKVCache(on[0], on[1], table.to(dev), torch.tensor(lengths, dtype=torch.int32, device=dev))
    return cache, pools, table, g


def flag():
    from otf_llm import _native
    torch.cuda.synchronize()
    return _native.device_error(clear=True)


def same(a, b):
    """Equal bits, NaN included."""
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


# ---- append -----------------------------------------------------------------------------------


def check_append(cuda_dev, lengths, new, page, heads, kv, dim, rot, interleaved, scaling, dtype, order, uniform,
                 positions=None, in_place=False, extra=0, seed=1):
    from otf_llm.paged import Rotary
    cache, pools, table, g = make(cuda_dev, lengths, page, kv, dim, dtype, order, seed=seed,
                                  room=[max(n, 0) + t + 1 for n, t in zip(lengths, new)])
    n = sum(new)
    qkv = torch.randn(n + extra, heads + 2 * kv, dim, generator=g).to(dtype)
    dq = qkv.to(cuda_dev)
    q, k, v = dq.split([heads, kv, kv], dim=1)
    rotary = Rotary(dim, rot_dim=rot, theta=10000.0, scaling=scaling, interleaved=interleaved, device=cuda_dev)
    starts = None if uniform else torch.tensor([0] + new).cumsum(0).to(torch.int32).to(cuda_dev)
    pos = None if positions is None else torch.tensor(positions, dtype=torch.int32, device=cuda_dev)
    out = q if in_place else torch.full((n + extra, heads, dim), 7.0, dtype=dtype, device=cuda_dev)
    got = cache.append(q, k, v, rotary, starts=starts, positions=pos, q_out=out)
    assert got is out and flag() == 0
    want_q = (qkv[:, :heads] if in_place else torch.full((n + extra, heads, dim), 7.0)).double()
    tol_q = torch.zeros_like(want_q)
    want_k, want_v = pools[0].clone(), pools[1].clone()
    row, u = 0, torch.finfo(dtype).eps / 2
    f, factor = rotary.frequencies, rotary.factor
    k_got, v_got = cache.k_pages.cpu(), cache.v_pages.cpu()
    for b, t in enumerate(new):
        for j in range(t):
            if lengths[b] >= 0:
                s = lengths[b] + j
                p = positions[row] if positions is not None else s
                at = ref.place(table, page, b, s)
                # c and s within 2^-21 (the angle's last bit of a turn, and sincospi's), two
                # products and a sum in fp32, one rounding
                for x, want, tol in ((qkv[row, :heads], want_q[row], tol_q[row]), (qkv[row, heads:heads + kv], None, None)):
                    y = ref.rotate(x, p, f, factor, rot, interleaved)
                    most = u * y.abs() + 2.0 ** -20 * factor * x.double().abs().amax() + torch.finfo(dtype).tiny * u
                    if want is not None:
                        want.copy_(y)
                        tol.copy_(most)
                        if rot < dim:
                            tol[:, rot:] = 0
                    else:
                        if rot < dim:
                            most[:, rot:] = 0
                        assert bool(((k_got[at].double() - y).abs() <= most).all()), (b, j)
                        want_k[at] = k_got[at]
                want_v[at] = qkv[row, heads + kv:]
            row += 1
    assert bool(((out.cpu().double() - want_q).abs() <= tol_q).all())
    assert same(k_got, want_k) and same(v_got, want_v)      # nothing else was written


APPEND = [
    ([0], [1], 16, 1, 1, 64, 64, False, "none"),
    ([5, 0, -1, 33], [1, 1, 1, 1], 16, 8, 2, 128, 128, False, "none"),
    ([0, 7, 100], [9, 0, 40], 20, 6, 2, 64, 32, True, "linear"),
    ([3, 0], [17, 5], 1, 28, 4, 128, 24, False, "yarn"),
    ([250, 1], [3, 30], 3, 5, 5, 128, 128, True, "llama3"),
    ([15, 16], [2, 2], 8, 64, 8, 64, 0, False, "none"),
    ([2, 9, -3, 40], [4, 6, 2, 3], 128, 16, 1, 128, 10, True, "none"),
    ([1], [70], 64, 32, 32, 64, 6, False, "linear"),
]
SCALING = {"none": None, "linear": {"rope_type": "linear", "factor": 4.0},
           "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                      "original_max_position_embeddings": 64},
           "yarn": {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 128}}


@pytest.mark.parametrize("dtype,order", [("fp16", "token"), ("bf16", "head")])
@pytest.mark.parametrize("lengths,new,page,heads,kv,dim,rot,interleaved,scaling", APPEND)
def test_append_matches_definition(lengths, new, page, heads, kv, dim, rot, interleaved, scaling, dtype, order, cuda_dev):
    check_append(cuda_dev, lengths, new, page, heads, kv, dim, rot, interleaved, SCALING[scaling], TYPES[dtype], order,
                 uniform=False, extra=2)


def test_append_uniform_rows_in_place_and_given_positions(cuda_dev):
    check_append(cuda_dev, [4, 0, 19], [3, 3, 3], 16, 8, 2, 128, 64, False, None, torch.float16, "token", uniform=True,
                 in_place=True)
    check_append(cuda_dev, [4, 0, 19], [1, 1, 1], 16, 8, 2, 64, 64, True, None, torch.bfloat16, "token", uniform=True,
                 positions=[1000003, -5, 2 ** 31 - 1])


def test_append_many_sequences(cuda_dev):
    lengths = [(7 * b) % 23 for b in range(75)]
    check_append(cuda_dev, lengths, [b % 3 for b in range(75)], 8, 2, 1, 64, 64, False, None, torch.float16, "token",
                 uniform=False, extra=1)


def test_append_keys_and_values_alone_and_nothing_turned(cuda_dev):
    cache, pools, table, g = make(cuda_dev, [3, 0], 4, 2, 64, torch.float16, room=[8, 8])
    k, v = torch.randn(4, 2, 64, generator=g).half(), torch.randn(4, 2, 64, generator=g).half()
    assert cache.append(None, k.to(cuda_dev), v.to(cuda_dev)) is None
    kp, vp = cache.k_pages.cpu(), cache.v_pages.cpu()
    for row, (b, s) in enumerate(((0, 3), (0, 4), (1, 0), (1, 1))):
        at = ref.place(table, 4, b, s)
        assert torch.equal(kp[at], k[row]) and torch.equal(vp[at], v[row])
    assert flag() == 0
    assert cache.append(None, k[:0].to(cuda_dev), v[:0].to(cuda_dev)) is None


def test_append_leaves_out_what_has_no_place(cuda_dev):
    from otf_llm.paged import Rotary
    cache, pools, table, g = make(cuda_dev, [2, 30, 5], 16, 2, 64, torch.float16, room=[16, 32, 16])
    cache.page_table[2, 0] = 10 ** 6                       # a page outside the pool
    q, k, v = (torch.randn(9, h, 64, generator=g).half().to(cuda_dev) for h in (4, 2, 2))
    before = cache.k_pages.clone()
    cap = cache.capacity
    cache.lengths[1] = cap - 1                             # its second and third token do not fit
    cache.page_table[1] = int(table[1, 0])
    out = torch.full_like(q, 7.0)
    cache.append(q, k, v, Rotary(64, device=cuda_dev), q_out=out)
    assert flag() == 1
    assert not bool((out[:4] == 7.0).any()) and bool((out[4:] == 7.0).all())
    changed = (cache.k_pages.cpu().view(torch.int16) != before.cpu().view(torch.int16)).any(-1).any(-1)
    assert changed.nonzero().tolist() == sorted([[int(table[0, 0]), 2], [int(table[0, 0]), 3], [int(table[0, 0]), 4],
                                                 [int(table[1, 0]), (cap - 1) % 16]])


# ---- attend -----------------------------------------------------------------------------------


def check_attend(cuda_dev, totals, tokens, page, heads, kv, dim, dtype, order="token", weights=False, scale=None, seed=2,
                 spread=1.0, prepare=None):
    cache, pools, table, g = make(cuda_dev, totals, page, kv, dim, dtype, order, seed=seed)
    if prepare is not None:
        prepare(cache, pools, table)
    cache.lengths.copy_(torch.tensor([n - tokens if n > 0 else -1 for n in totals], dtype=torch.int32))
    q = (torch.randn(len(totals), tokens, heads, dim, generator=g) * spread).to(dtype)
    out = torch.full((len(totals), tokens, heads, dim), 7.0, dtype=dtype, device=cuda_dev)
    w0 = w = None
    if weights:
        w0 = torch.rand(len(totals), kv, cache.capacity, generator=g)
        w = w0.to(cuda_dev)
    got = cache.attend(q.to(cuda_dev), weights=w, out=out, scale=scale)
    assert got is out and flag() == 0
    out = out.cpu().double()
    want_w = w0.double() if weights else None
    tol_w = want_w * 2.0 ** -22 if weights else None
    for b, n in enumerate(totals):
        if n <= 0:
            assert bool((out[b] == 7.0).all())
            continue
        k, v = (ref.gather(p, table, b, n) for p in pools)
        for t in range(tokens):
            m = n - tokens + t + 1
            y, p, mass, size = ref.attend(q[b, t], k[:m], v[:m], dim ** -0.5 if scale is None else scale)
            tol = ref.attend_tolerance(y, mass, size, dim, dtype)
            off = (out[b, t] - y).abs() - tol
            assert bool((off <= 0).all()), (b, t, float(off.max()), float((out[b, t] - y).abs().max()))
            if weights:
                rep = heads // kv
                want_w[b, :, :m] += p.view(kv, rep, m).sum(1)
                tol_w[b, :, :m] += (p * (size * 2.0 ** -14 + 2.0 ** -18)).view(kv, rep, m).sum(1) + 2.0 ** -40
    if weights:
        off = (w.cpu().double() - want_w).abs() - tol_w
        assert bool((off <= 0).all()), float(off.max())
    return cache, q


ATTEND = [
    ([1], 1, 16, 1, 1, 64),
    ([1, 2, 15, 16, 17, 31, 32, 33], 1, 16, 8, 2, 128),
    ([700], 1, 16, 32, 8, 128),
    ([0, 300, 0, 5], 1, 20, 6, 2, 64),
    ([129, 127, 128, 64, 65], 1, 1, 28, 4, 128),
    ([513, 40], 1, 3, 48, 1, 64),
    ([260, 7], 1, 128, 16, 16, 128),
    ([5, 6, 64, 200], 5, 16, 8, 2, 128),
    ([16, 17, 200], 16, 20, 4, 4, 64),
    ([300, 8], 8, 16, 64, 8, 128),
    ([2, 90], 2, 8, 40, 8, 64),
    ([1100, 3], 3, 64, 71, 1, 128),
]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("dtype,order", [("fp16", "token"), ("bf16", "head")])
@pytest.mark.parametrize("totals,tokens,page,heads,kv,dim", ATTEND)
def test_attend_matches_definition(totals, tokens, page, heads, kv, dim, dtype, order, weights, cuda_dev):
    check_attend(cuda_dev, totals, tokens, page, heads, kv, dim, TYPES[dtype], order, weights)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attend_peaked_and_flat_scores(dtype, cuda_dev):
    check_attend(cuda_dev, [500, 33], 1, 16, 8, 2, 128, TYPES[dtype], spread=30.0)      # one key takes nearly all
    check_attend(cuda_dev, [3000], 2, 16, 8, 2, 64, TYPES[dtype], spread=0.0, weights=True)  # all equal
    check_attend(cuda_dev, [90], 1, 16, 8, 2, 128, TYPES[dtype], scale=-0.3)
    check_attend(cuda_dev, [90, 9], 3, 16, 8, 2, 64, TYPES[dtype], scale=0.0, weights=True)


def test_attend_many_sequences_and_long_ones(cuda_dev):
    check_attend(cuda_dev, [1 + (37 * b) % 90 for b in range(150)], 1, 16, 4, 2, 64, torch.float16)
    check_attend(cuda_dev, [9000, 1, 40], 1, 64, 4, 1, 64, torch.float16, weights=True)
    # runs that cross short, long and missing sequences
    check_attend(cuda_dev, [(1 + (97 * b) % 701) * (b % 11 != 5) for b in range(70)], 1, 16, 4, 2, 64, torch.bfloat16,
                 weights=True)
    check_attend(cuda_dev, [3 + (61 * b) % 400 for b in range(40)], 3, 20, 12, 2, 64, torch.float16, "head", weights=True)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attend_rows_do_not_see_later_tokens(bad, dtype, cuda_dev):
    """The newest tokens hold `bad`: rows before them stay finite and right, rows that see them do not."""
    for totals, tokens, page, heads, kv, dim in (([40, 5, 129], 4, 16, 6, 2, 64), ([33, 7, 66, 400], 5, 20, 28, 4, 128),
                                                 ([64, 80, 17], 16, 16, 4, 4, 128), ([40, 31], 8, 8, 32, 2, 64)):
        check_later_tokens(bad, TYPES[dtype], cuda_dev, totals, tokens, page, heads, kv, dim)


def check_later_tokens(bad, dt, cuda_dev, totals, tokens, page, heads, kv, dim):
    cache, pools, table, g = make(cuda_dev, totals, page, kv, dim, dt)
    for b, n in enumerate(totals):
        for pool, on in zip(pools, (cache.k_pages, cache.v_pages)):
            for s in (n - 2, n - 1):
                pool[ref.place(table, page, b, s)] = bad
                on[ref.place(table, page, b, s)] = bad
    cache.lengths.sub_(tokens)
    q = torch.randn(len(totals), tokens, heads, dim, generator=g).to(dt)
    w = torch.zeros(len(totals), kv, cache.capacity, device=cuda_dev)
    out = cache.attend(q.to(cuda_dev), weights=w).cpu().double()
    for b, n in enumerate(totals):
        k, v = (ref.gather(p, table, b, n) for p in pools)
        for t in range(tokens - 2):
            m = n - tokens + t + 1
            y, p, mass, size = ref.attend(q[b, t], k[:m], v[:m], dim ** -0.5)
            assert bool(((out[b, t] - y).abs() <= ref.attend_tolerance(y, mass, size, dim, dt)).all())
        finite = bool(torch.isfinite(out[b, tokens - 1]).all())
        assert not finite


def test_attend_reads_bad_pages_as_zeros_and_raises_the_flag(cuda_dev):
    cache, pools, table, g = make(cuda_dev, [40, 20], 16, 2, 64, torch.float16)
    cache.page_table[0, 1] = -1
    cache.lengths.sub_(1)
    q = torch.randn(2, 4, 64, generator=g).half()
    out = cache.attend(q.to(cuda_dev)).cpu().double()
    assert flag() == 1
    k, v = (ref.gather(p, torch.where(table < 0, 0, table), 0, 40) for p in pools)
    k[16:32], v[16:32] = 0, 0
    y, p, mass, size = ref.attend(q[0], k, v, 0.125)
    assert bool(((out[0] - y).abs() <= ref.attend_tolerance(y, mass, size, 64, torch.float16)).all())
    # a sequence longer than its table is left out whole, the other one is not
    cache.page_table.copy_(table)
    cache.lengths[0] = cache.capacity
    out = torch.full_like(q, 7.0).to(cuda_dev)
    cache.attend(q.to(cuda_dev), out=out)
    assert flag() == 1
    assert bool((out[0] == 7.0).all()) and not bool((out[1] == 7.0).any())


def test_attend_without_any_sequence(cuda_dev):
    cache, pools, table, g = make(cuda_dev, [-1, -5, -1], 16, 2, 64, torch.float16, room=[300, 16, 16])
    q = torch.randn(3, 4, 64, generator=g).half().to(cuda_dev)
    out, w = torch.full_like(q, 7.0), torch.zeros(3, 2, cache.capacity, device=cuda_dev)
    cache.attend(q, out=out, weights=w)
    cache.append(q, q[:, :2], q[:, :2], q_out=out)
    assert flag() == 0 and bool((out == 7.0).all()) and not bool(w.any())


def test_refusals_of_the_python_surface(cuda_dev):
    from otf_llm.paged import PagedKVCache, Rotary
    cache, pools, table, g = make(cuda_dev, [20, 30], 16, 2, 64, torch.float16)
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device=cuda_dev)
    kv = q[:, :2]
    w = torch.zeros(2, 2, cache.capacity, device=cuda_dev)
    bad = [lambda: cache.attend(q.bfloat16()), lambda: cache.attend(q.cpu()), lambda: cache.attend(q[:1]),
           lambda: cache.attend(q[:, :3]), lambda: cache.attend(q[..., :32]), lambda: cache.attend(q.transpose(0, 1)),
           lambda: cache.attend(q.new_zeros(2, 17, 4, 64)), lambda: cache.attend(q, out=q),
           lambda: cache.attend(q, out=q.new_zeros(2, 8, 64)), lambda: cache.attend(q, weights=w[..., :-1]),
           lambda: cache.attend(q, weights=w.half()), lambda: cache.attend(q.new_zeros(4, 4, 64)[::2][:, ::2]),
           lambda: cache.append(q, kv, kv[:1]), lambda: cache.append(q[:1], kv, kv), lambda: cache.append(q, q, kv),
           lambda: cache.append(q, kv[:1], kv[:1]), lambda: cache.append(None, kv[:1], kv[:1]),
           lambda: cache.append(None, kv, kv, q_out=q), lambda: cache.append(q, kv, kv, Rotary(128, device=cuda_dev)),
           lambda: cache.append(q, kv, kv, Rotary(64, device="cpu")),
           lambda: cache.append(q, kv, kv, starts=torch.zeros(3, dtype=torch.int64, device=cuda_dev)),
           lambda: cache.append(q, kv, kv, starts=torch.zeros(2, dtype=torch.int32, device=cuda_dev)),
           lambda: cache.append(q, kv, kv, positions=torch.zeros(3, dtype=torch.int32, device=cuda_dev)),
           lambda: cache.evict(w, 0, 0), lambda: cache.evict(w, 8, 9), lambda: cache.evict(w, cache.capacity + 1, 0),
           lambda: cache.evict(w[..., :-1].contiguous(), 8, 2), lambda: cache.evict(w, 8, 2, weights_out=w.clone()),
           lambda: cache.evict(w, 8, 2, to=cache, weights_out=w.clone()), lambda: cache.evict(w, 8, 2, to=cache),
           lambda: Rotary(64, rot_dim=66), lambda: Rotary(64, rot_dim=7),
           lambda: PagedKVCache(cache.k_pages, cache.v_pages, cache.page_table.long(), cache.lengths),
           lambda: PagedKVCache(cache.k_pages, cache.v_pages, cache.page_table, cache.lengths[:1]),
           lambda: PagedKVCache(cache.k_pages, cache.v_pages[:, :8], cache.page_table, cache.lengths),
           lambda: PagedKVCache(cache.k_pages.float(), cache.v_pages.float(), cache.page_table, cache.lengths),
           lambda: PagedKVCache(cache.k_pages[..., :32], cache.v_pages[..., :32], cache.page_table, cache.lengths)]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()
            pytest.fail(f"refusal {i}")
    with pytest.raises(AttributeError):
        cache.lengths = cache.lengths + 1
    assert flag() == 0


FIRST_IN_CAPTURE = """
import torch
from otf_llm.paged import PagedKVCache, Rotary
from otf_llm.speculative import verify_drafts
dev = torch.device("cuda:0")
table = torch.arange(80, dtype=torch.int32, device=dev).view(2, 40)
cache = PagedKVCache.allocate(80, 16, 2, 64, table, torch.zeros(2, dtype=torch.int32, device=dev))
rotary = Rotary(64, device=dev)
q = torch.randn(2, 4, 64, device=dev).half()
w = torch.zeros(2, 2, cache.capacity, device=dev)
logits = torch.randn(2, 3, 500, device=dev)
tokens = logits[:, :2].argmax(2)
uniforms, noise = torch.rand(2, 2, device=dev), torch.empty(2, 500, device=dev).exponential_()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    t = cache.append(q, q[:, :2], q[:, 2:], rotary)
    out = cache.attend(t, weights=w)
    cache.advance()
    cache.evict(w, 8, 2)
    got = verify_drafts(logits, tokens, uniforms=uniforms, noise=noise)
for _ in range(12):
    g.replay()
torch.cuda.synchronize()
assert cache.lengths.tolist() == [8, 8] and torch.isfinite(out).all()
assert torch.allclose(out[:, :2], q[:, 2:3].expand(2, 2, 64), atol=1e-2)      # one value in every place
want = verify_drafts(logits, tokens, uniforms=uniforms, noise=noise)
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("captured")
"""


def test_first_call_of_a_process_may_be_captured(cuda_dev):
    import os
    import subprocess
    import sys

    from conftest import PKG
    env = dict(os.environ, PYTHONPATH=PKG + os.pathsep + os.environ.get("PYTHONPATH", ""))
    r = subprocess.run([sys.executable, "-c", FIRST_IN_CAPTURE], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_attend_strided_queries_and_outputs(cuda_dev):
    cache, pools, table, g = make(cuda_dev, [33, 50], 16, 2, 64, torch.float16)
    cache.lengths.sub_(3)
    wide = torch.randn(2, 3, 12, 64, generator=g).half().to(cuda_dev)
    q = wide[:, :, 2:10]
    room = torch.zeros(2, 3, 16, 64, dtype=torch.float16, device=cuda_dev)
    out = cache.attend(q, out=room[:, :, 4:12])
    assert torch.equal(out, cache.attend(q.contiguous()))
    assert not bool(room[:, :, :4].any()) and not bool(room[:, :, 12:].any())


def test_offsets_beyond_32_bits(cuda_dev):
    """A pool of over 2^31 values a side: the used pages lie at its end."""
    from otf_llm.paged import PagedKVCache
    n, page, kv, dim = 135000, 16, 8, 128
    k, v = (torch.empty(n, page, kv, dim, dtype=torch.float16, device=cuda_dev) for _ in range(2))
    table = torch.tensor([[n - 1, n - 4, n - 2]], dtype=torch.int32, device=cuda_dev)
    cache = PagedKVCache(k, v, table, torch.zeros(1, dtype=torch.int32, device=cuda_dev))
    g = torch.Generator().manual_seed(3)
    kk, vv = torch.randn(40, kv, dim, generator=g).half(), torch.randn(40, kv, dim, generator=g).half()
    cache.append(None, kk.to(cuda_dev), vv.to(cuda_dev))
    q = torch.randn(1, 16, dim, generator=g).half()
    cache.lengths.fill_(39)
    out = cache.attend(q.to(cuda_dev)).cpu().double()
    y, p, mass, size = ref.attend(q[0], kk.double(), vv.double(), dim ** -0.5)
    assert bool(((out[0] - y).abs() <= ref.attend_tolerance(y, mass, size, dim, torch.float16)).all())
    cache.lengths.fill_(40)
    w = torch.rand(1, kv, cache.capacity, generator=g)
    kept = cache.evict(w.to(cuda_dev), 20, 4)
    for h in range(kv):
        keep = ref.evict(w[0, h], 40, 20, 4)
        assert kept[0, h].tolist() == keep
        at = [ref.place(table, page, 0, s) for s in range(20)]
        assert torch.equal(torch.stack([k[a][h] for a in at]).cpu(), kk[keep, h])
    assert flag() == 0


# ---- evict ------------------------------------------------------------------------------------


def check_evict(cuda_dev, lengths, budget, recent, page, kv, dim, dtype, order, apart, weights=None, seed=4):
    from otf_llm.paged import PagedKVCache
    cache, pools, table, g = make(cuda_dev, lengths, page, kv, dim, dtype, order, seed=seed,
                                  room=[max(n, budget) for n in lengths])
    w = torch.rand(len(lengths), kv, cache.capacity, generator=g) ** 4
    w[w < 0.05] = 0.0
    if weights is not None:
        weights(w)
    dw = w.to(cuda_dev)
    if apart:
        to, to_pools, to_table, _ = make(cuda_dev, [0] * len(lengths), page, kv, dim, dtype, "token", seed=seed + 1,
                                         room=[budget] * len(lengths))
        wo = torch.full((len(lengths), kv, budget + 5), 9.0, device=cuda_dev)
        kept = cache.evict(dw, budget, recent, to=to, weights_out=wo)
        assert same(cache.k_pages.cpu(), pools[0]) and cache.lengths.tolist() == lengths
        assert torch.equal(dw.cpu().view(torch.int32), w.view(torch.int32))
    else:
        to, to_pools, to_table, wo = cache, [p.clone() for p in pools], table, dw
        kept = cache.evict(dw, budget, recent)
    assert flag() == 0
    kept = kept.cpu()
    want = [p.clone() for p in to_pools]
    want_w = torch.zeros_like(wo.cpu()) if apart else w.clone()
    for b, n in enumerate(lengths):
        for h in range(kv):
            keep = ref.evict(w[b, h], max(n, 0), budget, recent)
            assert kept[b, h].tolist() == keep + [-1] * (budget - len(keep)), (b, h)
            if n < 0:
                if apart:
                    want_w[b, h] = 9.0
                continue
            if not apart and n > budget:
                want_w[b, h, :n] = 0
            for j, s in enumerate(keep):
                for side in (0, 1):
                    at, src = ref.place(to_table, page, b, j), ref.place(table, page, b, s)
                    want[side][at[0], at[1], h] = pools[side][src[0], src[1], h]
                want_w[b, h, j] = w[b, h, s]
    assert to.lengths.tolist() == [min(n, budget) for n in lengths]
    assert same(to.k_pages.cpu(), want[0]) and same(to.v_pages.cpu(), want[1])
    assert torch.equal(wo.cpu().view(torch.int32), want_w.view(torch.int32))


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("lengths,budget,recent,page,kv,dim,dtype,order", [
    ([1], 1, 0, 16, 1, 64, "fp16", "token"),
    ([100, 30, 31, 29, 0, -1], 30, 8, 16, 2, 64, "fp16", "token"),
    ([77, 200], 64, 64, 20, 3, 128, "bf16", "head"),
    ([300], 7, 0, 1, 2, 128, "fp16", "head"),
    ([1500, 40], 1100, 3, 128, 1, 64, "bf16", "token"),
    ([260, 33], 32, 1, 3, 2, 64, "fp16", "token"),
])
def test_evict_matches_definition(lengths, budget, recent, page, kv, dim, dtype, order, apart, cuda_dev):
    check_evict(cuda_dev, lengths, budget, recent, page, kv, dim, TYPES[dtype], order, apart)


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("kind", ["equal", "zero", "signs", "odd", "rising", "falling", "tiny"])
def test_evict_ties_and_odd_weights(kind, apart, cuda_dev):
    def weights(w):
        n = w.shape[2]
        if kind == "equal":
            w.fill_(0.25)
        elif kind == "zero":
            w.zero_()
            w[..., ::2] = -0.0
        elif kind == "signs":
            w.sub_(0.3)
        elif kind == "odd":
            w[..., 5::7] = float("nan")
            w[..., 3::11] = float("inf")
            w[..., 4::13] = -float("inf")
        elif kind == "rising":
            w.copy_(torch.arange(n).float().expand_as(w))
        elif kind == "falling":
            w.copy_(-torch.arange(n).float().expand_as(w))
        else:
            w.mul_(1e-42)                                   # subnormal
    check_evict(cuda_dev, [150, 40, 64], 40, 5, 16, 2, 64, torch.float16, "token", apart, weights)


def test_evict_long_sequence(cuda_dev):
    check_evict(cuda_dev, [5000], 700, 100, 64, 2, 64, torch.float16, "token", False)


def test_evict_layers_that_share_their_lengths(cuda_dev):
    from otf_llm.paged import PagedKVCache
    first, pools, table, g = make(cuda_dev, [90, 20, 41], 16, 2, 64, torch.float16)
    second = PagedKVCache(first.k_pages.clone(), first.v_pages.clone(), first.page_table, first.lengths)
    spare = torch.zeros(3, dtype=torch.int32, device=cuda_dev)
    weights = [torch.rand(3, 2, first.capacity, generator=g).to(cuda_dev) for _ in range(2)]
    want = [[[ref.evict(w[b, h].cpu(), n, 40, 8) for h in range(2)] for b, n in enumerate((90, 20, 41))] for w in weights]
    for i, cache in enumerate((first, second)):
        kept = cache.evict(weights[i], 40, 8, lengths_out=spare if i == 0 else None).cpu()
        assert first.lengths.tolist() == ([90, 20, 41] if i == 0 else [40, 20, 40])
        for b in range(3):
            for h in range(2):
                assert kept[b, h, :len(want[i][b][h])].tolist() == want[i][b][h]
                for j, s in enumerate(want[i][b][h]):
                    at, src = ref.place(table, 16, b, j), ref.place(table, 16, b, s)
                    assert torch.equal(cache.k_pages[at][h].cpu(), pools[0][src][h])
    assert spare.tolist() == [40, 20, 40] and flag() == 0


@pytest.mark.parametrize("batch,kv,lengths,budget,recent", [
    (1, 3, [20001], 3000, 17), (1, 2, [70003], 9000, 0), (2, 8, [33000, 8193], 8192, 8000), (50, 4, [9000, 100, 8200], 500, 60),
    (1, 1, [300000], 1000, 999)])
@pytest.mark.parametrize("kind", ["spread", "ties", "equal"])
def test_evict_selects_from_many_weights(batch, kv, lengths, budget, recent, kind, cuda_dev):
    """Selections over several CTAs and over more weights than they hold, against a stable sort.  The source's
    tables name one page again and again."""
    from otf_llm.paged import PagedKVCache
    g = torch.Generator(device=cuda_dev).manual_seed(budget)
    lens = [lengths[b % len(lengths)] for b in range(batch)]
    room = max(lens) + 40
    pages = torch.randn(1, 64, kv, 64, generator=g, device=cuda_dev).half()
    cache = PagedKVCache(pages, pages.clone(), torch.zeros(batch, -(-room // 64), dtype=torch.int32, device=cuda_dev),
                         torch.tensor(lens, dtype=torch.int32, device=cuda_dev))
    w = torch.rand(batch, kv, cache.capacity, generator=g, device=cuda_dev) ** 5
    if kind == "ties":
        w = (w * 12).round()
    elif kind == "equal":
        w.fill_(-1.5)
    each = -(-budget // 64)
    to = PagedKVCache.allocate(batch * each, 64, kv, 64, torch.arange(batch * each, dtype=torch.int32, device=cuda_dev).view(batch, each),
                               torch.zeros(batch, dtype=torch.int32, device=cuda_dev))
    wo = torch.empty(batch, kv, budget, device=cuda_dev)
    kept = cache.evict(w, budget, recent, to=to, weights_out=wo)
    assert flag() == 0 and to.lengths.tolist() == [min(n, budget) for n in lens]
    for b, n in enumerate(lens):
        if n <= budget:
            want = torch.arange(n, device=cuda_dev).expand(kv, n)
        else:
            old = w[b, :, :n - recent].sort(dim=1, descending=True, stable=True).indices[:, :budget - recent]
            want = torch.cat([old.sort(dim=1).values, torch.arange(n - recent, n, device=cuda_dev).expand(kv, recent)], 1)
        m = want.shape[1]
        assert torch.equal(kept[b, :, :m].long(), want) and bool((kept[b, :, m:] == -1).all())
        assert torch.equal(wo[b, :, :m], w[b].gather(1, want)) and not bool(wo[b, :, m:].any())
        got = to.k_pages.view(batch, each * 64, kv, 64)[b, :m]
        assert torch.equal(got, torch.stack([cache.k_pages[0, want[h] % 64, h] for h in range(kv)], 1))


# ---- graphs, streams, all together ----------------------------------------------------------------


def test_two_captured_graphs_and_another_stream(cuda_dev):
    """Two graphs of attend calls and an eager call on a third stream run at the same time and agree
    with calls one after another."""
    caches = [make(cuda_dev, [400 + 50 * i, 30, 777], 16, 2, 64, torch.float16, seed=10 + i) for i in range(3)]
    qs = [torch.randn(3, 8, 64, generator=c[3]).half().to(cuda_dev) for c in caches]
    want = []
    for (c, *_), q in zip(caches, qs):
        c.lengths.sub_(1)
        w = torch.zeros(3, 2, c.capacity, device=cuda_dev)
        want.append((c.attend(q, weights=w), w))
    outs = [(torch.zeros_like(q), torch.zeros_like(w)) for q, (_, w) in zip(qs, want)]
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(4):
                outs[i][1].zero_()
                caches[i][0].attend(qs[i], weights=outs[i][1], out=outs[i][0])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            outs[2][1].zero_()
            caches[2][0].attend(qs[2], weights=outs[2][1], out=outs[2][0])
    torch.cuda.synchronize()
    for (o, w), (wo, ww) in zip(outs, want):
        assert torch.equal(o, wo) and torch.equal(w, ww)
    assert flag() == 0


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_prompt_decode_evict_verify_together(dtype, cuda_dev):
    """Prompts enter the cache, tokens are decoded with weights kept, the cache is cut in place, decoding
    goes on at the old positions, and drafted tokens are scored and verified, against the same
    steps in 64 bits on what the cache holds."""
    from otf_llm.paged import Rotary
    from otf_llm.speculative import verify_drafts
    dt, heads, kv, dim, page = TYPES[dtype], 8, 2, 64, 16
    prompts = [50, 9, 31]
    cache, pools, table, g = make(cuda_dev, [0, 0, 0], page, kv, dim, dt, room=[96] * 3, fill=0.0)
    rotary = Rotary(dim, rot_dim=32, theta=10000.0, device=cuda_dev)
    starts = torch.tensor([0, 50, 59, 90], dtype=torch.int32, device=cuda_dev)

    def rows(n):
        return [torch.randn(n, h, dim, generator=g).to(dt).to(cuda_dev) for h in (heads, kv, kv)]
    q, k, v = rows(90)
    cache.append(q, k, v, rotary, starts=starts)
    cache.lengths.copy_(torch.tensor(prompts, dtype=torch.int32))
    weights = torch.zeros(3, kv, cache.capacity, device=cuda_dev)
    seen = list(prompts)
    sums = torch.zeros(3, kv, cache.capacity, dtype=torch.float64)

    def step(tokens):
        q, k, v = rows(3 * tokens)
        pos = torch.tensor([n + t for n in seen for t in range(tokens)], dtype=torch.int32, device=cuda_dev)
        q = cache.append(q, k, v, rotary, positions=pos)
        out = cache.attend(q.view(3, tokens, heads, dim), weights=weights)
        kp, vp = cache.k_pages.cpu(), cache.v_pages.cpu()
        for b, n in enumerate(cache.lengths.tolist()):
            kk, vv = ref.gather(kp, table, b, n + tokens), ref.gather(vp, table, b, n + tokens)
            for t in range(tokens):
                m = n + t + 1
                y, p, mass, size = ref.attend(q[b * tokens + t].cpu(), kk[:m], vv[:m], dim ** -0.5)
                off = (out[b, t].cpu().double() - y).abs()
                assert bool((off <= ref.attend_tolerance(y, mass, size, dim, dt)).all())
                sums[b, :, :m] += p.view(kv, -1, m).sum(1)
        cache.advance(tokens)
        for b in range(3):
            seen[b] += tokens
        return out

    for _ in range(4):
        step(1)
    assert float((weights.cpu().double() - sums).abs().max()) < 1e-4
    kept = cache.evict(weights, 24, 6).cpu()
    assert cache.lengths.tolist() == [24, 13, 24]
    for b in (0, 2):
        for h in range(kv):
            keep = kept[b, h].tolist()
            assert keep[-6:] == list(range(seen[b] - 6, seen[b])) and keep == sorted(set(keep))
            sums[b, h, :24] = sums[b, h, keep].clone()
            sums[b, h, 24:] = 0
    assert float((weights.cpu().double() - sums).abs().max()) < 1e-4
    step(1)
    out = step(4)
    vocab = 500
    mat = torch.randn(heads * dim, vocab, generator=g).to(cuda_dev)
    logits = out.float().reshape(3, 4, -1) @ mat
    tokens = logits[:, :3].argmax(2)
    tokens[1, 1] = (tokens[1, 1] + 1) % vocab
    got, accepted = verify_drafts(logits, tokens, temperature=0.0)
    assert accepted.tolist() == [3, 1, 3]
    best = logits.argmax(2)
    assert got[1].tolist() == [int(tokens[1, 0]), int(best[1, 1]), -1, -1]
    assert got[0].tolist() == tokens[0].tolist() + [int(best[0, 3])]
    assert flag() == 0


@pytest.mark.parametrize("scale", [1e-35, -3e-36, 0.0, 1e-44])
def test_attend_scales_below_the_smallest_normal_products(scale, cuda_dev):
    """Scores of up to 1e35 under scales that bring them back to some units, and to nothing."""
    check_attend(cuda_dev, [90, 9], 3, 16, 8, 2, 64, torch.bfloat16, spread=1e34, scale=scale, weights=True)
    check_attend(cuda_dev, [700], 1, 16, 40, 1, 128, torch.bfloat16, spread=1e34, scale=scale)


@pytest.mark.parametrize("totals,tokens,heads,kv", [
    ([40, 300, 0, 17, 90], 16, 16, 2),                      # a pass of two sequences, and the last by itself
    ([70, 33], 16, 32, 2),                                  # a sequence a pass
    ([45, 130, 2000], 16, 51, 3),                           # a KV head a pass
])
def test_attend_with_weights_under_a_table_with_much_room(totals, tokens, heads, kv, cuda_dev):
    """Short sequences under a table for 2^20 tokens, whose scores would not fit the scratch at once: in passes,
    with the results of the definition, and nothing added elsewhere."""
    from otf_llm.paged import PagedKVCache
    page, dim, dt = 64, 64, torch.float16
    small, pools, table, g = make(cuda_dev, totals, page, kv, dim, dt)
    wide = torch.full((len(totals), (1 << 20) // page), -7, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    lengths = torch.tensor([n - tokens if n > 0 else -1 for n in totals], dtype=torch.int32, device=cuda_dev)
    cache = PagedKVCache(small.k_pages, small.v_pages, wide.to(cuda_dev), lengths)
    q = torch.randn(len(totals), tokens, heads, dim, generator=g).to(dt)
    out = torch.full_like(q, 7.0).to(cuda_dev)
    w = torch.full((len(totals), kv, cache.capacity + 3), 0.5, device=cuda_dev)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    cache.attend(q.to(cuda_dev), weights=w, out=out)
    assert flag() == 0 and torch.cuda.max_memory_allocated() - before < (2 << 30) + (64 << 20)
    out = out.cpu().double()
    for b, n in enumerate(totals):
        if n == 0:
            assert bool((out[b] == 7.0).all()) and bool((w[b] == 0.5).all())
            continue
        k, v = (ref.gather(p, table, b, n) for p in pools)
        want, tol = torch.zeros(kv, n, dtype=torch.float64), torch.full((kv, n), 2.0 ** -22, dtype=torch.float64)
        for t in range(tokens):
            m = n - tokens + t + 1
            y, p, mass, size = ref.attend(q[b, t], k[:m], v[:m], dim ** -0.5)
            assert bool(((out[b, t] - y).abs() <= ref.attend_tolerance(y, mass, size, dim, dt)).all()), (b, t)
            want[:, :m] += p.view(kv, -1, m).sum(1)
            # the scores' and the sums' roundings, and those of adding up in fp32
            tol[:, :m] += (p * (size * 2.0 ** -14 + 2.0 ** -18)).view(kv, -1, m).sum(1) + 2.0 ** -22
        assert bool(((w[b, :, :n].cpu().double() - 0.5 - want).abs() <= tol).all()), b
        assert bool((w[b, :, n:] == 0.5).all())


def test_attend_walks_long_sequences_under_a_bounded_grid(cuda_dev):
    """Weights of more tokens than the weights' grid covers at once: one sequence of 300,000 tokens among 63
    missing ones over 8 KV heads, whose weights sum to the rows."""
    from otf_llm.paged import PagedKVCache
    g = torch.Generator(device=cuda_dev).manual_seed(5)
    n, kv, heads, page = 300000, 8, 16, 64
    room = -(-n // page)
    k, v = (torch.randn(40, page, kv, 64, generator=g, device=cuda_dev).half() for _ in range(2))
    table = torch.randint(0, 40, (64, room), dtype=torch.int32, generator=g, device=cuda_dev)
    lengths = torch.full((64,), -1, dtype=torch.int32, device=cuda_dev)
    lengths[37] = n - 1
    cache = PagedKVCache(k, v, table, lengths)
    q = torch.randn(64, heads, 64, generator=g, device=cuda_dev).half()
    w = torch.zeros(64, kv, cache.capacity, device=cuda_dev)
    cache.attend(q, weights=w)
    assert flag() == 0
    keys = k[table[37].long()].flatten(0, 1)[:n].double()
    p = torch.softmax(torch.einsum("hd,nhd->hn", q[37].double(), keys.repeat_interleave(2, 1)) / 8, -1).view(kv, 2, n).sum(1)
    # a score is off by 68 roundings of 2^-24 of at most 64 x 25 / 8
    assert bool(((w[37, :, :n].double() - p).abs() <= p * 2.0 ** -8 + 2.0 ** -40).all())
    w[37, :, :n] = 0
    assert not bool(w.any())


def test_documented_flow_of_ragged_prompts_and_drafts(cuda_dev):
    """Prompts of different lengths, decoded tokens, drafts of which each sequence keeps its own number, and
    a cut, over two layers that share table and lengths, through ``advance`` alone: every attention is that
    over the tokens that each sequence has kept."""
    from otf_llm.paged import PagedKVCache, Rotary
    from otf_llm.speculative import verify_drafts
    dt, heads, kv, dim, page, batch, K, vocab = torch.float16, 4, 2, 64, 16, 4, 3, 300
    g = torch.Generator().manual_seed(21)
    prompts = [50, 9, 0, 31]                                # the third place has no sequence
    table = torch.randperm(40, generator=g)[:32].to(torch.int32).view(batch, 8)
    lengths = torch.tensor([0, 0, -1, 0], dtype=torch.int32, device=cuda_dev)
    caches = [PagedKVCache.allocate(40, page, kv, dim, table.to(cuda_dev), lengths) for _ in range(2)]
    rotary = Rotary(dim, device=cuda_dev)
    kept = [[[] for _ in range(batch)] for _ in caches]     # the (key, value) rows of each layer and sequence
    turned = list(prompts)                                  # tokens so far

    def rows(n):
        return [torch.randn(n, h, dim, generator=g).to(dt) for h in (heads, kv, kv)]

    def turn(x, position):
        return ref.rotate(x, position, rotary.frequencies, 1.0, dim, False)

    def step(T):
        """T rows of every sequence through both layers; what they are, kept in full by the caller."""
        new, outs = [], []
        for cache, have in zip(caches, kept):
            q, k, v = rows(batch * T)
            out = cache.attend(cache.append(q.to(cuda_dev), k.to(cuda_dev), v.to(cuda_dev), rotary).view(batch, T, heads, dim))
            for b in range(batch):
                if b == 2:
                    continue
                mine = [(turn(k[b * T + t], turned[b] + t).to(dt).double(), v[b * T + t].double()) for t in range(T)]
                for t in range(T):
                    seen = have[b] + mine[:t + 1]
                    kk, vv = (torch.stack([pair[i] for pair in seen]) for i in (0, 1))
                    y, p, mass, size = ref.attend(turn(q[b * T + t], turned[b] + t).to(dt), kk, vv, dim ** -0.5)
                    # keys and queries turned in 64 bits may round to the other neighbour: an eps of either, so
                    # 2 eps size of a score, which count in the product and in the sum below it
                    tol = ref.attend_tolerance(y, mass, size, dim, dt) + 4 * torch.finfo(dt).eps * size * mass
                    assert bool(((out[b, t].cpu().double() - y).abs() <= tol).all()), (b, t)
                new.append((have[b], mine))
            outs.append(out)
        return new, outs

    starts = torch.tensor([0] + prompts).cumsum(0).to(torch.int32)
    for cache, have in zip(caches, kept):
        q, k, v = rows(sum(prompts))
        cache.append(q.to(cuda_dev), k.to(cuda_dev), v.to(cuda_dev), rotary, starts=starts.to(cuda_dev))
        for b in range(batch):
            have[b] += [(turn(k[starts[b] + t], t).to(dt).double(), v[starts[b] + t].double()) for t in range(prompts[b])]
    caches[0].advance(starts.to(cuda_dev).diff())
    assert lengths.tolist() == [50, 9, -1, 31]

    for _ in range(2):
        new, _ = step(1)
        caches[0].advance()
        for have, mine in new:
            have += mine
        turned[:] = [n + 1 for n in turned]
    assert lengths.tolist() == [52, 11, -1, 33]
    for want in ([3, 0, 0, 1], [1, 2, 0, 3]):               # drafts taken
        new, outs = step(K + 1)
        logits = torch.randn(batch, K + 1, vocab, generator=g).to(cuda_dev)
        drafts = logits[:, :K].argmax(2)
        for b in range(batch):
            if want[b] < K:
                drafts[b, want[b]] = (drafts[b, want[b]] + 1) % vocab
        _, accepted = verify_drafts(logits, drafts, temperature=0.0)
        assert accepted.tolist() == want
        caches[0].advance(accepted + 1)
        n = [b for b in range(batch) if b != 2] * 2
        for b, (have, mine) in zip(n, new):
            have += mine[:want[b] + 1]
        turned[:] = [m + w + 1 for m, w in zip(turned, want)]
        assert [x for x in lengths.tolist() if x >= 0] == [turned[b] for b in (0, 1, 3)] and int(lengths[2]) == -1
    step(1)
    assert flag() == 0


def test_advance_refuses_what_is_no_number_for_each_sequence(cuda_dev):
    cache, *_ = make(cuda_dev, [20, 30], 16, 2, 64, torch.float16)
    for bad in (torch.ones(2, dtype=torch.int64, device=cuda_dev), torch.ones(3, dtype=torch.int32, device=cuda_dev),
                torch.ones(2, dtype=torch.int32), torch.ones(4, dtype=torch.int32, device=cuda_dev)[::2],
                torch.ones((), dtype=torch.int32, device=cuda_dev), torch.ones(2, device=cuda_dev)):
        with pytest.raises(ValueError):
            cache.advance(bad)
    assert cache.lengths.tolist() == [20, 30]


@pytest.mark.parametrize("heads,kv,dim,rot,page", [(4, 2, 64, 64, 16), (32, 8, 128, 128, 20), (28, 4, 128, 24, 3), (0, 3, 64, 0, 16)])
def test_append_clears_the_weights_of_new_tokens(heads, kv, dim, rot, page, cuda_dev):
    """Nothing else of the weights changes, and what is appended is what it is without them."""
    from otf_llm.paged import PagedKVCache, Rotary
    lengths, new = [5, 0, -1, 33, 7], [3, 40, 2, 1, 5]
    cache, pools, table, g = make(cuda_dev, lengths, page, kv, dim, torch.float16, room=[80] * 5)
    cache.page_table[4] = -1                                # its tokens are left out
    other = PagedKVCache(cache.k_pages.clone(), cache.v_pages.clone(), cache.page_table, cache.lengths)
    rotary = Rotary(dim, rot_dim=rot, device=cuda_dev)
    n = sum(new) + 2
    q, k, v = (torch.randn(n, h, dim, generator=g).half().to(cuda_dev) if h else None for h in (heads, kv, kv))
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(cuda_dev)
    w0 = torch.rand(5, kv, cache.capacity + 7, generator=g) + 0.5
    w = w0.to(cuda_dev)
    out = None if q is None else torch.zeros_like(q)
    cache.append(q, k, v, rotary, starts=starts, q_out=out, weights=w)
    assert flag() == 1
    want = None if q is None else torch.zeros_like(q)
    other.append(q, k, v, rotary, starts=starts, q_out=want)
    assert flag() == 1 and same(cache.k_pages, other.k_pages) and same(cache.v_pages, other.v_pages)
    assert q is None or torch.equal(out, want)
    for b in (0, 1, 3):
        w0[b, :, lengths[b]:lengths[b] + new[b]] = 0
    assert torch.equal(w.cpu(), w0)
    for bad in (w[..., :cache.capacity - 1].contiguous(), w.half(), w[:4], w.cpu(), w[..., 1:]):
        with pytest.raises(ValueError):
            cache.append(q, k, v, rotary, starts=starts, weights=bad)


def test_weights_after_refused_drafts_and_a_new_sequence(cuda_dev):
    """Drafts attended with weights, some refused, the next tokens in their places, a cut: the weights are those
    of the tokens that there are, from all rows that attended; and a new sequence in a place starts at 0."""
    dt, heads, kv, dim, page, T = torch.float16, 4, 2, 64, 16, 5
    cache, pools, table, g = make(cuda_dev, [0, 0, 0], page, kv, dim, dt, room=[96] * 3, fill=0.0)
    weights = torch.zeros(3, kv, cache.capacity, device=cuda_dev)
    have = [0, 0, 0]
    want, tol = (torch.zeros(3, kv, cache.capacity, dtype=torch.float64) for _ in range(2))

    def step(tokens, taken):
        q, k, v = (torch.randn(3 * tokens, h, dim, generator=g).to(dt) for h in (heads, kv, kv))
        cache.append(None, k.to(cuda_dev), v.to(cuda_dev), weights=weights)
        cache.attend(q.view(3, tokens, heads, dim).to(cuda_dev), weights=weights)
        pages = cache.k_pages.cpu()
        for b in range(3):
            kk = ref.gather(pages, table, b, have[b] + tokens)
            want[b, :, have[b]:have[b] + tokens] = tol[b, :, have[b]:have[b] + tokens] = 0
            for t in range(tokens):
                m = have[b] + t + 1
                _, p, _, size = ref.attend(q[b * tokens + t], kk[:m], kk[:m], dim ** -0.5)
                want[b, :, :m] += p.view(kv, -1, m).sum(1)
                tol[b, :, :m] += (p * (size * 2.0 ** -14 + 2.0 ** -18)).view(kv, -1, m).sum(1) + 2.0 ** -22
            have[b] += taken[b]
        cache.advance(torch.tensor(taken, dtype=torch.int32, device=cuda_dev))

    def check():
        assert cache.lengths.tolist() == have
        for b, n in enumerate(have):
            # the roundings of the scores (68 of 2^-24 of their size, twice), of the exponentials and of the sums
            assert bool(((weights[b, :, :n].cpu().double() - want[b, :, :n]).abs() <= tol[b, :, :n]).all()), b

    for taken in ([5, 1, 3], [1, 5, 2], [4, 4, 1], [5, 5, 5], [2, 1, 5], [5, 5, 3]):
        step(T, taken)
        check()
    step(1, [1, 1, 1])
    check()
    cache.lengths[1] = have[1] = 0                          # another sequence takes the second place
    step(9, [9, 9, 9])
    step(1, [1, 1, 1])
    check()
    before = weights.cpu()
    kept = cache.evict(weights, 12, 4).cpu()
    for b in range(3):
        for h in range(kv):
            keep = ref.evict(before[b, h], have[b], 12, 4)
            assert kept[b, h].tolist() == keep + [-1] * (12 - len(keep))
    assert flag() == 0


def test_outputs_in_one_buffer_with_their_inputs(cuda_dev):
    """Queries and outputs as views of one buffer: refused where they share an element, and otherwise right."""
    import random

    from test_paged_host import overlaps
    cache, pools, table, g = make(cuda_dev, [20, 5, 33, 9, 17], 16, 2, 64, torch.float16, room=[48] * 5)
    rng, seen = random.Random(4), [0, 0]
    room = torch.randn(12000, generator=g).half().to(cuda_dev)
    k, v = (torch.randn(5, 2, 64, generator=g).half().to(cuda_dev) for _ in range(2))
    for _ in range(150):
        ldq = ldo = 8 * rng.randint(32, 80)
        if rng.random() < 0.4:
            ldo = 8 * rng.randint(32, 80)
        delta = 8 * rng.randint(-5 * 60, 5 * 60)
        buf = room.clone()
        q, out = (buf.as_strided((5, 4, 64), (ld, 64, 1), at) for ld, at in ((ldq, 4000), (ldo, 4000 + delta)))
        over = overlaps(0, ldq, 256, delta, ldo, 256, 5)
        seen[over] += 1
        if over:
            with pytest.raises((RuntimeError, ValueError)):
                cache.attend(q, out=out)
            if delta or ldq != ldo:
                with pytest.raises((RuntimeError, ValueError)):
                    cache.append(q, k, v, q_out=out)
            assert torch.equal(buf, room)
            continue
        for call in (lambda o: cache.append(q, k, v, q_out=o), lambda o: cache.attend(q, out=o)):
            call(out)
            got = out.clone()
            want = room.clone()
            want.as_strided((5, 4, 64), (ldo, 64, 1), 4000 + delta).copy_(got)
            assert torch.equal(buf, want) and torch.equal(got, call(None))
    assert min(seen) > 20 and flag() == 0
    # keys and values beside queries that are turned in place, as a fused projection leaves them
    qkv = torch.randn(5, 8, 64, generator=g).half().to(cuda_dev)
    q, k, v = qkv.split([4, 2, 2], dim=1)
    want = cache.append(q, k, v).clone()
    assert torch.equal(cache.append(q, k, v, q_out=q), want)
    with pytest.raises(RuntimeError):
        cache.append(q, k, v, q_out=qkv[:, 1:5])
    # weights, and where they go to, beside one another
    other, *_ = make(cuda_dev, [0] * 5, 16, 2, 64, torch.float16, room=[16] * 5, seed=9)
    w = torch.rand(5 * 2 * (cache.capacity + 16), generator=g).to(cuda_dev)
    cut = 5 * 2 * cache.capacity
    weights, wo = w[:cut].view(5, 2, cache.capacity), w[cut:].view(5, 2, 16)
    kept = cache.evict(weights, 16, 4, to=other, weights_out=wo)
    assert bool((wo == torch.where(kept >= 0, weights.gather(2, kept.clamp(min=0).long()), 0.0)).all())
    with pytest.raises(RuntimeError):
        cache.evict(weights, 16, 4, to=other, weights_out=w[cut - 1:cut - 1 + 160].view(5, 2, 16))
    assert flag() == 0


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("tokens,heads,kv,dim,page", [(1, 8, 2, 64, 16), (1, 16, 2, 128, 16), (2, 24, 3, 64, 20), (5, 16, 4, 128, 16),
                                                      (3, 8, 1, 128, 8), (16, 4, 2, 64, 32)])
def test_attend_as_exact_as_its_output(tokens, heads, kv, dim, page, dtype, cuda_dev):
    """Probabilities in two 16-bit numbers: the bound that tells a lost rest, and a lost token among hundreds, for
    every number of row eights."""
    dt, totals = TYPES[dtype], [2 + tokens, 5 + tokens, 17, 40, 300, 611]
    cache, pools, table, g = make(cuda_dev, totals, page, kv, dim, dt, seed=tokens)
    cache.lengths.sub_(tokens)
    q = (0.3 * torch.randn(len(totals), tokens, heads, dim, generator=g)).to(dt)
    out = cache.attend(q.to(cuda_dev)).cpu().double()
    assert flag() == 0
    for b, n in enumerate(totals):
        k, v = (ref.gather(p, table, b, n) for p in pools)
        for t in range(tokens):
            m = n - tokens + t + 1
            y, p, mass, size = ref.attend(q[b, t], k[:m], v[:m], dim ** -0.5)
            tol = ref.attend_tolerance_two(y, mass, size, dim, dt, m, float(v.abs().max()))
            assert bool(((out[b, t] - y).abs() <= tol).all()), (b, t, float(((out[b, t] - y).abs() / tol).max()))
