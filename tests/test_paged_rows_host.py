"""Attention of many rows, tree walks, kept paths and log probabilities without a GPU: refusals, and the oracles'
own checks."""
import ctypes

import pytest
import torch

import paged_oracle as ref
import rows_oracle as rows
from test_paged_host import FAKE, INVALID, UNSUPPORTED, cache


def test_no_cpu_path():
    from otf_llm.logprobs import token_logprobs
    from otf_llm.speculative import verify_tree
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs(torch.zeros(1, 8), torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        verify_tree(torch.zeros(1, 8), torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.int32), temperature=0.0)


def attend(**other):
    from otf_llm import _native as N
    given = dict(cache=ctypes.byref(cache(**{k[2:]: v for k, v in other.items() if k.startswith("c_")})), q=FAKE, ldq=512,
                 heads=8, starts=FAKE, n=12, parents=None, window=0, sinks=0, scale=0.125, out=FAKE << 1, ldo=512, ws=FAKE,
                 bytes=1 << 40)
    given.update({k: v for k, v in other.items() if not k.startswith("c_")})
    return N.lib().otf_paged_attn_rows(*given.values(), None)


BAD_ROWS = [(dict(cache=None), INVALID), (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(heads=0), INVALID),
            (dict(heads=7), INVALID), (dict(n=0), INVALID), (dict(n=-1), INVALID), (dict(ldq=511), INVALID),
            (dict(ldq=504), INVALID), (dict(ldo=500), INVALID), (dict(q=FAKE + 8), INVALID), (dict(out=FAKE), INVALID),
            (dict(out=FAKE + 1024), INVALID), (dict(window=-1), INVALID), (dict(sinks=-1), INVALID), (dict(sinks=2), INVALID),
            (dict(parents=FAKE, window=63), INVALID), (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
            (dict(scale=3e38), INVALID), (dict(starts=None, n=13), INVALID), (dict(ws=None), INVALID), (dict(ws=FAKE + 16), INVALID),
            (dict(bytes=1000), INVALID), (dict(starts=None, parents=FAKE, n=195), UNSUPPORTED), (dict(n=1 << 31), UNSUPPORTED),
            (dict(n=(1 << 31) // 4 - 60, out=FAKE << 30), UNSUPPORTED), (dict(c_head_dim=96), UNSUPPORTED), (dict(c_batch=4097), UNSUPPORTED),
            (dict(c_dtype=2), UNSUPPORTED), (dict(c_lengths=None), INVALID)]


@pytest.mark.parametrize("other,status", BAD_ROWS)
def test_abi_refuses_bad_rows(other, status):
    assert attend(**other) == status


def test_rows_workspace():
    from otf_llm import _native as N
    size = N.lib().otf_paged_attn_rows_workspace_bytes
    for bad in ((0, 1, 8, 2, 64), (1, 0, 8, 2, 64), (1, 1, 7, 2, 64), (1, 1, 8, 0, 64), (1, 1, 8, 2, 96), (4097, 1, 8, 2, 64),
                (1, 1 << 31, 8, 2, 64)):
        assert size(*bad) == -1
    # a part for each end of a run on 148 CTAs: 8 rows at least, 256 at most
    assert size(1, 1, 2, 2, 64) >= 296 * 8 * 64 * 4
    assert size(1, 1 << 28, 8, 2, 128) == size(1, 64, 8, 2, 128) >= 296 * 256 * 128 * 4


def tree(**other):
    from otf_llm import _native as N
    given = dict(target=FAKE, ldt=100, tokens=FAKE, parents=FAKE, starts=FAKE, n=12, noise=FAKE, nseq=400, ldn=100, temps=None,
                 temperature=1.0, out=FAKE, path=FAKE, accepted=FAKE, batch=3, depth=3, vocab=100, ws=FAKE, bytes=1 << 30)
    given.update(other)
    return N.lib().otf_verify_tree(*given.values(), None)


BAD_TREES = [(dict(target=None), INVALID), (dict(tokens=None), INVALID), (dict(parents=None), INVALID), (dict(out=None), INVALID),
             (dict(path=None), INVALID), (dict(accepted=None), INVALID), (dict(batch=0), INVALID), (dict(depth=-1), INVALID),
             (dict(vocab=0), INVALID), (dict(n=0), INVALID), (dict(starts=None, n=13), INVALID), (dict(ldt=99), INVALID),
             (dict(temperature=-1.0), INVALID), (dict(temperature=float("nan")), INVALID), (dict(noise=None), INVALID),
             (dict(noise=None, temperature=0.0, temps=FAKE), INVALID), (dict(ldn=99), INVALID), (dict(nseq=-1), INVALID),
             (dict(ws=None), INVALID), (dict(bytes=8), INVALID), (dict(ws=FAKE + 8), INVALID), (dict(depth=64), UNSUPPORTED),
             (dict(batch=65536), UNSUPPORTED), (dict(starts=None, n=195), UNSUPPORTED), (dict(n=1 << 31), UNSUPPORTED),
             (dict(vocab=(1 << 30) + 1, ldt=1 << 31, ldn=1 << 31), UNSUPPORTED)]


@pytest.mark.parametrize("other,status", BAD_TREES)
def test_abi_refuses_bad_trees(other, status):
    assert tree(**other) == status


@pytest.mark.parametrize("temperature", [1e-50, 1e-46, 5e-324, 9e-21, 1.1e20, float("inf"), -0.1])
def test_abi_refuses_temperatures_beside_the_range(temperature):
    """Also those that fp32 would hold as 0."""
    assert tree(temperature=temperature) == INVALID


def test_tree_workspace():
    from otf_llm import _native as N
    size = N.lib().otf_verify_tree_workspace_bytes
    assert size(0, 10) == size(1, 0) == size(1 << 31, 1) == size(1, (1 << 30) + 1) == -1
    assert size(26, 32000) == 26 * 4 * 16 and size(64 * 40, 128256) == 0 and size(1, 1) == 16 and size(65536, 1) == 0


BAD_PATHS = [(dict(accepted=None), INVALID), (dict(path=None), INVALID), (dict(depth=-1), INVALID), (dict(ld=3), INVALID),
             (dict(depth=64, ld=64), UNSUPPORTED), (dict(cache=None), INVALID)]


@pytest.mark.parametrize("other,status", BAD_PATHS)
def test_abi_refuses_bad_paths(other, status):
    from otf_llm import _native as N
    given = dict(cache=ctypes.byref(cache()), path=FAKE, ld=4, accepted=FAKE, depth=4)
    given.update(other)
    assert N.lib().otf_paged_keep(*given.values(), None) == status


BAD_LOGITS = [(dict(x=None), INVALID), (dict(tokens=None), INVALID), (dict(lp=None), INVALID), (dict(h=None), INVALID),
              (dict(ranks=None), INVALID), (dict(n=0), INVALID), (dict(vocab=0), INVALID), (dict(ld=99), INVALID),
              (dict(top=-1), INVALID), (dict(tt=None), INVALID), (dict(tl=None), INVALID), (dict(dtype=3), UNSUPPORTED),
              (dict(x=FAKE + 2), INVALID), (dict(x=FAKE + 1, dtype=0), INVALID), (dict(top=33), UNSUPPORTED),
              (dict(n=(1 << 26) + 1), UNSUPPORTED), (dict(vocab=(1 << 30) + 1, ld=1 << 31), UNSUPPORTED)]


@pytest.mark.parametrize("other,status", BAD_LOGITS)
def test_abi_refuses_bad_logits(other, status):
    from otf_llm import _native as N
    given = dict(x=FAKE, ld=100, dtype=2, tokens=FAKE, n=3, vocab=100, top=5, lp=FAKE, h=FAKE, ranks=FAKE, tt=FAKE, tl=FAKE)
    given.update(other)
    assert N.lib().otf_token_logprobs(*given.values(), None) == status


# ---- the oracles ------------------------------------------------------------------------------


def test_oracle_sees_windows_sinks_and_ways():
    assert rows.seen(3, 1, None, 0) == [0, 1, 2, 3, 4]
    assert rows.seen(10, 0, 3, 2) == [0, 1, 8, 9, 10]
    assert rows.seen(1, 2, 2, 5) == [0, 1, 2, 3]
    assert rows.seen(5, 3, None, 0, [-1, 0, 0, 1]) == [0, 1, 2, 3, 4, 5, 6, 8]
    assert rows.seen(100, 2, 64, 1, [-1, 0, -1])[:2] == [0, 37] and rows.seen(100, 1, 64, 1, [-1, 0, -1])[:2] == [0, 38]
    assert rows.levels([-1, 0, 1, 0, 3, -1]) == [0, 1, 2, 1, 2, 0]


def test_oracle_walks():
    target = torch.zeros(4, 9)
    target[0, 5], target[2, 7] = 1.0, 1.0
    assert rows.walk(target, torch.tensor([0, 5, 5, 7]), [-1, 0, 0, 2], None, 0, 3) == ([5, 0], [1], 1)
    assert rows.walk(target, torch.tensor([0, 4, 5, 7]), [-1, 0, 0, 2], None, 0, 3) == ([5, 7, 0], [2, 3], 2)
    assert rows.walk(target, torch.tensor([0, 4, 5, 7]), [-1, 0, 0, 2], None, 0, 1) == ([5, 7], [2], 1)


def test_tolerance_catches_planted_mistakes():
    """Attention without one token of the window, with one too many, or with a node's sibling: beyond the bound.  Within
    it: probabilities rounded once where that is allowed."""
    g = torch.Generator().manual_seed(2)
    for dtype in (torch.float16, torch.bfloat16):
        k, v = (torch.randn(90, 1, 64, generator=g).to(dtype).double() for _ in range(2))
        q = torch.randn(1, 64, generator=g).to(dtype)
        at = rows.seen(89, 0, 40, 3)
        want = ref.attend(q, k[at], v[at], 0.125) + (len(at), float(v[at].abs().max()))
        most = rows.tolerance(want, 64, dtype, True)
        for other in (at[1:], at + [10], at[:-1]):
            wrong = ref.attend(q, k[other], v[other], 0.125)[0].to(dtype).double()
            assert bool(((wrong - want[0]).abs() > most).any())
        once = ref.attend_as_products_see(q, k[at], v[at], 0.125, dtype, rest=False)
        assert bool(((once - want[0]).abs() <= most).all())


def test_logprob_oracle_against_torch():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 40, generator=g).double() * 3
    lp = torch.log_softmax(x, 1)
    for r, (a, h, rank, best, theirs) in enumerate(rows.logprobs(x, [1, 2, 3, 4, 5], 4)):
        assert abs(a - float(lp[r, r + 1])) < 1e-12 and abs(h + float((lp.exp() * lp).sum(1)[r])) < 1e-12
        assert best == lp[r].topk(4).indices.tolist() and rank == int((lp[r] > lp[r, r + 1]).sum())
