"""Log probabilities, entropy, ranks and the likeliest tokens against 64 bits."""
import math

import pytest
import torch

import rows_oracle as ref
from test_gpu_paged import TYPES, flag

pytestmark = pytest.mark.gpu
ALL = dict(TYPES, fp32=torch.float32)


def far(vocab):
    """How far the sums under the logarithms may be, relatively: a weight's exponential, 2^-20 of it for exponents of 16 at most that matter (what is smaller adds less), and fp32
    sums of vocab / 256 / 16 + 40 roundings; they enter the logarithm of 1 + l, so l / (1 + l) <= 1 of it."""
    return 2.0 ** -20 + (vocab / 4096 + 60) * 2.0 ** -24


def check(dev, x, tokens, top):
    from otf_llm.logprobs import token_logprobs
    got = token_logprobs(x.to(dev), torch.tensor(tokens, device=dev), top=top)
    assert flag() == 0
    want = ref.logprobs(x.double(), tokens, top)
    rel = far(x.shape[1])
    lps, hs, ranks = got.logprobs.tolist(), got.entropy.tolist(), got.ranks.tolist()
    for r, (lp, h, rank, best, theirs) in enumerate(want):
        # d is exact but for its rounding; log1p(l) keeps l's relative error
        assert ranks[r] == rank, r
        assert got.top_tokens[r].tolist() == best, r
        for g, w in [(lps[r], lp)] + list(zip(got.top_logprobs[r].tolist(), theirs)):
            if math.isinf(w) or w == 0:
                assert g == w, (r, g, w)
            else:
                assert abs(g - w) <= rel * min(1.0, abs(w)) + 2.0 ** -23 * abs(w) + 1e-40, (r, g, w)
        # the second sum's terms e^d d: twice the error of the weights, up to |d| of 16
        assert abs(hs[r] - h) <= 4 * rel * max(h, 1e-30) + 1e-40, (r, hs[r], h)
    return got


def logits(n, vocab, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, vocab, generator=g) * 2.5
    at = torch.randint(0, vocab, (n, 4), generator=g)
    x.scatter_add_(1, at, torch.rand(n, 4, generator=g) * 8 + 4)
    return x.to(dtype), torch.randint(0, vocab, (n,), generator=g).tolist()


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,vocab,top", [(1, 1, 1), (3, 2, 5), (2, 31, 32), (5, 511, 20), (2, 513, 0), (4, 4097, 7),
                                         (1, 32000, 20), (40, 1003, 5), (700, 600, 3)])
def test_logprobs_match_definition(n, vocab, top, dtype, cuda_dev):
    x, tokens = logits(n, vocab, n + vocab, ALL[dtype])
    check(cuda_dev, x, tokens, top)


@pytest.mark.parametrize("order", ["up", "down", "equal"])
def test_likeliest_in_the_worst_orders(order, cuda_dev):
    n, vocab = 2, 9001
    x = torch.arange(vocab, dtype=torch.float32) / 1000
    x = {"up": x, "down": x.flip(0), "equal": torch.zeros(vocab)}[order].repeat(n, 1)
    check(cuda_dev, x, [0, vocab - 1], 32)
    check(cuda_dev, x.bfloat16(), [vocab // 2, 3], 32)


def test_peaked_rows_keep_their_precision(cuda_dev):
    """One token with nearly all of the weight: log probabilities and entropies far below 2^-24 come out to their own
    precision."""
    x = torch.full((3, 5000), -3.0)
    x[0, 77], x[1, 4999], x[2, 0] = 30.0, 50.0, 15.0
    got = check(cuda_dev, x, [77, 4999, 0], 2)
    assert -1e-9 < float(got.logprobs[0]) < 0 and 0 < float(got.entropy[1]) < 1e-16


def test_masked_and_odd_values(cuda_dev):
    from otf_llm.logprobs import token_logprobs
    inf, nan = math.inf, math.nan
    x, _ = logits(6, 1500, 3)
    x[0, ::2] = -inf
    x[1, 5:] = torch.finfo(torch.float32).min
    x[2, :100] = nan
    x[3] = -inf
    x[3, 1400] = 2.0
    x[4] = -inf
    x[5] = nan
    x[5, 3] = -1.0
    check(cuda_dev, x[:4], [0, 7, 50, 1400], 4)
    got = token_logprobs(x[4:].to(cuda_dev), torch.tensor([9, 3], device=cuda_dev), top=3)
    assert flag() == 0
    assert got.logprobs.tolist() == [-inf, 0.0] and got.entropy.tolist() == [0.0, 0.0] and got.ranks.tolist() == [9, 0]
    assert got.top_tokens.tolist() == [[-1, -1, -1], [3, -1, -1]]
    assert got.top_logprobs.tolist() == [[-inf] * 3, [0.0, -inf, -inf]]
    # two infinities share all weight, as the largest finite numbers would
    y = x[:1].clone()
    y[0, 11] = y[0, 900] = inf
    got = token_logprobs(y.to(cuda_dev), torch.tensor([900], device=cuda_dev), top=2)
    assert abs(float(got.logprobs) + math.log(2)) < 1e-6 and got.top_tokens.tolist() == [[11, 900]]
    assert int(got.ranks) == 1 and abs(float(got.entropy) - math.log(2)) < 1e-6


def test_no_token_and_tokens_outside(cuda_dev):
    from otf_llm.logprobs import token_logprobs
    x, tokens = logits(4, 700, 9)
    plain = token_logprobs(x.to(cuda_dev), torch.tensor(tokens, device=cuda_dev), top=3)
    got = token_logprobs(x.to(cuda_dev), torch.tensor([-1, tokens[1], -100, 700], device=cuda_dev), top=3)
    assert flag() == 1
    assert got.logprobs[[0, 2]].tolist() == [0.0, 0.0] and math.isnan(float(got.logprobs[3]))
    assert got.ranks.tolist() == [-1, int(plain.ranks[1]), -1, -1]
    for a, b in ((got.entropy, plain.entropy), (got.top_tokens, plain.top_tokens), (got.top_logprobs, plain.top_logprobs),
                 (got.logprobs[1], plain.logprobs[1])):
        assert torch.equal(a, b)
    empty = token_logprobs(x[:0].to(cuda_dev), torch.zeros(0, dtype=torch.int64, device=cuda_dev), top=3)
    assert empty.logprobs.shape == (0,) and empty.top_tokens.shape == (0, 3)


def test_strides_and_alignment_do_not_change_results(cuda_dev):
    """Rows apart, and rows that start on no 16-byte border."""
    from otf_llm.logprobs import token_logprobs
    for dtype in ALL.values():
        x, tokens = logits(9, 1111, 4, dtype)
        t = torch.tensor(tokens, device=cuda_dev)
        plain = token_logprobs(x.to(cuda_dev), t, top=6)
        wide = torch.full((9, 1120), math.nan, dtype=dtype, device=cuda_dev)
        wide[:, 3:1114] = x.to(cuda_dev)
        for a, b in zip(token_logprobs(wide[:, 3:1114], t, top=6), plain):
            assert torch.equal(a, b)
    assert flag() == 0


def test_captured_and_on_a_stream(cuda_dev):
    from otf_llm.logprobs import token_logprobs
    x, tokens = logits(3, 5000, 5)
    dx, dt = x.to(cuda_dev), torch.tensor(tokens, device=cuda_dev)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        token_logprobs(dx, dt, top=4)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = token_logprobs(dx, dt, top=4)
        y, other = logits(3, 5000, 6)
        dx.copy_(y)
        dt.copy_(torch.tensor(other))
        graph.replay()
    side.synchronize()
    for a, b in zip(held, token_logprobs(y.to(cuda_dev), torch.tensor(other, device=cuda_dev), top=4)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("vocab,at", [(1500, (600, 1400, 0, 511, 512)), (32000, (31999, 17001, 513, 4097, 16384))])
def test_ranks_of_masked_tokens_behind_the_first_logits(vocab, at, dtype, cuda_dev):
    """Tokens of -inf and NaN, which counts as -inf, in every part of a row: all that is larger and the masked ones
    of lower indexes come before them, wherever those lie."""
    x, _ = logits(len(at), vocab, vocab, ALL[dtype])
    x[:, 1::2] = -math.inf
    x[1:, 2::6] = math.nan
    x[2] = -math.inf
    for r, token in enumerate(at):
        x[r, token] = math.nan if r % 2 else -math.inf
    if not x[2].isfinite().any():
        x[2, 3] = 1.0
    check(cuda_dev, x, list(at), 3)
    # and of tokens that are as large as many others
    y = torch.full((len(at), vocab), torch.finfo(ALL[dtype]).min, dtype=ALL[dtype])
    y[:, ::3] = 0.0
    y[:, 1::3] = -0.0
    check(cuda_dev, y, list(at), 3)
