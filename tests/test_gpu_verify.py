"""Verification of drafted tokens against the definition in 64 bits."""
import pytest
import torch

import paged_oracle as ref

pytestmark = pytest.mark.gpu


def flag():
    from otf_llm import _native
    torch.cuda.synchronize()
    return _native.device_error(clear=True)


def inputs(batch, drafts, vocab, drafted, seed, near=0.6, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    target = torch.randn(batch, drafts + 1, vocab, generator=g) * spread
    draft = target[:, :drafts] + near * torch.randn(batch, drafts, vocab, generator=g) if drafted else None
    if drafted and drafts:
        tokens = torch.softmax(draft.double(), -1).view(-1, vocab).multinomial(1, generator=g).view(batch, drafts)
    else:
        tokens = torch.where(torch.rand(batch, drafts, generator=g) < 0.7, target[:, :drafts].argmax(2),
                             torch.randint(0, vocab, (batch, drafts), generator=g))
    uniforms = torch.rand(batch, drafts, generator=g)
    noise = torch.empty(batch, vocab).exponential_(generator=g)
    return target, tokens, draft, uniforms, noise


def check(dev, target, tokens, draft, uniforms, noise, temperature, counts=None, error=0):
    from otf_llm.speculative import verify_drafts
    on = [None if t is None else t.to(dev) for t in (target, tokens, draft, uniforms, noise)]
    each = temperature if isinstance(temperature, list) else [temperature] * target.shape[0]
    t = torch.tensor(each, device=dev) if isinstance(temperature, list) else temperature
    c = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=dev)
    got, accepted = verify_drafts(on[0], on[1], draft_logits=on[2], uniforms=on[3], noise=on[4], temperature=t, counts=c)
    assert flag() == error
    for b in range(target.shape[0]):
        want, taken = ref.verify(target[b], tokens[b], None if draft is None else draft[b],
                                 None if uniforms is None else uniforms[b], None if noise is None else noise[b],
                                 each[b], tokens.shape[1] if counts is None else counts[b])
        assert (got[b].tolist(), int(accepted[b])) == (want, taken), b
    return got, accepted


@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0, 5.0])
@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("batch,drafts,vocab", [(1, 0, 1), (1, 1, 2), (3, 0, 1000), (2, 4, 8191), (5, 3, 8192),
                                                (2, 2, 8193), (4, 5, 32000), (1, 32, 777), (2, 3, 50257)])
def test_verify_matches_definition(batch, drafts, vocab, drafted, temperature, cuda_dev):
    check(cuda_dev, *inputs(batch, drafts, vocab, drafted, seed=batch * 100 + drafts + vocab), temperature)


@pytest.mark.parametrize("temperature", [0.0, 0.8])
@pytest.mark.parametrize("batch,drafts,vocab,drafted", [(1, 4, 128256, True), (3, 2, 100001, False), (40, 2, 40001, True),
                                                        (9, 1, 300000, False), (700, 1, 50, True), (2, 32, 70000, False)])
def test_verify_large_calls(batch, drafts, vocab, drafted, temperature, cuda_dev):
    """Calls on either side of the switches between one launch and three, and between cluster sizes."""
    args = inputs(batch, drafts, vocab, drafted, seed=vocab)
    counts = [(3 * b) % (drafts + 1) for b in range(batch)]
    check(cuda_dev, *args, temperature, counts=None if batch % 2 else counts)


def test_verify_counts_and_temperatures_of_each_sequence(cuda_dev):
    args = inputs(6, 4, 3001, True, seed=5)
    check(cuda_dev, *args, [0.0, 1.0, 0.3, 0.0, 2.0, 1.0], counts=[4, 0, 2, 3, 1, 4])
    args = inputs(6, 4, 3001, False, seed=6)
    check(cuda_dev, *args, [1.0, 0.0, 0.3, 2.0, 0.0, 1.0], counts=[0, 0, 4, 4, 4, 1])


def test_verify_ties_go_to_the_lowest_index(cuda_dev):
    target, tokens, _, _, _ = inputs(2, 2, 20000, False, seed=7)
    target[:] = target.round()
    check(cuda_dev, target, target[:, :2].argmax(2), None, None, None, 0.0)
    # equal weights and equal noise: the first of them all, and of those that the draft leaves
    target[:] = 0.0
    noise = torch.ones(2, 20000)
    got, accepted = check(cuda_dev, target, torch.zeros(2, 2, dtype=torch.int64), None, torch.full((2, 2), 0.5), noise, 1.0)
    assert got.tolist() == [[1, -1, -1]] * 2 and accepted.tolist() == [0, 0]


def test_verify_masked_logits(cuda_dev):
    """Logits of -inf are never taken or drawn; all of the target's mass in one place."""
    target, tokens, draft, uniforms, noise = inputs(4, 3, 9000, True, seed=8)
    target[:, :, 1::2] = -float("inf")
    draft[:, :, ::3] = -float("inf")
    tokens[0, 0] = 1                                        # nothing under the target
    check(cuda_dev, target, tokens, draft, uniforms, noise, 1.0)
    target[:, :, :] = -float("inf")
    target[:, :, 4242] = -3.0
    got, accepted = check(cuda_dev, target, torch.full((4, 3), 4242), None, uniforms, noise, 1.0)
    assert accepted.tolist() == [3] * 4 and bool((got == 4242).all())
    # the lowest finite logits instead of -inf
    target[target == -float("inf")] = torch.finfo(torch.float32).min
    check(cuda_dev, target, torch.full((4, 3), 4242), None, uniforms, noise, 0.9)


def test_verify_nan_logits_count_as_masked(cuda_dev):
    from otf_llm.speculative import verify_drafts
    target, tokens, draft, uniforms, noise = (t.to(cuda_dev) for t in inputs(4, 3, 9001, True, seed=13))
    target[:, :, 1::3], draft[:, :, 2::5] = float("nan"), float("nan")
    for temperature in (0.0, 0.8):
        rest = dict(uniforms=uniforms, noise=noise, temperature=temperature)
        got = verify_drafts(target, tokens, draft_logits=draft, **rest)
        want = verify_drafts(target.nan_to_num(nan=-float("inf")), tokens,
                             draft_logits=draft.nan_to_num(nan=-float("inf")), **rest)
        assert flag() == 0 and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("vocab", [1, 500, 700001])
def test_verify_greedy_of_nothing_but_masked_logits(vocab, cuda_dev):
    """A row of -inf, or of NaN, or of both holds no token at temperature 0 either: a drafted one is refused
    there, and none follows; sequences with a logit above them are as without masks."""
    from otf_llm.speculative import verify_drafts
    target = torch.full((4, 3, vocab), -float("inf"))
    target[1, :, ::2] = float("nan")
    target[2] = float("nan")
    target[3, :, vocab // 2] = -1e30
    tokens = torch.full((4, 2), vocab // 2)
    tokens[:3] = 0
    got, accepted = verify_drafts(target.to(cuda_dev), tokens.to(cuda_dev), temperature=0.0)
    assert flag() == 1
    assert got.tolist() == [[-1] * 3] * 3 + [[vocab // 2] * 3] and accepted.tolist() == [0, 0, 0, 2]


def test_verify_equal_distributions(cuda_dev):
    """Draft and target the same: all taken; one refused all the same (u = 1 cannot be below) leaves nothing
    of p - q, and p is drawn from."""
    target, tokens, _, uniforms, noise = inputs(3, 3, 5000, True, seed=9)
    draft = target[:, :3].clone()
    got, accepted = check(cuda_dev, target, tokens, draft, uniforms, noise, 1.0)
    assert accepted.tolist() == [3, 3, 3]
    uniforms = uniforms.clone()
    uniforms[1, 1] = 1.0
    got, accepted = check(cuda_dev, target, tokens, draft, uniforms, noise, 1.0)
    assert accepted.tolist() == [3, 1, 3]


def test_verify_flags_what_it_cannot_do(cuda_dev):
    from otf_llm.speculative import verify_drafts
    target, tokens, _, uniforms, noise = (None if t is None else t.to(cuda_dev) for t in inputs(3, 2, 100, False, seed=10))
    whole = dict(uniforms=uniforms, noise=noise)
    base, took = verify_drafts(target, tokens, **whole)
    assert flag() == 0
    for counts in ([2, 3, 2], [2, -1, 2]):
        got, accepted = verify_drafts(target, tokens, counts=torch.tensor(counts, dtype=torch.int32, device=cuda_dev), **whole)
        assert flag() == 1 and got[1].tolist() == [-1] * 3 and int(accepted[1]) == 0
        assert torch.equal(got[::2], base[::2]) and torch.equal(accepted[::2], took[::2])
    for bad in (-1.0, float("nan"), float("inf")):
        got, accepted = verify_drafts(target, tokens, temperature=torch.tensor([1.0, bad, 1.0], device=cuda_dev), **whole)
        assert flag() == 1 and got[1].tolist() == [-1] * 3 and torch.equal(got[::2], base[::2])
    empty = target.clone()
    empty[1] = -float("inf")
    got, accepted = verify_drafts(empty, tokens, **whole)
    assert flag() == 1 and got[1].tolist() == [-1] * 3 and torch.equal(got[::2], base[::2])
    empty[1] = float("nan")
    for t in (0.0, 1.0):
        got, accepted = verify_drafts(empty, tokens, temperature=t, **whole)
        assert flag() == 1 and got[1].tolist() == [-1] * 3
    for outside in (-1, 100, 2 ** 40):
        t = tokens.clone()
        t[1, 0] = outside
        got, accepted = verify_drafts(target, t, **whole)
        assert flag() == 1 and int(accepted[1]) == 0 and 0 <= int(got[1, 0]) < 100 and torch.equal(got[::2], base[::2])


def test_verify_strided_inputs_and_graph(cuda_dev):
    from otf_llm.speculative import verify_drafts
    target, tokens, draft, uniforms, noise = inputs(4, 3, 1001, True, seed=11)
    wide = torch.zeros(4, 6, 1203)
    wide[:, 1:5, 5:1006] = target
    target = wide.to(cuda_dev)[:, 1:5, 5:1006]
    tok = torch.zeros(4, 7, dtype=torch.int64)
    tok[:, 2:5] = tokens
    tok = tok.to(cuda_dev)[:, 2:5]
    rest = dict(draft_logits=draft.to(cuda_dev), uniforms=uniforms.to(cuda_dev), noise=noise.to(cuda_dev))
    want = verify_drafts(target.contiguous(), tok.contiguous(), **rest)
    assert all(torch.equal(a, b) for a, b in zip(want, verify_drafts(target, tok, **rest)))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = verify_drafts(target, tok, **rest)
    got[0].zero_()
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and flag() == 0


def test_verify_draws_from_the_target(cuda_dev):
    """Over many sequences the first produced token is distributed as the target's softmax, whatever the
    draft: expected counts within five standard deviations."""
    from otf_llm.speculative import verify_drafts
    n, vocab = 20000, 12
    g = torch.Generator().manual_seed(12)
    p_log, q_log = torch.randn(vocab, generator=g), torch.randn(vocab, generator=g)
    tokens = torch.softmax(q_log.double(), 0).multinomial(n, replacement=True, generator=g).view(n, 1)
    got, _ = verify_drafts(p_log.expand(n, 2, vocab).contiguous().to(cuda_dev), tokens.to(cuda_dev),
                           draft_logits=q_log.expand(n, 1, vocab).contiguous().to(cuda_dev),
                           uniforms=torch.rand(n, 1, generator=g).to(cuda_dev),
                           noise=torch.empty(n, vocab).exponential_(generator=g).to(cuda_dev))
    seen = torch.bincount(got[:, 0].cpu(), minlength=vocab).double()
    p = torch.softmax(p_log.double(), 0)
    assert bool(((seen - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all())


def test_verify_large_equal_distributions(cuda_dev):
    """As above, over several CTAs of a race: nothing of p - q is left, p is drawn from."""
    target, tokens, _, uniforms, noise = inputs(8, 2, 200003, True, seed=31)
    uniforms = uniforms.clone()
    uniforms[::2, 1] = 1.0
    got, accepted = check(cuda_dev, target, tokens, target[:, :2].clone(), uniforms, noise, 1.0)
    assert accepted.tolist() == [1, 2] * 4


def test_verify_large_ties_go_to_the_lowest_index(cuda_dev):
    batch, vocab = 6, 600000
    target, tokens = torch.zeros(batch, 2, vocab), torch.zeros(batch, 1, dtype=torch.int64)
    target[:, :, :1000] = -float("inf")
    tokens[::2] = 1000
    got, accepted = check(cuda_dev, target, tokens, None, torch.full((batch, 1), 0.5), torch.ones(batch, vocab), 1.0)
    assert got.tolist() == [[1001, -1], [1000, -1]] * 3 and accepted.tolist() == [0] * batch


@pytest.mark.parametrize("batch,drafts,vocab,drafted", [(1, 12, 128256, True), (4, 5, 128256, True), (5, 2, 110001, True),
                                                        (2, 32, 60000, True), (150, 16, 4001, False)])
def test_verify_on_either_side_of_the_switches(batch, drafts, vocab, drafted, cuda_dev):
    check(cuda_dev, *inputs(batch, drafts, vocab, drafted, seed=vocab + batch), 0.9)


@pytest.mark.parametrize("temperature", [1e-6, 1e-8, 1e-10, 3e-10, 1e-12, 1e-20])
@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("batch,vocab", [(2, 3001), (8, 200003)])
def test_verify_lowest_finite_masks_at_small_temperatures(batch, vocab, drafted, temperature, cuda_dev):
    """Logits masked with the lowest finite number, down to the smallest temperature, in one launch and in
    three: the masked ones weigh nothing, and the largest of the others is taken and drawn."""
    target, tokens, draft, uniforms, noise = inputs(batch, 3, vocab, drafted, seed=vocab)
    target[:, :, 1::2] = torch.finfo(torch.float32).min
    if drafted:
        draft[:, :, ::3] = torch.finfo(torch.float32).min
    tokens = (draft if drafted else target[:, :3]).argmax(2)
    tokens[0, 1] = 1                                        # a masked one
    check(cuda_dev, target, tokens, draft, uniforms, noise, temperature)
