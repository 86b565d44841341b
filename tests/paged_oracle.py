"""The paged cache's operators in 64 bits, token by token, for the tests."""
import math

import torch


def place(page_table, page_size, b, s):
    return int(page_table[b, s // page_size]), s % page_size


def rotate(x, position, frequencies, factor, rot, interleaved):
    """x [heads, dim] turned by one position (float64)."""
    x = x.double().clone()
    a = position * frequencies.double()
    c, s = a.cos() * factor, a.sin() * factor
    if interleaved:
        i, j = torch.arange(0, rot, 2), torch.arange(1, rot, 2)
    else:
        i = torch.arange(rot // 2)
        j = i + rot // 2
    u, w = x[:, i].clone(), x[:, j].clone()
    x[:, i] = u * c - w * s
    x[:, j] = w * c + u * s
    return x


def gather(pages, page_table, b, n):
    """The first n tokens of sequence b, [n, kv_heads, dim] in float64."""
    size = pages.shape[1]
    got = [pages[place(page_table, size, b, s)].double() for s in range(n)]
    return torch.stack(got) if got else torch.zeros(0, *pages.shape[2:], dtype=torch.float64)


def attend(q, k, v, scale):
    """q [heads, dim], k and v [n, kv_heads, dim] float64 -> (out [heads, dim], p [heads, n],
    sum_j p_j |v_j| [heads, dim], the largest sum_i |q_i k_ij| [heads, 1])."""
    q = q.double()
    rep = q.shape[0] // k.shape[1]
    kk, vv = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    p = torch.softmax(torch.einsum("hd,nhd->hn", q, kk) * scale, -1)
    size = torch.einsum("hd,nhd->hn", q.abs(), kk.abs()).amax(-1, keepdim=True) * abs(scale)
    return torch.einsum("hn,nhd->hd", p, vv), p, torch.einsum("hn,nhd->hd", p, vv.abs()), size


def attend_tolerance(ref, mass, size, dim, dtype):
    """How far an output may be: the result's rounding and that of the probabilities to the same
    type (half a step of each), and the scores' fp32 sums (dim + 4 roundings of 2^-24 of the
    largest sum of magnitudes, and the exponent's, which doubles as the sum in the denominator)."""
    u = torch.finfo(dtype).eps / 2
    score = (dim + 4) * 2.0 ** -24 * size + size * 2.0 ** -22
    return u * (ref.abs() + mass) + (2 * score + 2.0 ** -16) * mass + torch.finfo(dtype).tiny * 2 ** -8


def evict(weights, length, budget, recent):
    """Places kept of one sequence's head: weights [n] -> list, in order."""
    if length <= budget:
        return list(range(length))
    old = length - recent

    def key(i):
        w = float(weights[i])
        return (-math.inf if math.isnan(w) else -w if not math.isinf(w) else math.copysign(1e300, -w) * 10, i)
    # a NaN before everything, then the larger weights, then the lower places
    order = sorted(range(old), key=lambda i: (0 if math.isnan(float(weights[i])) else 1, key(i)))
    return sorted(order[:budget - recent]) + list(range(old, length))


def verify(target, tokens, draft, uniforms, noise, temperature, count):
    """One sequence in float64: (tokens list with -1 behind, accepted)."""
    drafts, vocab = tokens.shape[0], target.shape[1]

    def soft(x):
        return torch.softmax(x.double() / temperature, -1)
    taken = 0
    while taken < count:
        d = int(tokens[taken])
        if not 0 <= d < vocab:
            break
        if temperature == 0:
            ok = d == int(target[taken].argmax())
        else:
            q = 1.0 if draft is None else float(soft(draft[taken])[d])
            ok = float(uniforms[taken]) * q < float(soft(target[taken])[d])
        if not ok:
            break
        taken += 1
    if temperature == 0:
        last = int(target[taken].argmax())
    else:
        p = soft(target[taken])
        w = p.clone()
        if taken < count:
            if draft is not None:
                w = (p - soft(draft[taken])).clamp(min=0)
            elif 0 <= int(tokens[taken]) < vocab:
                w[int(tokens[taken])] = 0
            if float(w.sum()) == 0:
                w = p
        last = int((w / noise.double()).argmax())
    return [int(x) for x in tokens[:taken]] + [last] + [-1] * (drafts - taken), taken


def attend_tolerance_two(ref, mass, size, dim, dtype, n, largest):
    """How far an output over n tokens (values of `largest` size at most) may be where probabilities go into the
    products as two 16-bit numbers, hi and the rounded rest: the result's own rounding, half a step, and
    - the scores' fp32 sums, as in attend_tolerance, twice (product and denominator);
    - hi + rest: half a step of half a step of each probability, twice; 2^-22 for the exponential, twice;
    - fp32 sums of 16 products at a time: (n / 16 + 32) roundings of 2^-23 (some hardware truncates), twice;
    - fp16 alone: rests below its smallest number, 2^-33 of the largest probability for each token."""
    u = torch.finfo(dtype).eps / 2
    score = (dim + 4) * 2.0 ** -24 * size + size * 2.0 ** -22
    rel = 2 * score + 2 * u * u + 2 * 2.0 ** -22 + 2 * (n / 16 + 32) * 2.0 ** -23
    off = rel * mass + (n * 2.0 ** -33 * largest if dtype == torch.float16 else 0.0)
    return u * (ref.abs() + off) + off + torch.finfo(dtype).tiny * u


def attend_as_products_see(q, k, v, scale, dtype, rest=True, turned=False, lost=None):
    """attend's output in float64 from probabilities rounded as the products take them: as two numbers of dtype, or
    (planted mistakes) without the rest, with neighbours' rests exchanged, or without one token."""
    rep = q.shape[0] // k.shape[1]
    kk, vv = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    s = torch.einsum("hd,nhd->hn", q.double(), kk) * scale
    p = torch.exp(s - s.amax(-1, keepdim=True)) * (256 if dtype == torch.float16 else 1)
    hi = p.to(dtype).double()
    lo = (p - hi).to(dtype).double()
    if turned:
        m = lo.shape[1] // 2 * 2
        lo[:, :m] = lo[:, :m].view(lo.shape[0], -1, 2).flip(-1).reshape(lo.shape[0], m)
    p = hi + lo if rest else hi
    if lost is not None:
        p[:, lost] = 0
    return (torch.einsum("hn,nhd->hd", p, vv) / p.sum(-1)[:, None]).to(dtype).double()
