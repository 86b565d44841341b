"""Attention of many rows over the paged cache, tree walks and log probabilities in 64 bits, row by row, for the
tests; what paged_oracle.py has is used from there."""
import math

import torch

import paged_oracle as ref


def levels(parents):
    out = []
    for p in parents:
        out.append(0 if p < 0 else out[p] + 1)
    return out


def seen(length, t, window, sinks, parents=None):
    """The places that row t of a sequence sees, as a list of places in order."""
    if parents is None:
        p = length + t
        return [s for s in range(p + 1) if window is None or s > p - window or s < sinks]
    way, at = [], t
    while at >= 0:
        way.append(at)
        at = parents[at]
    p = length + len(way) - 1
    return [s for s in range(length) if window is None or s > p - window or s < sinks] + [length + i for i in sorted(way)]


def attend(pools, table, length, q, heads_of, window, sinks, scale, parents=None):
    """q [tokens, heads, dim] of sequence `heads_of`: lists of paged_oracle.attend's results, row by row, with the number
    of tokens that each saw and the largest value among them."""
    k = ref.gather(pools[0], table, heads_of, length + q.shape[0])
    v = ref.gather(pools[1], table, heads_of, length + q.shape[0])
    rows = []
    for t in range(q.shape[0]):
        at = seen(length, t, window, sinks, parents)
        rows.append(ref.attend(q[t], k[at], v[at], scale) + (len(at), float(v[at].abs().max())))
    return rows


def tolerance(row, dim, dtype, once):
    """How far an output may be.  once: probabilities rounded once to dtype (blocks of many rows), which is
    attend_tolerance's bound and, in fp16, half of the smallest step, 2^-25, of each probability below 2^-14 under a
    factor of 2^8 at least, so 2^-33 of the largest probability for each token; the sum is of probabilities before their
    rounding, which adds as much again for the denominator.  Otherwise as two numbers: attend_tolerance_two's."""
    out, _, mass, size, n, largest = row
    two = ref.attend_tolerance_two(out, mass, size, dim, dtype, n, largest)
    if not once:
        return two
    u = torch.finfo(dtype).eps / 2
    return two + 2 * u * mass


def walk(target, tokens, parents, noise, temperature, depth):
    """One sequence's walk in float64: (tokens, path, accepted)."""
    at, out, path = 0, [], []
    while True:
        if temperature == 0:
            drawn = int(target[at].argmax())
        else:
            score = target[at].double() / temperature - noise[len(path)].double().log()
            drawn = int(score.argmax())
        out.append(drawn)
        below = [i for i in range(len(parents)) if parents[i] == at and int(tokens[i]) == drawn]
        if len(path) == depth or not below:
            return out, path, len(path)
        at = below[0]
        path.append(at)


def logprobs(x, tokens, top):
    """x [rows, vocab] float64 (NaN as -inf): lists per row of (log probability, entropy, rank, [tokens], [their log
    probabilities])."""
    rows = []
    for r in range(x.shape[0]):
        y = torch.where(x[r].isnan(), -math.inf, x[r].double())
        d = y - y.max()
        e = torch.exp(d)
        rest = e.clone()
        rest[int(y.argmax())] = 0.0
        more = math.log1p(float(rest.sum()))            # of the sum of exponentials, without the largest's 1
        h = more - float(torch.where(e > 0, e * d, 0.0).sum() / e.sum())
        order = sorted(range(y.shape[0]), key=lambda i: (-float(y[i]), i))
        order = [i for i in order[:top] if float(y[i]) > -math.inf]
        t = int(tokens[r])
        lp = float(d[t]) - more if t >= 0 else 0.0
        rank = int(((y > y[t]) | ((y == y[t]) & (torch.arange(y.shape[0]) < t))).sum()) if t >= 0 else -1
        rows.append((lp, h, rank, order + [-1] * (top - len(order)),
                     [float(d[i]) - more for i in order] + [-math.inf] * (top - len(order))))
    return rows
