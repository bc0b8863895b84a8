"""A batch whose values cancel in pairs of keys of nearly the same weight, so that outputs are small beside what they are sums of and a rounding
of the weights shows."""
import numpy as np

import paged_cases as cases


def fill(g, b, kind):
    """Pools and tokens of a batch: keys of -1, 0 and 1 (scores are exact), the second of two in one value apart; values r and -r."""
    k, v, _ = b.fill(g, np.nan)
    tokens = []
    ahead = one(g, b.prefix, b.kv, b.dim)
    for t in range(b.prefix):
        p, slot = b.prefix_table[t // b.page], t % b.page
        k[p, :, slot], v[p, :, slot] = ahead[0, t], ahead[1, t]
    for s, n in enumerate(b.lengths):
        own = one(g, n, b.kv, b.dim)
        for t in range(n):
            p, slot = b.place(s, t)
            k[p, :, slot], v[p, :, slot] = own[0, t], own[1, t]
        tokens.append(np.concatenate([ahead, own], 1))
    return k, v, tokens


def one(g, n, kv, dim):
    keys, values = g.integers(-1, 2, (n, kv, dim)).astype(np.float64), g.choice([-1.0, -0.5, 0.5, 1.0], (n, kv, dim))
    last = n - n % 2
    keys[1:last:2] = keys[0:last:2]
    at = g.integers(0, dim, (last // 2, kv))
    for j in range(last // 2):
        for h in range(kv):
            keys[2 * j + 1, h, at[j, h]] = 0
    values[1:last:2] = -values[0:last:2]
    return np.stack([keys, values])


def queries(g, rows, n_q, dim):
    return g.choice([-1.0, 1.0], (rows, n_q, dim))


def bound(out, size, keys, largest, kind):
    """Of an attention that multiplies with weights in two parts.  Scores are exact; their product with scale log2(e), the factor and the
    difference from the maximum are rounded, 2^-24 of `largest` + 14 each and one more for the maximum's own, in numerator and denominator; an
    exponential is 2^-22 off, twice, and once more in a join; sums of `keys` terms 2^-23 a term, twice; a weight's second part half a step."""
    half = cases.HALF_STEP[kind]
    weight = 2 * 0.7 * 4 * (largest + 14) * 2.0 ** -24 + 3 * 2 * 2.0 ** -22 + 2 * keys * 2.0 ** -23 + half ** 2
    return half * np.abs(out) + weight * (1 + half) * size + 2.0 ** -25


def rounded_attention(b, tokens, q, scale, kind, parts):
    """The attention with its weights in one or two parts of the type, everything else in 64 bits."""
    out = np.zeros(q.shape)
    group = q.shape[1] // b.kv
    for s, n in enumerate(b.rows):
        k, v = tokens[s]
        for i in range(n):
            keys = b.prefix + b.lengths[s] - n + i + 1
            x = float(scale) * np.einsum("hd,khd->hk", q[b.start[s] + i], k[:keys].repeat(group, 1))
            p = np.exp(x - x.max(1, keepdims=True))
            used = cases.rounded(p, kind)
            if parts == 2:
                used = used + cases.rounded(p - used, kind)
            out[b.start[s] + i] = np.einsum("hk,khd->hd", used, v[:keys].repeat(group, 1)) / p.sum(1)[:, None]
    return cases.rounded(out, kind)


def largest_score(b, tokens, q, scale):
    """|score scale log2(e)| at most."""
    return max(float(np.abs(np.einsum("rhd,khd->rhk", q[b.start[s]:b.start[s] + n], tokens[s][0].repeat(q.shape[1] // b.kv, 1))).max(initial=0)) for s, n in enumerate(b.rows) if n) * abs(float(scale)) * 1.4427
