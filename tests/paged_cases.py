"""A packed batch over a paged cache in numpy, and its operators from their formulas in 64 bits."""
import numpy as np

HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}  # a rounding, relative to the value


def to_bits(a, kind):
    """Values as the device holds them (bf16: round to nearest even, in the upper half of an fp32)."""
    if kind == "f32":
        return np.asarray(a, np.float32)
    if kind == "f16":
        return np.asarray(a, np.float16)
    u = np.asarray(a, np.float32).view(np.uint32)
    up = ((u >> 16) & 1) + 0x7FFF
    return np.where(np.isnan(np.asarray(a, np.float32)), 0x7FC0, (u + up) >> 16).astype(np.uint16)


def from_bits(a, kind):
    if kind == "bf16":
        return (np.asarray(a, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return np.asarray(a).astype(np.float64)


def rounded(a, kind):
    return from_bits(to_bits(a, kind), kind)


class Batch:
    """Sequences of `rows` new rows and `lengths` tokens on pages handed out in no order; pools [pages, kv, page, dim] as seen."""

    def __init__(self, g, rows, lengths, page, kv, dim, prefix=0, order="heads", spare=2, behind=0):
        self.rows, self.lengths, self.page, self.kv, self.dim, self.prefix, self.order = list(rows), list(lengths), page, kv, dim, prefix, order
        self.start = np.concatenate([[0], np.cumsum(self.rows)]).astype(np.int32)
        self.live, self.total = int(self.start[-1]), int(self.start[-1]) + behind
        need, wide = [-(-n // page) for n in self.lengths], -(-prefix // page)
        self.pages = sum(need) + wide + spare
        ids = g.permutation(self.pages).astype(np.int32)
        self.table = np.full((len(self.rows), max(1, max(need, default=1)) + 1), -7, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = ids[at:at + n]
            at += n
        self.prefix_table = ids[at:at + wide] if wide else np.zeros(1, np.int32)

    def strides(self):
        page, kv, dim = self.page, self.kv, self.dim
        return (kv * page * dim, page * dim, dim) if self.order == "heads" else (kv * page * dim, dim, kv * dim)

    def memory(self, pool):
        """A pool as it lies in memory."""
        return np.ascontiguousarray(pool if self.order == "heads" else pool.transpose(0, 2, 1, 3))

    def seen(self, memory):
        """The other way."""
        a = memory.reshape((self.pages, self.kv, self.page, self.dim) if self.order == "heads" else (self.pages, self.page, self.kv, self.dim))
        return a if self.order == "heads" else a.transpose(0, 2, 1, 3)

    def place(self, s, token):
        return self.table[s, token // self.page], token % self.page

    def fill(self, g, value):
        """Pools whose places without a token hold `value`, and of every sequence its tokens' keys and values [prefix + length, kv, dim]."""
        k = np.full((self.pages, self.kv, self.page, self.dim), value, np.float64)
        v = k.copy()
        ahead = g.standard_normal((2, self.prefix, self.kv, self.dim))
        for t in range(self.prefix):
            k[self.prefix_table[t // self.page], :, t % self.page], v[self.prefix_table[t // self.page], :, t % self.page] = ahead[0, t], ahead[1, t]
        tokens = []
        for s, n in enumerate(self.lengths):
            own = g.standard_normal((2, n, self.kv, self.dim))
            for t in range(n):
                p, i = self.place(s, t)
                k[p, :, i], v[p, :, i] = own[0, t], own[1, t]
            tokens.append(np.concatenate([ahead, own], 1))
        return k, v, tokens


def rotate(x, angle, factor, layout):
    """x [rows, heads, dim], angle [rows, pairs]."""
    y, n = np.array(x, np.float64), 2 * angle.shape[1]
    a, b = (slice(0, n // 2), slice(n // 2, n)) if layout == 1 else (slice(0, n, 2), slice(1, n, 2))
    c, s = factor * np.cos(angle)[:, None], factor * np.sin(angle)[:, None]
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def attend(batch, tokens, q, scale, window=0):
    """Outputs and, for a bound, sum p |v| and sum p |scale| |q| |k| of every row and head; q [rows, n_q, dim]."""
    out, size, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
    group = q.shape[1] // batch.kv
    for s, n in enumerate(batch.rows):
        k, v = tokens[s]
        for i in range(n):
            r, mine = batch.start[s] + i, batch.prefix + batch.lengths[s] - n + i
            lo = max(0, mine + 1 - window) if window else 0
            keys = np.arange(lo, mine + 1) if mine >= batch.prefix else np.zeros(0, int)  # a row without a token sees nothing
            if not keys.size:
                continue
            kk, vv = k[keys].repeat(group, 1), v[keys].repeat(group, 1)  # [keys, n_q, dim]
            x = scale * np.einsum("hd,khd->hk", q[r], kk)
            p = np.exp(x - x.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            out[r], size[r] = np.einsum("hk,khd->hd", p, vv), np.einsum("hk,khd->hd", p, np.abs(vv))
            reach[r] = (abs(scale) * np.einsum("hd,khd->hk", np.abs(q[r]), np.abs(kk))).max(1)
    return out, size, reach


def attend_bound(out, size, reach, kind, dim):
    """Half a step of the output; of each weight: the products' fp32 sums (dim terms of at most `reach` in all, twice: numerator
    and denominator), the exponential and the long sums (2^-15), and one rounding of the weight to the type."""
    weight = 2 * (dim + 4) * 2.0 ** -24 * reach[..., None] + 2.0 ** -15 + HALF_STEP[kind]
    return HALF_STEP[kind] * np.abs(out) + weight * (1 + HALF_STEP[kind]) * size + 1e-7


def law(x, t):
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    p = np.zeros(x.size)
    if x.max() == -np.inf:
        return p
    if not t > 0:
        p[int(np.argmax(x))] = 1
        return p
    p = np.exp((x - x.max()) / float(np.float32(t)))
    return p / p.sum()


def verify(start, target, draft, tokens, temperature, random):
    """target [rows, vocab], draft [steps, seqs, vocab] or None; (out_tokens, accepted)."""
    out, kept = np.full(len(tokens), -99, np.int32), []
    for s in range(len(start) - 1):
        r0, n = start[s], start[s + 1] - start[s]
        if n <= 0:
            kept.append(0)
            continue
        t, line = temperature[s], []
        p = None
        for j in range(n):
            p = law(target[r0 + j], t)
            if j == n - 1:
                break
            x = tokens[r0 + 1 + j]
            inside = 0 <= x < p.size
            q = np.zeros(p.size) if draft is None else law(draft[j, s], t)
            if draft is None and inside:
                q[x] = 1
            if not (inside and (p[x] > 0 if not t > 0 else float(random[r0 + j]) * q[x] < p[x])):
                rest = np.maximum(p - q, 0)
                if t > 0 and rest.sum() > 0:
                    p = rest
                break
            line.append(x)
        run = np.cumsum(p)
        if run[-1] > 0:
            past = np.nonzero((run > float(random[r0 + n - 1]) * run[-1]) & (p > 0))[0]
            drawn = int(past[0]) if past.size else int(np.nonzero(p)[0][-1])
        else:
            drawn = -1
        kept.append(len(line))
        out[r0:r0 + n] = line + [drawn] + [-1] * (n - len(line) - 1)
    return out, np.array(kept, np.int32)
