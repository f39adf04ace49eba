"""Plain implementations in 64 bits of the operators of a served batch, and batches for their tests."""
import math

import numpy as np


def rope_frequencies(rot, theta, kind=None, factor=1.0, original=0, beta_fast=32.0, beta_slow=1.0, factors=None):
    f = np.array([theta ** (-2.0 * i / rot) for i in range(rot // 2)])
    magnitude = 1.0
    if factors is not None:
        f = f / np.asarray(factors, dtype=np.float32).astype(np.float64)
    if kind == "linear":
        f = f / factor
    if kind == "yarn":
        lo = max(0, math.floor(rot * math.log(original / (2 * math.pi * beta_fast)) / (2 * math.log(theta))))
        hi = min(rot - 1, math.ceil(rot * math.log(original / (2 * math.pi * beta_slow)) / (2 * math.log(theta))))
        g = np.clip((np.arange(rot // 2) - lo) / max(hi - lo, 0.001), 0, 1)
        f = f * (1 - g) + f / factor * g
        magnitude = 0.1 * math.log(factor) + 1
    return f, magnitude


def rotate(x, positions, f, magnitude, interleaved):
    """x [tokens, heads, head_dim]."""
    x = np.asarray(x, dtype=np.float64)
    y, n = x.copy(), len(f)
    angle = np.outer(np.asarray(positions, dtype=np.float64), f)
    c, s = magnitude * np.cos(angle)[:, None, :], magnitude * np.sin(angle)[:, None, :]
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    if interleaved:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = a * c - b * s, a * s + b * c
    else:
        y[..., :n], y[..., n:2 * n] = a * c - b * s, a * s + b * c
    return y


def rotation_bound(x, f, magnitude, interleaved):
    """Sine and cosine are off by at most 2^-23 (conversion, product and constant of the angle 3 x 2^-25 pi / 4, the series 2^-24), the magnitude and the
    products add 2 x 2^-25 each: below 2^-22 of |a| + |b|."""
    z = rotate(np.abs(np.asarray(x, dtype=np.float64)), np.zeros(len(x)), f, magnitude, interleaved)
    n = len(f)
    out = np.zeros_like(z)
    a, b = (z[..., 0:2 * n:2], z[..., 1:2 * n:2]) if interleaved else (z[..., :n], z[..., n:2 * n])
    if interleaved:
        out[..., 0:2 * n:2] = out[..., 1:2 * n:2] = a + b
    else:
        out[..., :n] = out[..., n:2 * n] = a + b
    return out * 2.0 ** -22


class Batch:
    """counts: rows of each sequence; lens: its positions then.  Pages are drawn from a pool; the leading `shared` ones are everybody's."""

    def __init__(self, rng, counts, lens, page, shared=0, pad_rows=0, spare=3, pages=None, max_len=None):
        self.counts, self.lens, self.page, self.shared = list(counts), list(lens), page, shared
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.tokens = int(self.starts[-1]) + pad_rows
        self.max_len = max([1] + list(lens)) if max_len is None else max_len
        n = len(self.counts)
        self.width = max(shared, -(-self.max_len // page))
        need = shared + n * (self.width - shared)
        self.pages = need + spare if pages is None else pages
        ids = rng.permutation(self.pages)[:need].astype(np.int32)
        self.tables = np.concatenate([np.tile(ids[:shared], (n, 1)), ids[shared:].reshape(n, self.width - shared)], 1).astype(np.int32)

    def places(self):
        """(row, sequence, position) of every row of a sequence."""
        return [(int(self.starts[s]) + j, s, self.lens[s] - c + j) for s, c in enumerate(self.counts) for j in range(c)]


def attention(q, k, v, batch, scale):
    """q [tokens, heads, hd], k and v [pages, kv, page, hd] -> y of the rows of sequences (zero where nothing is seen), and a bound per row."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    kv, hd = k.shape[1], k.shape[3]
    heads = q.shape[1]
    group = heads // kv
    y, bound = np.zeros_like(q), np.zeros((q.shape[0], heads))
    for row, s, pos in batch.places():
        if pos < 0:
            continue
        ids = batch.tables[s][: pos // batch.page + 1]
        ks = k[ids].transpose(1, 0, 2, 3).reshape(kv, -1, hd)[:, : pos + 1]
        vs = v[ids].transpose(1, 0, 2, 3).reshape(kv, -1, hd)[:, : pos + 1]
        for h in range(heads):
            z = scale * (ks[h // group] @ q[row, h])
            w = np.exp(z - z.max())
            w /= w.sum()
            y[row, h] = w @ vs[h // group]
            # a score is off by (hd + 8) 2^-24 of the sum of its products' magnitudes (sums in FP32; two FP16 parts of q leave 2^-22 of each), a weight by
            # that and 2^-21; both ends of the division; then one rounding per product of 16 keys
            ds = (hd + 8) * 2.0 ** -24 * abs(scale) * (np.abs(ks[h // group]) @ np.abs(q[row, h])).max() + 2.0 ** -20
            bound[row, h] = (2 * ds + (len(z) / 16 + 64) * 2.0 ** -24) * np.abs(vs[h // group]).max()
    return y, bound


def verify(logits, starts, tokens, q, temperatures, uniforms):
    """(out [rows], accepted [sequences]); rows of no sequence keep -7."""
    logits = np.asarray(logits, dtype=np.float64)
    out, accepted = np.full(logits.shape[0], -7, dtype=np.int32), np.zeros(len(temperatures), dtype=np.int32)
    vocab = logits.shape[1]

    def p_of(r, t):
        z = np.where(np.isnan(logits[r]), -np.inf, logits[r])
        if t <= 0 or not z.max() > -np.inf:
            p = np.zeros(vocab)
            finite = np.where(np.isnan(logits[r]), -1.0, (z == z.max()).astype(float))
            p[int(np.argmax(finite))] = 1.0
            return p
        with np.errstate(invalid="ignore"):
            w = np.where(z == z.max(), 1.0, np.exp((z - z.max()) / np.float64(t)))
        return w / w.sum()

    for s, t in enumerate(np.asarray(temperatures, dtype=np.float64)):
        a, b = int(starts[s]), int(starts[s + 1])
        if a == b:
            continue
        out[a:b] = -1
        r, kept = a, 0
        rest = None
        while True:
            p = p_of(r, t)
            if r == b - 1:
                rest = p
                break
            x = int(tokens[r + 1])
            qx = 1.0 if q is None else (float(q[r][x]) if 0 <= x < vocab else 0.0)
            if 0 <= x < vocab and float(uniforms[r][0]) * qx < p[x]:
                out[r] = x
                kept += 1
                r += 1
                continue
            if t <= 0:
                rest = p
            elif q is None:
                rest = p.copy()
                if 0 <= x < vocab:
                    rest[x] = 0
            else:
                rest = np.maximum(p - np.asarray(q[r], dtype=np.float64), 0)
            break
        accepted[s] = kept
        c = np.cumsum(rest)
        u = 0.0 if t <= 0 else float(uniforms[r][1])
        hit = np.nonzero((c > u * c[-1]) & (rest > 0))[0]
        out[r] = int(hit[0]) if len(hit) else int(np.nonzero(rest > 0)[0][-1])
    return out, accepted
