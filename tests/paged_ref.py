"""The paged cache and the filters of sampling in 64 bits: what the device entries compute, from their definitions."""
import numpy as np


class Paged:
    """Pools [n_pages][kv][page][hd] as float64 and page numbers [batch][max_pages]."""

    def __init__(self, n_pages, kv, page, hd, table, dtype):
        self.k, self.v = (np.full((n_pages, kv, page, hd), np.nan) for _ in range(2))
        self.page, self.table, self.dtype = page, np.asarray(table).astype(np.int64), dtype
        self.n_pages, self.kv, self.hd = n_pages, kv, hd

    def hold(self, x):
        with np.errstate(over="ignore"):
            return x.astype(np.float16 if self.dtype == "f16" else np.float32).astype(np.float64)

    def append(self, k, v, start, count):
        """Rows [batch][n][kv][hd] (f32, rotated already); the lengths."""
        cap, lens = self.table.shape[1] * self.page, []
        for b, (st, c) in enumerate(zip(start, count)):
            c = min(max(c, 0), k.shape[1])
            c = 0 if st < 0 or st > cap else min(c, cap - st)
            lens.append(max(0, min(st, cap)) + c)
            for i in range(c):
                p = self.table[b, (st + i) // self.page]
                if 0 <= p < self.n_pages:
                    self.k[p, :, (st + i) % self.page] = self.hold(k[b, i])
                    self.v[p, :, (st + i) % self.page] = self.hold(v[b, i])
        return lens

    def places(self, pages, lo, hi):
        """(entries of [lo, hi) that have a page, their pages, their slots)"""
        j = np.arange(lo, hi)
        p = np.asarray(pages)[j // self.page] if len(j) else j
        there = (p >= 0) & (p < self.n_pages)
        return j[there], p[there], j[there] % self.page

    def attention(self, q, lens, window, scale, shared=0, shared_pages=()):
        """q [batch][n_q][heads][hd]; (out, a bound on the errors of out)."""
        batch, n_q, heads, hd = q.shape
        group = heads // self.kv
        out, bound = np.zeros(q.shape), np.zeros(q.shape)
        for b, n in enumerate(lens):
            common, rest = self.places(shared_pages, 0, min(n, shared)), self.places(self.table[b], min(n, shared), n)
            at, pages, slots = (np.concatenate(x) for x in zip(common, rest))
            rows = [pool[pages, :, slots] for pool in (self.k, self.v)]
            for t in range(n_q):
                hi = n - (n_q - 1 - t)
                lo = max(0, hi - window) if window else 0
                seen = (at >= lo) & (at < hi)
                if not seen.any():
                    continue
                K, V = (x[seen].transpose(1, 0, 2) for x in rows)  # [kv][entries][hd]
                qq = q[b, t].astype(np.float64).reshape(self.kv, group, hd)
                with np.errstate(invalid="ignore"):
                    s = scale * (qq @ K.transpose(0, 2, 1))
                    e = np.exp(s - s.max(2, keepdims=True))
                    p = e / e.sum(2, keepdims=True)
                    out[b, t] = (p @ V).reshape(heads, hd)
                # A score is a sum of hd products, each q held to 2^-22 of its size: off by at most (hd + 16) 2^-24 of the
                # sum of the products' sizes (and q to 2^-38 of its row's largest: below that for rows whose values are of a
                # size). It moves a weight by as much relatively, once as numerator and once in the sum; a weight is
                # held to 2^-22, exp2 to 2^-22, the sums over entries go 16 or 32 at a time, then over tiles, waves
                # and at most 512 chunks.
                size = scale * (np.abs(qq) @ np.abs(K).transpose(0, 2, 1)).max(2, keepdims=True)
                rel = (2 * (hd + 16) * size + 48 + n / 16 + 600) * 2.0 ** -24
                # as a pair of fp16 numbers of 2^13 p, p relative to a maximum that is at most the largest share's: off by at most
                # 2^-25 2^-13 of the largest at fp16's lower end (f32 pages: nothing)
                fixed = seen.sum() * 2.0 ** -38 * np.abs(V).max(1, keepdims=True)
                bound[b, t] = (rel * (p @ np.abs(V)) + fixed).reshape(heads, hd)
        return out, bound


def rotated(x, rope):
    """Rows [..., heads, hd] f32 with adjacent pairs turned by rope [..., pairs, 2], each step rounded to f32."""
    y = x.copy()
    pairs = rope.shape[-2]
    a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
    c, s = rope[..., None, :, 0], rope[..., None, :, 1]
    y[..., 0:2 * pairs:2] = a * c - b * s
    y[..., 1:2 * pairs:2] = a * s + b * c
    return y


def sample(x, temperature, r, top_k=0, top_p=1.0, min_p=0.0):
    """(index, probability) of one row; (0xFFFFFFFF, NaN) where there is no token."""
    x = np.asarray(x, np.float32).astype(np.float64) + 0.0
    t, r, top_p, min_p = (float(np.float32(a)) for a in (temperature, r, top_p, min_p))
    top = x.max()
    if not (np.isfinite(top) and 0 <= t < np.inf and 0 <= r < 1 and top_p == top_p and min_p == min_p):
        return 0xFFFFFFFF, np.nan
    if t == 0:
        return int(np.argmax(x)), 1.0
    order = np.argsort(-x, kind="stable")
    if 0 < top_k < len(x):
        order = order[:top_k]
    w = np.exp((x - top) / t)
    ranked = w[order]
    keep = ranked >= min(min_p, 1.0)
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(ranked)[:-1]])
        keep &= (before < top_p * ranked.sum()) | (np.arange(len(order)) == 0)
    kept = np.zeros_like(w)
    kept[order[keep]] = ranked[keep]
    upto = np.cumsum(kept)
    i = int(np.searchsorted(upto, r * upto[-1], side="right"))
    return i, kept[i] / upto[-1]
