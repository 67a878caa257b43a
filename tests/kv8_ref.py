"""The 8-bit KV cache of include/iek.h in numpy, 64 bits, one sequence and head after the other."""
import numpy as np
import torch

BLOCK = 32
TOP = {"i8": 127.0, "e4m3": 448.0}


def decode(codes: np.ndarray, dtype: str) -> np.ndarray:
    """Code bytes (uint8) as values."""
    if dtype == "i8":
        return codes.view(np.int8).astype(np.float64)
    return torch.from_numpy(np.ascontiguousarray(codes)).view(torch.float8_e4m3fn).double().numpy()


def rounded(x: np.ndarray, dtype: str) -> np.ndarray:
    """x to the nearest code value, ties to even."""
    if dtype == "i8":
        return np.rint(x)
    mag = np.maximum(np.abs(x), 2.0 ** -6)
    step = 2.0 ** (np.floor(np.log2(mag)) - 3)
    return np.rint(x / step) * step


def scale_of(amax: float, dtype: str) -> float:
    if not np.isfinite(amax):
        return np.nan
    s = 2.0 ** -100
    while amax > TOP[dtype] * s:
        s *= 2
    return s


class Cache:
    """values of slot j: code[b, h, j] * scale[b, h, j // 32], codes as values."""

    def __init__(self, batch, kv, cap, hd, dtype):
        nblk = -(-cap // BLOCK)
        self.dtype, self.cap = dtype, cap
        self.code = [np.zeros((batch, kv, cap, hd)) for _ in range(2)]
        self.scale = [np.zeros((batch, kv, nblk)) for _ in range(2)]

    def value(self, which, b, h, n):
        s = self.scale[which][b, h, np.arange(n) // BLOCK]
        return self.code[which][b, h, :n] * s[:, None]

    def append(self, k, v, start, count):
        """k, v [batch][n][kv][hd]; returns the lengths."""
        lens = []
        for b, (st, ct) in enumerate(zip(start, count)):
            ct = min(ct, k.shape[1])
            ct = 0 if st < 0 or st > self.cap else max(0, min(ct, self.cap - st))
            lens.append(max(0, min(st, self.cap)) + ct)
            for which, x in ((0, k), (1, v)):
                for h in range(x.shape[2]):
                    for lo in range(st - st % BLOCK, st + ct, BLOCK) if ct else ():
                        a, e = max(lo, st), min(lo + BLOCK, st + ct)
                        rows = x[b, a - st:e - st, h].astype(np.float64)
                        s = scale_of(np.abs(rows).max(), self.dtype)
                        old = self.scale[which][b, h, lo // BLOCK]
                        if lo < st and not old <= s:
                            s = s if np.isnan(s) else old
                        if lo < st and s > old:
                            self.code[which][b, h, lo:st] = rounded(self.code[which][b, h, lo:st] * (old / s), self.dtype)
                        self.scale[which][b, h, lo // BLOCK] = s
                        if not np.isnan(s):
                            self.code[which][b, h, a:e] = rounded(rows / s, self.dtype)
        return lens

    def attention(self, q, lens, window, scale):
        """q [batch][n_q][heads][hd]; (out, weights [batch][kv][cap], a bound on the f32 errors of out)."""
        batch, n_q, heads, hd = q.shape
        kv = self.code[0].shape[1]
        group = heads // kv
        out, bound = np.zeros(q.shape), np.zeros(q.shape)
        weights = np.zeros((batch, kv, self.cap))
        for b, n in enumerate(lens):
            for h in range(kv):
                keys, vals = self.value(0, b, h, n), self.value(1, b, h, n)
                for t in range(n_q):
                    hi = n - (n_q - 1 - t)
                    lo = max(0, hi - window) if window else 0
                    if hi <= lo:
                        continue
                    qq = q[b, t, h * group:(h + 1) * group].astype(np.float64)
                    s = scale * (qq @ keys[lo:hi].T)
                    e = np.exp(s - s.max(1, keepdims=True))
                    p = e / e.sum(1, keepdims=True)
                    out[b, t, h * group:(h + 1) * group] = p @ vals[lo:hi]
                    weights[b, h, lo:hi] += p.sum(0)
                    # A score is a sum of hd products (each q held to 2^-22 of its size): off by at most
                    # (hd + 16) 2^-24 of the sum of the products' sizes. That error moves a weight by as
                    # much relatively, once as numerator and once in the sum; the sums over entries go
                    # 32 at a time, then over tiles, waves and at most 256 chunks.
                    size = scale * (np.abs(qq) @ np.abs(keys[lo:hi]).T).max(1, keepdims=True)
                    rel = (2 * (hd + 16) * size + 32 + n / 32 + 300) * 2.0 ** -24
                    # A share may be held in fixed point relative to the largest of its block: as a pair of
                    # fp16, of 2^14 p and of 2^11 times the rest, it is off by at most half of fp16's smallest
                    # step, 2^-25 2^-11 2^-14 = 2^-50, of the largest share (2^-49 for a cut rest).
                    fixed = (hi - lo) * 2.0 ** -49 * np.abs(vals[lo:hi]).max(0)
                    bound[b, t, h * group:(h + 1) * group] = rel * (p @ np.abs(vals[lo:hi])) + fixed
        return out, weights, bound

    def kept(self, w, n, keep, first, last):
        """The slots of one head that an eviction keeps."""
        slots = np.arange(n)
        if n <= keep:
            return slots
        mid = slots[first:n - last]
        x = w[first:n - last].astype(np.float64)
        key = np.where(np.isnan(x), np.inf, x)
        best = mid[np.lexsort((mid, -key, ~np.isnan(x)))[:keep - first - last]]
        return np.concatenate([slots[:first], np.sort(best), slots[n - last:]])

    def evict(self, w, lens, keep, first, last, cap=None):
        """(the cache that is left, its weights, lengths and old slots per sequence and head)"""
        batch, kv, _, hd = self.code[0].shape
        to = Cache(batch, kv, cap or self.cap, hd, self.dtype)
        w_out = np.zeros((batch, kv, to.cap))
        index = {}
        for b, n in enumerate(lens):
            for h in range(kv):
                left = index[b, h] = self.kept(w[b, h], n, keep, first, last)
                w_out[b, h, :len(left)] = w[b, h, left]
                for which in range(2):
                    was = self.scale[which][b, h, left // BLOCK]
                    for lo in range(0, len(left), BLOCK):
                        s = was[lo:lo + BLOCK].max()  # (NaN if one is)
                        rows = self.code[which][b, h, left[lo:lo + BLOCK]]
                        if not np.isnan(s):
                            rows = rounded(rows * (was[lo:lo + BLOCK] / s)[:, None], self.dtype)
                        to.code[which][b, h, lo:lo + len(rows)] = rows
                        to.scale[which][b, h, lo // BLOCK] = s
        return to, w_out, [min(n, keep) for n in lens], index
