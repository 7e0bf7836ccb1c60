"""A plain 64-bit implementation of the 4-bit cache (include/we_cache4.h) in numpy, for its tests."""
import numpy as np

import oracle_lib as O
import we

NP = {we.F32: np.float32, we.F16: np.uint16, we.BF16: np.uint16}
HALF_STEP = {we.F32: 2.0 ** -24, we.F16: 2.0 ** -11, we.BF16: 2.0 ** -8}  # of a rounding to the type, relative


def store(x, dtype):
    """x rounded to the type, as the array that is uploaded"""
    x = np.asarray(x, np.float32)
    if dtype == we.F32:
        return x.copy()
    if dtype == we.F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    return O.bf16_rne(x.reshape(-1)).reshape(x.shape)


def value(a, dtype):
    """the f64 values of an array of the type"""
    if dtype == we.F32:
        return a.astype(np.float64)
    if dtype == we.F16:
        return a.view(np.float16).astype(np.float64)
    return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def quantize(x):
    """codes u8 [..., dim / 2] and scales u32 [..., dim / 64] of x (f64 values of f32 numbers), with the format's f32 steps"""
    g = x.astype(np.float32).reshape(*x.shape[:-1], x.shape[-1] // 64, 64)
    with np.errstate(invalid="ignore", divide="ignore"):
        g = np.clip(g, np.float32(-65504), np.float32(65504))
        lo, hi = g.min(-1), g.max(-1)  # a NaN stays one
        mn, sc = lo.astype(np.float16), ((hi - lo) / np.float32(15)).astype(np.float16)
        mn[np.isnan(lo)] = sc[np.isnan(lo)] = np.uint16(0x7e00).view(np.float16)
        s = sc.astype(np.float32)[..., None]
        u = np.where(s > 0, np.clip(np.rint((g - mn.astype(np.float32)[..., None]) / s), 0, 15), 0).astype(np.uint8)
    u = u.reshape(x.shape)
    codes = u[..., 0::2] | (u[..., 1::2] << 4)
    return codes, sc.view(np.uint16).astype(np.uint32) | (mn.view(np.uint16).astype(np.uint32) << 16)


def dequantize(codes, scales):
    u = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1]).astype(np.float64)
    sc = (scales & 0xffff).astype(np.uint16).view(np.float16).astype(np.float64).repeat(64, -1)
    mn = (scales >> 16).astype(np.uint16).view(np.float16).astype(np.float64).repeat(64, -1)
    with np.errstate(invalid="ignore"):
        return mn + sc * u


class Cache:
    """A cache's bytes on the host: the four regions as views of one array."""

    def __init__(self, batch, kv, dim, cap, fill=None):
        rows = batch * kv * cap
        self.batch, self.kv, self.dim, self.cap = batch, kv, dim, cap
        self.bytes = np.zeros(rows * (dim + dim // 8), np.uint8)
        if fill is not None:  # anything, NaN scales included
            self.bytes[:] = fill.integers(0, 256, self.bytes.size, dtype=np.uint8)
        at = np.cumsum([0, rows * dim // 2, rows * dim // 16, rows * dim // 2, rows * dim // 16])
        shape = (batch, kv, cap)
        self.kc, self.vc = (self.bytes[at[i]:at[i + 1]].reshape(*shape, dim // 2) for i in (0, 2))
        self.ks, self.vs = (self.bytes[at[i]:at[i + 1]].view(np.uint32).reshape(*shape, dim // 64) for i in (1, 3))

    def put(self, b, slot, k, v):
        """K and V rows [n, kv, dim] into slots slot .. of sequence b"""
        n = k.shape[0]
        for x, codes, scales in ((k, self.kc, self.ks), (v, self.vc, self.vs)):
            c, s = quantize(x.swapaxes(0, 1))
            codes[b, :, slot:slot + n], scales[b, :, slot:slot + n] = c, s

    def values(self, b, n):
        """K and V [kv, n, dim] of the first n slots"""
        return (dequantize(self.kc[b, :, :n], self.ks[b, :, :n]), dequantize(self.vc[b, :, :n], self.vs[b, :, :n]))

    def handle(self, graph):
        return we.Cache4(graph, self.batch, self.kv, self.dim, self.cap, data=graph.buffer(self.bytes))


def attention(cache, q, lens, counts, causal):
    """(out [b, tokens, heads, dim] with NaN in the rows that are left alone, received [b, kv, cap], and per sequence the
    bounds (a, v): the largest sum of |q| |K| / sqrt(dim) and the largest |minimum| + 15 scale of V) in f64"""
    b, tokens, heads, dim = q.shape
    group = heads // cache.kv
    out = np.full(q.shape, np.nan)
    received = np.zeros((b, cache.kv, cache.cap))
    bounds = []
    for i in range(b):
        n, c = max(0, min(lens[i], cache.cap)), max(0, min(counts[i], tokens))
        k, v = cache.values(i, n)
        big = 0.0
        for h in range(heads):
            g = h // group
            for t in range(c):
                vis = n - c + t + 1 if causal else n
                out[i, t, h] = 0
                if vis <= 0:
                    continue
                s = k[g, :vis] @ q[i, t, h] / np.sqrt(dim)
                big = max(big, (np.abs(k[g, :vis]) @ np.abs(q[i, t, h])).max() / np.sqrt(dim))
                p = np.exp(s - s.max())
                p /= p.sum()
                out[i, t, h] = p @ v[g, :vis]
                received[i, g, :vis] += p
        sc = (cache.vs[i, :, :n] & 0xffff).astype(np.uint16).view(np.float16).astype(np.float64)
        mn = (cache.vs[i, :, :n] >> 16).astype(np.uint16).view(np.float16).astype(np.float64)
        bounds.append((big, (np.abs(mn) + 15 * sc).max() if n else 0.0))
    return out, received, bounds


def tolerance(want, bounds, dtype):
    """What an output row may be off, per sequence [b, 1, 1, 1] and value. With A the sum of |q K| / sqrt(dim) of a score and
    V the largest |minimum| + 15 scale:
      * a score is a sum of dim products in f32 (fewer than 16 roundings of partial sums below 3 A: code, minimum and their
        total) of q in 22 bits or more: off by 16 * 3 A 2^-24 + A 2^-22 < 52 A 2^-24, its probability by that and 2^-21 (exp2
        and its argument) of itself; with the same in the denominator, the output by twice that times V;
      * p times the scale rounds to f16 (half a step 2^-12: 11 bits; as two f16 values, F32: 2^-23), V's codes are exact;
      * the sums over slots in f32: below 64 roundings that meet a partial sum of at most V: 2^-18 V;
      * the result rounds to its type."""
    tol = []
    for i, (a, v) in enumerate(bounds):
        p = 52 * a * 2.0 ** -24 + 2.0 ** -21
        tol.append((2 * p + (2.0 ** -23 if dtype == we.F32 else 2.0 ** -12) + 2.0 ** -18) * v)
    return np.abs(np.nan_to_num(want)) * HALF_STEP[dtype] + np.array(tol).reshape(-1, 1, 1, 1)


def weight_tolerance(received, bounds):
    """received sums probabilities, each off by 2 p of itself as above, in f32 (2^-20 covers 16 roundings of partial sums)."""
    p = np.array([52 * a * 2.0 ** -24 + 2.0 ** -21 for a, _ in bounds]).reshape(-1, 1, 1)
    return received * (2 * p + 2.0 ** -20) + 2.0 ** -40


def evict(cache, keep, lens, weight, pos, seen, sinks, recent):
    """(lens, weight, pos) after the eviction; moves the cache's rows in place"""
    weight, pos, left_of = weight.copy(), pos.copy(), []
    for i, n in enumerate(lens):
        n = max(0, min(n, cache.cap))
        left = min(n, keep)
        left_of.append(left)
        for g in range(cache.kv):
            w, p = weight[i, g, :n] + 0.0, pos[i, g, :n].astype(np.int64)
            key = np.where(np.isnan(w), np.inf, w)
            safe = (p < sinks) | (p >= seen[i] - recent)
            out = np.lexsort((np.arange(n), np.isnan(w), key, safe))[:n - left]
            stays = np.ones(n, bool)
            stays[out] = False
            come = np.arange(left)
            come[~stays[:left]] = left + np.flatnonzero(stays[left:])
            for a in (weight, pos, cache.kc, cache.ks, cache.vc, cache.vs):
                a[i, g, :left] = a[i, g][come]
    return left_of, weight, pos
