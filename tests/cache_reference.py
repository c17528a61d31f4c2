"""The 4-bit cache from its definition (include/homcomp_cache.h), in numpy and 64 bits: what the cache's tests compare with."""
import numpy as np

EPS = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}   # a rounding is off by at most this times the value


def bf16_values(bits):
    return (np.asarray(bits, np.uint32) << 16).view(np.float32).astype(np.float64)


def quantise(x):
    """Rows [..., d] -> (codes, s, lo) with s, lo [..., d / 32] in 64 bits; a block that cannot be held has s = NaN."""
    x = np.asarray(x, np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    fine = np.isfinite(b).all(-1)
    b = np.where(fine[..., None], b, 0.0)
    low = b.min(-1)
    bits = low.astype(np.float32).view(np.uint32)
    lo_bits = (bits >> 16) + (((bits >> 31) != 0) & ((bits & 0xffff) != 0))
    lo = bf16_values(lo_bits)
    with np.errstate(over="ignore", invalid="ignore"):
        span = b.max(-1) - lo
        s16 = (span / 15).astype(np.float16)
        s16 = np.where(15 * s16.astype(np.float64) < span, np.nextafter(s16, np.float16(np.inf)), s16)
    fine &= np.isfinite(s16) & np.isfinite(lo)
    s = np.where(fine, s16.astype(np.float64), np.nan)
    lo = np.where(fine, lo, 0.0)
    codes = np.zeros(b.shape, np.int64)
    with np.errstate(invalid="ignore"):
        for j in range(15):
            codes += b >= lo[..., None] + (j + 0.5) * s[..., None]
    codes = np.where(s[..., None] > 0, codes, 0)
    return codes.reshape(x.shape), s, lo


def values(codes, s, lo):
    c = codes.reshape(*codes.shape[:-1], -1, 32)
    return (lo[..., None] + s[..., None] * c).reshape(codes.shape)


class Pages:
    """Reads the bytes of pages as the header describes them."""

    def __init__(self, raw, heads, d, page):
        self.nb, self.page, self.heads, self.d = d // 32, page, heads, d
        self.raw = np.asarray(raw, np.uint8).reshape(-1, heads, page // 32, 1280 * self.nb)

    def row(self, page, head, slot):
        """(codes, s, lo) of the key and of the value of one slot of a page, and all the byte places they lie at."""
        rec, t, nb = self.raw[page, head, slot // 32], slot % 32, self.nb
        j = np.arange(self.d)
        bit = 4 * (j % 8 // 2) + 16 * (j % 2)
        at_k = t * 16 * nb + (j % 32 // 8) * 4 * nb + 4 * (j // 32) + bit // 8
        bit_v = 4 * (j % 64 // 16)
        at_v = 512 * nb + (t // 8) * 128 * nb + (j // 64 * 16 + j % 16) * 16 + (t % 8) * 2 + bit_v // 8
        b = np.arange(nb)
        octet = ((t // 8) * nb + b) * 16 + (t % 8) * 2
        word = lambda at: rec[at].astype(np.uint16) | (rec[at + 1].astype(np.uint16) << 8)
        f16 = lambda w: w.view(np.float16).astype(np.float64)
        sides = [1024 * nb + octet, 1088 * nb + octet, 1152 * nb + (t * nb + b) * 2, 1216 * nb + octet]
        sk, sv, lk, lv = f16(word(sides[0])), f16(word(sides[1])), bf16_values(word(sides[2])), bf16_values(word(sides[3]))
        places = np.concatenate([at_k, at_v] + [x for s in sides for x in (s, s + 1)])
        return ((rec[at_k] >> (bit % 8)) & 15, sk, lk), ((rec[at_v] >> (bit_v % 8)) & 15, sv, lv), places

    def rows(self, table_row, head, n):
        """What slots 0 .. n - 1 of a sequence stand for: K, V [n, d], and which of them have a page."""
        k, v, there = np.zeros((n, self.d)), np.zeros((n, self.d)), np.zeros(n, bool)
        for slot in range(n):
            p = int(table_row[slot // self.page])
            if 0 <= p < len(self.raw):
                key, value, _ = self.row(p, head, slot % self.page)
                k[slot], v[slot], there[slot] = values(*key), values(*value), True
        return k, v, there


def attention(q, keys, vals, there, lengths, starts, group, scale, causal, window, type_, prior=None):
    """q [rows, heads, d] in 64 bits; keys, vals, there: per sequence and head.  Returns out, lse, weights (list per sequence of [heads, L])
    and how far each may be off (the same shapes), see `bounds` in the text below.

    Bounds.  One score: a product of 32 terms in 32 bits, one multiply-add per block, the product of the lo part (its 24 terms), two
    multiplications for the scale: under 64 + nb roundings of at most 2^-24 of M = |scale| sum |q| (s c + |lo|).  So |dS| <= (64 + nb) 2^-24 M = e.
    A weight exp(S - lse) is off by a factor of at most 1 + 2 e + 2^-20 (both exponents' errors; the power's own error and the running sum's
    L roundings are counted as 2^-20 + L 2^-24).  The output adds L terms w (s c + |lo|), then there is one rounding to the output's type.
    For 16-bit results a term is a product of w and x' as float16 numbers, 2^-11 of it for either rounding (of w: one part for bfloat16
    results, two for float16 ones, 2^-22), or of w in bfloat16 parts, 2^-8 or 2^-16: under 2^-8 and 2^-11 + 2^-16 in all; where numbers are
    below float16's normal ones 2^-24, which is under 2^-13 of a block's largest (s is at least 2^-13 there) and inside what 2 max |v| leaves.  For 32-bit results 2^-24."""
    heads, d = q.shape[1], q.shape[2]
    out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
    d_out, d_lse = np.zeros(q.shape), np.zeros(q.shape[:2])
    weights, d_weights = [], []
    part = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11 + 2.0 ** -16, "f32": 2.0 ** -24}[type_]
    for s, L in enumerate(lengths):
        first, n = starts[s], starts[s + 1] - starts[s]
        w = np.zeros((heads // group, L)) if prior is None else prior[s, :, :L].astype(np.float64).copy()
        dw = np.abs(w) * 2.0 ** -24
        for i in range(n):
            at = L - n + i
            j = np.arange(L)
            for g in range(heads):
                h = g // group
                see = there[s][h] & ((j <= at) if causal else True) & ((j > at - window) if window else True)
                if not see.any():
                    continue
                k, v = keys[s][h][see], vals[s][h][see]
                row = q[first + i, g]
                with np.errstate(invalid="ignore", over="ignore"):
                    sc = scale * (k @ row)
                    size = abs(scale) * (np.abs(k) + 2 * np.abs(k).max(-1, keepdims=True)) @ np.abs(row)   # s c + |lo| <= |x'| + 2 |lo|
                    top = sc.max()
                    p = np.exp(sc - top)
                    z = top + np.log(p.sum())
                    p = np.exp(sc - z)
                    out[first + i, g], lse[first + i, g] = p @ v, z
                    e = (64 + d / 32) * 2.0 ** -24 * size.max()
                    run = 2.0 ** -20 + L * 2.0 ** -24
                    d_lse[first + i, g] = e + run + abs(z) * 2.0 ** -22
                    big = p @ (np.abs(v) + 2 * np.nanmax(np.abs(v), -1, keepdims=True))   # (a block of NaNs says nothing about the others)
                    d_out[first + i, g] = big * (part + 2 * (e + run)) + EPS[type_] * np.abs(out[first + i, g])
                    w[h, see] += p
                    dw[h, see] += p * (2 * e + run + abs(z) * 2.0 ** -22) + 2.0 ** -23 * w[h, see]
        weights.append(w)
        d_weights.append(dw)
    return out, lse, weights, d_out, d_lse, d_weights


def evict(weights, lengths, keep, first, recent):
    """Per sequence and head the slots that stay, ascending."""
    stays = []
    for s, L in enumerate(lengths):
        for w in weights[s]:
            if L <= keep:
                stays.append(list(range(L)))
                continue
            mid = range(first, L - recent)
            order = sorted(mid, key=lambda j: (np.isnan(w[j]), 0.0 if np.isnan(w[j]) else -w[j], j))
            stays.append(sorted(list(range(first)) + list(order[:keep - first - recent]) + list(range(L - recent, L))))
    return stays
