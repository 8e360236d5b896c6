"""Bit patterns of 16-bit types and the inputs of the decoder-layer tests."""
import numpy as np

from oracle import layer as ol

F32, F16, BF16 = 0, 1, 2
#: a rounding to the type is off by at most half a step, relative to the value
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
#: ... or by half of the smallest subnormal
HALF_TINY = {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134}
FORMATS = {"int8": 0, "e4m3": 1, "e5m2": 2}


def to_bits(x, kind):
    x = np.asarray(x, np.float32)
    if kind == F32:
        return x
    if kind == F16:
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32).astype(np.uint64)
    out = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), out).astype(np.uint16)


def from_bits(b, kind):
    if kind == F32:
        return b.astype(np.float64)
    if kind == F16:
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def fp8_values(b, fmt):
    """The values of fp8 bit patterns, by the formats' definition."""
    b = b.astype(np.int64)
    sign = np.where(b & 0x80, -1.0, 1.0)
    if fmt == "e4m3":
        e, m = (b >> 3) & 15, b & 7
        v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * np.exp2(e - 10.0))
        return sign * np.where((b & 0x7F) == 0x7F, np.nan, v)
    e, m = (b >> 2) & 31, b & 3
    v = np.where(e == 0, m * 2.0 ** -16, (4 + m) * np.exp2(e - 17.0))
    return sign * np.where(e == 31, np.where(m == 0, np.inf, np.nan), v)


class Paged:
    """A paged cache and the requests on it: pages in random order, whatever lies behind a request's last key."""

    def __init__(self, rng, cached, new, heads, kv_heads, dim, page, kind, pad=0, slack_pages=2, garbage=0.0, width_slack=0):
        self.heads, self.kv_heads, self.dim, self.page, self.kind, self.pad = heads, kv_heads, dim, page, kind, pad
        self.cached, self.new = np.array(cached, np.int32), np.array(new, np.int32)
        n = len(cached)
        self.kv = (self.cached + self.new).astype(np.int32)
        self.cu = np.concatenate(([0], np.cumsum(self.new))).astype(np.int32)
        have = [-(-int(k) // page) for k in self.kv]
        self.width = max(have + [1]) + width_slack
        pages = sum(have) + slack_pages
        order = rng.permutation(pages).astype(np.int32)
        self.table = np.full((n, self.width), -1, np.int32)
        at = 0
        for r in range(n):
            self.table[r, :have[r]] = order[at:at + have[r]]
            at += have[r]
        shape = (pages, kv_heads, page, dim)
        self.k_bits = to_bits(rng.standard_normal(shape), kind)
        self.v_bits = to_bits(rng.standard_normal(shape), kind)
        if garbage is not None and not garbage == 0.0:
            used = np.zeros((pages, page), bool)
            for r in range(n):
                for j in range(int(self.kv[r])):
                    used[self.table[r, j // page], j % page] = True
            hole = ~used[:, None, :, None] & np.ones(shape, bool)
            self.k_bits[hole] = to_bits(np.float32(garbage), kind)
            self.v_bits[hole] = to_bits(np.float32(garbage), kind)
        self.tokens = int(self.cu[-1]) + pad
        self.q_bits = to_bits(1.5 * rng.standard_normal((self.tokens, heads, dim)), kind)
        self.out_bits = to_bits(rng.standard_normal((self.tokens, heads, dim)), kind)
        self.scale = float(np.float32(dim ** -0.5))

    def expected(self, window=0):
        k, v = from_bits(self.k_bits, self.kind), from_bits(self.v_bits, self.kind)
        q, out = from_bits(self.q_bits, self.kind), from_bits(self.out_bits, self.kind)
        want = ol.paged_attention(q, self.cu, self.kv, self.table, k, v, self.scale, window, out)
        spread = ol.paged_attention(q, self.cu, self.kv, self.table, k, np.abs(v), self.scale, window, np.abs(out))
        return want, spread

    def tolerance(self, want, spread):
        """Elementwise, from the roundings that the operator documents.  With u half a step of the type: the result is
        rounded once (u |want|); every probability is rounded for the product with V (u of sum p |v| = u * spread, and
        half of the type's smallest subnormal for each of the n keys, against a sum that is at least 1); the fp32 sums
        of the scores (dim products, then the scaling) move a score by at most ds = (dim + 2) 2**-23 |q| |k| scale, a
        probability by twice that relative; the fp32 sums over n keys and the power of two by (n + 8) 2**-23."""
        u, tiny = HALF_STEP[self.kind], HALF_TINY[self.kind]
        k, q = from_bits(self.k_bits, self.kind), from_bits(self.q_bits, self.kind)
        v = from_bits(self.v_bits, self.kind)
        fin = lambda x: np.where(np.isfinite(x), x, 0.0)  # noqa: E731
        norm = lambda x: np.sqrt((fin(x) ** 2).sum(-1)).max(initial=0.0)  # noqa: E731
        n = int(self.kv.max(initial=0))
        ds = (self.dim + 2) * 2.0 ** -23 * norm(k) * norm(q) * self.scale
        return u * np.abs(want) + (1 + u) * (u + 2 * ds + (n + 8) * 2.0 ** -23) * spread + n * tiny * np.abs(fin(v)).max(initial=0.0) + tiny
