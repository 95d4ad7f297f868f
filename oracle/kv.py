"""Oracle of the cached-attention operators (include/supra_kv.h) in float64: norms and rotation, the 8-bit cache and
attention over it. Plain numpy, written from the definitions; test infrastructure only."""

from __future__ import annotations

import numpy as np

BLOCK = 32
EPS = {"F32": 2.0 ** -23, "F16": 2.0 ** -10, "BF16": 2.0 ** -7}  # finfo(t).eps


# ---- the row types: host arrays of their bits, and the float64 values they hold

def to_type(x: np.ndarray, dtype: str) -> np.ndarray:
    """x rounded to the type, as an array the device buffers take (bfloat16: its 16 bits)."""
    x = np.asarray(x)
    if dtype == "F32":
        return x.astype(np.float32)
    if dtype == "F16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    u = x.astype(np.float32).view(np.uint32)
    r = (u + 0x7FFF + ((u >> 16) & 1)) >> 16
    r = np.where((u & 0x7FFFFFFF) > 0x7F800000, (u >> 16) | 0x40, r)
    return r.astype(np.uint16)


def values(a: np.ndarray, dtype: str) -> np.ndarray:
    """The float64 values of such an array."""
    if dtype == "BF16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


# ---- norms and rotation

def norm_rope(x, weight, eps, norm, positions, inv_freq, rotary_dim, near, rope_scale=1.0):
    """x [T, H, D] float64 -> (result, bound): bound[t, h, d] = |p| + |q| of the pair behind each element."""
    y = x.copy()
    if norm:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps)
    if weight is not None:
        y = y * weight.astype(np.float64)
    size = np.abs(y)
    R = rotary_dim
    if R:
        i = np.arange(R // 2)
        a, b = (2 * i, 2 * i + 1) if near else (i, i + R // 2)
        f = positions.astype(np.float64)[:, None] * inv_freq
        c, s = np.cos(f)[:, None] * rope_scale, np.sin(f)[:, None] * rope_scale
        p, q = y[..., a], y[..., b]
        pair = (np.abs(p) + np.abs(q)) * abs(rope_scale)
        y[..., a], y[..., b] = p * c - q * s, q * c + p * s
        size[..., a], size[..., b] = pair, pair
    return y, size


# ---- e4m3 codes

def _table():
    t = np.zeros(256)
    for c in range(256):
        e, f = c >> 3 & 15, c & 7
        v = f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)
        t[c] = np.nan if c & 127 == 127 else -v if c & 128 else v
    return t


E4M3 = _table()
_GRID = E4M3[:127]


def encode(x: np.ndarray) -> np.ndarray:
    """Codes of the nearest e4m3 values, ties to even codes; NaN for what is not finite. |x| <= 448."""
    a = np.abs(np.where(np.isfinite(x), x, 0.0))
    hi = np.minimum(np.searchsorted(_GRID, a), 126)
    lo = np.maximum(hi - 1, 0)
    dh, dl = _GRID[hi] - a, a - _GRID[lo]
    pick = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    codes = pick | np.where(np.signbit(x), 128, 0)
    return np.where(np.isfinite(x), codes, 127).astype(np.uint8)


def exponent(amax: np.ndarray) -> np.ndarray:
    """The smallest byte e >= 0 with amax <= 448 * 2^(e - 127)."""
    e = np.zeros(np.shape(amax), np.int64)
    for byte in range(254, -1, -1):
        e = np.where(amax <= 448.0 * 2.0 ** (byte - 127), byte, e)
    return e


# ---- the cache

def v_slot(t):
    return 16 * (t // 4 % 2) + 4 * (t // 8) + t % 4


class Cache:
    """codes [2][pages, Hkv, 32, D] and exponent bytes [2][pages, Hkv] of K and V."""

    def __init__(self, pages, Hkv, D, rng=None):
        self.pages, self.Hkv, self.D = pages, Hkv, D
        shape = (2, pages, Hkv, BLOCK, D)
        self.codes = rng.integers(0, 256, shape, dtype=np.uint8) if rng is not None else np.zeros(shape, np.uint8)
        self.exp = rng.integers(0, 255, shape[:3], dtype=np.uint8) if rng is not None else np.zeros(shape[:3], np.uint8)

    def device_arrays(self):
        """(k, v, k_scale, v_scale) as the library lays them out."""
        P, H, D = self.pages, self.Hkv, self.D
        k = self.codes[0].reshape(P, H, BLOCK, D // 32, 32).transpose(0, 1, 3, 2, 4)
        v = np.empty((P, H, D, BLOCK), np.uint8)
        v[..., v_slot(np.arange(BLOCK))] = self.codes[1].transpose(0, 1, 3, 2)
        return np.ascontiguousarray(k), v, self.exp[0].copy(), self.exp[1].copy()

    def from_device(self, k, v, ks, vs):
        """The cache those arrays hold."""
        P, H, D = self.pages, self.Hkv, self.D
        c = Cache(P, H, D)
        c.codes[0] = k.reshape(P, H, D // 32, BLOCK, 32).transpose(0, 1, 3, 2, 4).reshape(P, H, BLOCK, D)
        c.codes[1] = v.reshape(P, H, D, BLOCK)[..., v_slot(np.arange(BLOCK))].transpose(0, 1, 3, 2)
        c.exp[0], c.exp[1] = ks.reshape(P, H), vs.reshape(P, H)
        return c

    def page_of(self, table, b, pos):
        if pos < 0 or pos // BLOCK >= table.shape[1]:
            return None
        p = table[b, pos // BLOCK]
        return int(p) if 0 <= p < self.pages else None

    def write(self, seqs, k, v):
        """k, v [T, Hkv, D] float64."""
        for b, n, r, row0, first in seqs:
            pos = np.arange(first, first + r)
            for block in np.unique(pos // BLOCK):
                page = self.page_of(seqs.table, b, int(block) * BLOCK)
                if page is None:
                    continue
                here = pos[pos // BLOCK == block]
                kept = int(here[0]) % BLOCK  # earlier tokens of the page
                for w, x in ((0, k), (1, v)):
                    new = x[row0 + here - first]  # [m, Hkv, D]
                    amax = np.abs(np.where(np.isfinite(new), new, 0.0)).max((0, 2))
                    e = exponent(amax)
                    old = np.minimum(self.exp[w, page].astype(np.int64), 254)
                    if kept:
                        e = np.maximum(e, old)
                        moved = E4M3[self.codes[w, page, :, :kept]] * 2.0 ** (old - e)[:, None, None]
                        same = (e == old)[:, None, None]
                        self.codes[w, page, :, :kept] = np.where(same, self.codes[w, page, :, :kept], encode(moved))
                    self.codes[w, page][:, here % BLOCK] = encode(new * 2.0 ** (127 - e)[:, None]).transpose(1, 0, 2)
                    self.exp[w, page] = e

    def token(self, table, b, pos):
        """(K, V) [Hkv, D] of a position, or None."""
        page = self.page_of(table, b, pos)
        if page is None:
            return None
        return tuple(E4M3[self.codes[w, page, :, pos % BLOCK]] * 2.0 ** (self.exp[w, page].astype(np.float64) - 127)[:, None] for w in (0, 1))

    def read(self, seqs, T):
        """(K, V, whose) [T, Hkv, D] float64, and which rows belong to a sequence."""
        k, v, mine = np.zeros((T, self.Hkv, self.D)), np.zeros((T, self.Hkv, self.D)), np.zeros(T, bool)
        for b, n, r, row0, first in seqs:
            for i in range(r):
                got = self.token(seqs.table, b, first + i)
                mine[row0 + i] = True
                if got is not None:
                    k[row0 + i], v[row0 + i] = got
        return k, v, mine

    def attention(self, seqs, q, scale, causal):
        """q [T, H, D] float64 -> (o, mean |v| under the same weights, largest sum of |q||k| over D, keys, whose rows)."""
        T, H, D = q.shape
        G = H // self.Hkv
        o, size, reach = np.zeros((T, H, D)), np.zeros((T, H, D)), np.zeros((T, H))
        count, mine = np.zeros(T, np.int64), np.zeros(T, bool)
        for b, n, r, row0, first in seqs:
            got = [(j, self.token(seqs.table, b, j)) for j in range(n)]
            at = np.array([j for j, g in got if g is not None], np.int64)
            K = np.array([g[0] for _, g in got if g is not None]).reshape(len(at), self.Hkv, D)
            V = np.array([g[1] for _, g in got if g is not None]).reshape(len(at), self.Hkv, D)
            for i in range(r):
                mine[row0 + i] = True
                m = int((at <= first + i).sum()) if causal else len(at)
                count[row0 + i] = m
                if m == 0:
                    continue
                for h in range(H):
                    qq, kk, vv = q[row0 + i, h], K[:m, h // G], V[:m, h // G]
                    with np.errstate(invalid="ignore"):
                        s = kk @ qq * scale
                        p = np.exp(s - s.max())
                        p = p / p.sum()
                        o[row0 + i, h], size[row0 + i, h] = p @ vv, p @ np.abs(vv)
                        reach[row0 + i, h] = (np.abs(kk) @ np.abs(qq)).max() * abs(scale)
        return o, size, reach, count, mine


class Seqs:
    """The sequences of a call as the device arrays give them, bounded as the kernels bound them."""

    def __init__(self, seq_len, table, T, max_rows, row_start=None):
        self.seq_len, self.table = np.asarray(seq_len, np.int32), np.asarray(table, np.int32).reshape(len(seq_len), -1)
        self.T, self.max_rows = T, max_rows
        self.row_start = None if row_start is None else np.asarray(row_start, np.int32)

    def __iter__(self):
        """(sequence, its length, rows, first row, position of the first row)"""
        for b, n in enumerate(self.seq_len.tolist()):
            n = min(max(n, 0), self.table.shape[1] * BLOCK)
            r0, r = b * self.max_rows, self.max_rows
            if self.row_start is not None:
                r0, r = int(self.row_start[b]), int(self.row_start[b + 1]) - int(self.row_start[b])
            if r < 0 or r0 < 0 or r0 >= self.T:
                r = 0
            first = n - r
            yield b, n, min(r, self.max_rows, max(self.T - r0, 0)), r0, first


# ---- how far a float32 evaluation may be off

def attention_tolerance(o, size, reach, count, D, dtype):
    """Bound of |result - o| for the operator's arithmetic, u = 2^-24.

    A score (in natural units) is a float32 sum of D products of exact codes with q held to 2^-22 of each element
    (float32 rows; exactly otherwise, in one term): off by at most (2 D + 4) u of the sum of |q||k|, which `reach`
    bounds, and by the roundings of its scaling and of its difference from the maximum, (4 + 2) u reach more. A
    probability is off by that, relatively, twice (itself and its sum), by 2^-23 of exp2, and by its float16 terms:
    half a step of 11 bits (2^-11), or 2^-22 in two terms. The sum over the keys in float32, split and merged, adds
    (keys + 16) u. The result's own rounding is half a step of the type."""
    u = 2.0 ** -24
    rel = 2 * (2 * D + 10) * u * reach * 2 + 2.0 ** -22 + (2.0 ** -21 if dtype == "F32" else 2.0 ** -11) + (count[:, None] + 16) * u
    return rel[..., None] * size + EPS[dtype] / 2 * np.abs(o) + tiny(dtype)


def rope_tolerance(y, size, D, dtype):
    """Bound for norms and rotation, u = 2^-24: the sum of squares (D + 2 roundings, halved by the root), root,
    quotient, two products; sine and cosine within 4 ulp at an angle held to half a step of pi; two products and a sum."""
    u = 2.0 ** -24
    return ((D + 2) / 2 + 4 + 4 + 3.2 + 2) * u * size + EPS[dtype] / 2 * np.abs(y) + tiny(dtype)


def tiny(dtype):
    """Half the smallest step of the type."""
    return {"F32": 2.0 ** -150, "F16": 2.0 ** -25, "BF16": 2.0 ** -134}[dtype]
