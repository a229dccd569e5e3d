"""The 8-bit paged K/V cache in numpy, from its definition (include/mp_hip.h):
bytes of a page, appending, reading, attention in 64 bits. Nothing here is
shared with the kernels."""
from __future__ import annotations

import math

import numpy as np

INT8, E4M3 = 0, 1
F32, BF16, F16 = 0, 1, 2
F = np.float32


def e4m3_values() -> np.ndarray:
    """What each byte stands for: sign, 4 exponent bits (bias 7), 3 mantissa bits; 0x7F and 0xFF are NaN."""
    out = np.empty(256, dtype=np.float64)
    for b in range(256):
        e, m = b >> 3 & 15, b & 7
        x = math.nan if (e, m) == (15, 7) else m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out[b] = -x if b & 128 else x
    return out


VALUES = {INT8: np.arange(256, dtype=np.float64) - 128, E4M3: e4m3_values()}


def encode(x: np.ndarray, fmt: int) -> np.ndarray:
    """The byte of the number nearest to x (ties: even mantissa or code); |x| is at most 127 or 448."""
    if fmt == INT8:
        return (np.rint(x.astype(np.float64)) + 128).astype(np.uint8)
    grid = VALUES[E4M3][:127]  # positive, ascending; even bytes have even mantissas
    a = np.abs(x.astype(np.float64))
    above = np.clip(np.searchsorted(grid, a), 1, 126)
    low, high = grid[above - 1], grid[above]
    up = (a - low > high - a) | ((a - low == high - a) & (above % 2 == 0))
    code = np.where(up, above, above - 1).astype(np.uint8)
    return np.where(np.signbit(x), code | 128, code).astype(np.uint8)


def scale_for(amax: float, fmt: int) -> np.float32:
    if not np.isfinite(amax):
        return F(np.nan)
    top = 127.0 if fmt == INT8 else 448.0
    e = -126
    while float(amax) > top * 2.0 ** e:
        e += 1
    return F(2.0 ** e)


def places(bt: int, dim: int):
    """Byte of (slot, dim) in a head's bytes of a page, for keys and for values."""
    slot, d = np.arange(bt)[:, None], np.arange(dim)[None]
    tile, s = slot // 16 * 16 * dim, slot % 16
    return (tile + d // 16 * 256 + s * 16 + d % 16,
            tile + d // 64 * 1024 + s // 4 * 256 + d % 16 * 16 + d % 64 // 16 * 4 + s % 4)


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray, dims: int, interleaved: bool) -> np.ndarray:
    """x [heads, dim] float32 turned by cos and sin [dims/2], each operation rounded to float32."""
    out = x.copy()
    half = dims // 2
    a_at = np.arange(half) * 2 if interleaved else np.arange(half)
    b_at = a_at + 1 if interleaved else a_at + half
    a, b = x[:, a_at], x[:, b_at]
    out[:, a_at], out[:, b_at] = a * cos - b * sin, b * cos + a * sin
    return out


class Cache:
    """Pools as the device holds them, and what the calls do to them."""

    def __init__(self, blocks, layers, kv_heads, bt, dim, fmt, rng):
        self.blocks, self.layers, self.kv_heads, self.bt, self.dim, self.fmt = blocks, layers, kv_heads, bt, dim, fmt
        shape = (blocks, layers, kv_heads, bt * dim)
        # Whatever was there before: any bytes (NaN codes among the E4M3 ones), any scales.
        self.bytes = [rng.integers(0, 256, shape, dtype=np.uint8) for _ in range(2)]
        self.scales = F(2.0) ** rng.integers(-9, 3, (blocks, layers, kv_heads, 2)).astype(F)
        self.places = places(bt, dim)

    def append(self, layer, k, v, tables, starts, used, rope=None):
        """k, v [rows, kv_heads, dim] float32; rope (cos, sin, dims, interleaved)."""
        for s in range(len(used)):
            r, position, end = starts[s], used[s], used[s] + starts[s + 1] - starts[s]
            if rope and rope[2]:
                end = min(end, len(rope[0]))
            while position < end:
                slot = position % self.bt
                n = min(self.bt - slot, end - position)
                page = position // self.bt
                block = tables[s, page] if page < tables.shape[1] else -1
                if 0 <= block < self.blocks:
                    rows = [k[r:r + n].copy(), v[r:r + n]]
                    if rope and rope[2]:
                        for i in range(n):
                            rows[0][i] = rotate(rows[0][i], rope[0][position + i], rope[1][position + i], *rope[2:])
                    for kind in range(2):
                        for h in range(self.kv_heads):
                            self._page(block, layer, h, kind, slot, rows[kind][:, h])
                r, position = r + n, position + n

    def _page(self, block, layer, head, kind, slot, x):
        data = self.bytes[kind][block, layer, head]
        at, n = self.places[kind], len(x)
        held = self.scales[block, layer, head, kind] if slot else F(0)
        new = scale_for(np.abs(x).max(), self.fmt)
        scale = held if np.isnan(held) or held >= new else new
        self.scales[block, layer, head, kind] = scale
        if np.isnan(scale):
            return  # the bytes of a page that reads as NaN are of no interest
        if slot and scale > held:
            old = VALUES[self.fmt][data[at[:slot]]] * float(held / scale)
            data[at[:slot]] = encode(old, self.fmt)
        data[at[slot:slot + n]] = encode(x * (F(1) / scale), self.fmt)

    def tokens(self, layer, kind, table, length):
        """[kv_heads, length, dim] float64 values of a sequence; NaN where it has no page."""
        out = np.full((self.kv_heads, length, self.dim), np.nan)
        for page in range(-(-length // self.bt)):
            block = table[page] if page < len(table) else -1
            if 0 <= block < self.blocks:
                n = min(self.bt, length - page * self.bt)
                data = self.bytes[kind][block, layer][:, self.places[kind][:n]]
                scale = self.scales[block, layer, :, kind].astype(np.float64)
                out[:, page * self.bt:page * self.bt + n] = VALUES[self.fmt][data] * scale[:, None, None]
        return out

    def attention(self, layer, q, table, length, scale):
        """One row q [heads, dim] over `length` tokens, in 64 bits: the result [heads, dim] and a bound on the
        error of its FP32 evaluation, [heads, 1] (see `bound`)."""
        heads = q.shape[0]
        if length <= 0:
            return np.zeros((heads, self.dim)), np.zeros((heads, 1))
        k, v = (self.tokens(layer, kind, table, length) for kind in range(2))
        group = heads // self.kv_heads
        out, err = np.empty((heads, self.dim)), np.empty((heads, 1))
        for h in range(heads):
            kh = h // group
            z = k[kh] @ q[h].astype(np.float64) * scale
            p = np.exp(z - z.max())
            p /= p.sum()
            out[h] = p @ v[kh]
            err[h] = bound(p, np.abs(k[kh]) @ np.abs(q[h]).astype(np.float64) * scale, v[kh])
        return out, err


def bound(p, z_abs, v):
    """How far FP32 arithmetic may be off, u = 2^-24 a rounding: a score is a sum of dim products of q's high and
    low parts (2 dim sums and the split's 2^-23, then three more roundings): |dz| <= (2 dim + 8) u z_abs. A
    probability has the relative error dz, exp2's (2 ulp) and the reference's; sums over T tokens of high and low
    parts, of l and of the split results add (2 T + 32) u of the absolute sums, p's own split 2^-22. Numerator and
    denominator both: twice."""
    u, (tokens, dim) = 2.0 ** -24, v.shape
    dz = (2 * dim + 8) * u * z_abs
    relative = p @ dz + (2 * tokens + 32) * u + 2.0 ** -21
    return 2 * relative * np.abs(v).max()


def rounded(x: np.ndarray, kind: int) -> np.ndarray:
    """float32 numbers rounded to a row type, as float32."""
    import torch
    t = {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16}[kind]
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(t).float().numpy()


def likely_bound(p, z, q, k, v, scale):
    """How far FP32 arithmetic is off where its roundings have random signs, u = 2^-24 a rounding, about six standard
    deviations. A score sums dim products of q's high and low parts: 2 dim roundings of partial sums that are about
    |q k| (the norm of the products), and the split's 2^-23 of each, 4 sqrt(2 dim) u |q k| in all; factor and
    reference round it again, where the difference to the reference is below 16 or as far as z is from the largest:
    (4 |z| + 4 |z - z_max| + 16) u. A probability has that relative error, averaged over the row as if all signs were
    the same; exp2, its split and the weights 8 u; sums over T tokens 2 sqrt(T) u. Numerator and denominator: twice."""
    u, (tokens, dim) = 2.0 ** -24, v.shape
    norm = np.sqrt((k ** 2) @ (q.astype(np.float64) ** 2)) * scale
    dz = u * (4 * math.sqrt(2 * dim) * norm + 4 * np.abs(z) + 4 * np.abs(z - z.max()) + 16)
    return 2 * (p @ dz + (2 * math.sqrt(tokens) + 8) * u) * np.abs(v).max()


def attention_close(cache, layer, q, table, length, scale):
    """Cache.attention with `likely_bound` in the place of the worst case."""
    heads = q.shape[0]
    k, v = (cache.tokens(layer, kind, table, length) for kind in range(2))
    out, err = np.empty((heads, cache.dim)), np.empty((heads, 1))
    for h in range(heads):
        kh = h // (heads // cache.kv_heads)
        z = k[kh] @ q[h].astype(np.float64) * scale
        p = np.exp(z - z.max())
        p /= p.sum()
        out[h] = p @ v[kh]
        err[h] = likely_bound(p, z, q[h], k[kh], v[kh], scale)
    return out, err
