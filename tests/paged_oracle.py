"""A KV cache in pages on the host, in plain numpy: rows in and out, 8 bits, and attention in 64 bits with the error that a
kernel may make."""
import math

import numpy as np

from oracle import oracle as orc

DT_FLOAT16, DT_BFLOAT16, DT_FLOAT8 = 4, 5, 16
HALF_STEP = {DT_FLOAT16: 2.0 ** -11, DT_BFLOAT16: 2.0 ** -8}  # largest relative error of one rounding

# The 127 finite magnitudes of e4m3: four significant bits from 2^-6 on, steps of 2^-9 below
E4M3 = np.array([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127])


def narrow(x):
    """float64 -> e4m3 bytes, to nearest, ties to even; not finite: NaN."""
    x = np.asarray(x, dtype=np.float64)
    a = np.minimum(np.abs(np.where(np.isfinite(x), x, 0)), 448.0)
    hi = np.searchsorted(E4M3, a)
    lo = np.maximum(hi - 1, 0)
    down, up = a - E4M3[lo], E4M3[hi] - a
    code = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.isfinite(x), code | (np.signbit(x) * 128), 127)
    return code.astype(np.uint8)


def widen8(codes):
    mag = np.append(E4M3, np.nan)[codes & 127]
    return np.where(codes & 128, -mag, mag)


def eight_bits(rows, dt):
    """float64 rows of 128 (values of the type) -> (codes, exponent bytes)."""
    most = 1.875 * 2.0 ** (15 if dt == DT_FLOAT16 else 127)
    finite = np.isfinite(rows)
    x = np.where(finite, np.clip(np.where(finite, rows, 0), -most, most), np.nan)
    amax = np.where(finite, np.abs(x), 0).max(-1)
    frac, power = np.frexp(amax / 448)
    byte = np.maximum(np.where(amax > 0, np.where(frac > 0.5, power, power - 1), -10 ** 6) + 127, 64)
    return narrow(x / 2.0 ** (byte[..., None] - 127.0)), byte.astype(np.uint8)


class Pool:
    """Pages of K or of V as bytes: [num_pages][stride]."""

    def __init__(self, num_pages, page_size, kv_heads, cache_dt, dt, stride=None, fill=0):
        self.n, self.ps, self.h, self.cache_dt, self.dt = num_pages, page_size, kv_heads, cache_dt, dt
        self.eight = cache_dt == DT_FLOAT8
        self.row_bytes = 128 if self.eight else 256
        self.values = kv_heads * page_size * self.row_bytes
        self.page_bytes = self.values + (kv_heads * page_size if self.eight else 0)
        self.stride = stride or self.page_bytes
        self.raw = np.full((num_pages, self.stride), fill, dtype=np.uint8)

    def rows_of(self, page):  # [kv head][row][bytes]: a view
        return self.raw[page, :self.values].reshape(self.h, self.ps, self.row_bytes)

    def bytes_of(self, page):
        return self.raw[page, self.values:self.page_bytes].reshape(self.h, self.ps)

    def put(self, page, row, x_bits):
        """x_bits [kv head][128] uint16 of dt."""
        if self.eight:
            codes, byte = eight_bits(orc.widen(x_bits, self.dt).astype(np.float64), self.dt)
            self.rows_of(page)[:, row] = codes
            self.bytes_of(page)[:, row] = byte
        else:
            self.rows_of(page)[:, row] = np.ascontiguousarray(x_bits).view(np.uint8).reshape(self.h, 256)

    def get(self, page, row):
        """float64 [kv head][128]"""
        x = np.ascontiguousarray(self.rows_of(page)[:, row])
        if self.eight:
            return widen8(x) * 2.0 ** (self.bytes_of(page)[:, row].astype(np.float64) - 127)[:, None]
        return orc.widen(x.view(np.uint16), self.dt).astype(np.float64)


def place(table_row, num_pages, page_size, key):
    i = key // page_size
    if key < 0 or i >= len(table_row) or not 0 <= table_row[i] < num_pages:
        return None
    return int(table_row[i]), key % page_size


def sequence_rows(pool, table_row, n):
    """(rows [n][kv head][128], there [n]) of a sequence; NaN-free zeros where a page is not there."""
    x, there = np.zeros((n, pool.h, 128)), np.zeros(n, dtype=bool)
    for key in range(n):
        at = place(table_row, pool.n, pool.ps, key)
        if at is not None:
            x[key], there[key] = pool.get(*at), True
    return x, there


def attend(q_bits, k_pool, v_pool, table, starts, lens, dt, group, window=0, sinks=0):
    """(out [tokens][heads][128] float64, bound on a kernel's error, rows that are a sequence's).

    The bound, first order: the weights w are rounded once (relative error u), the sum takes the rounded ones, so numerator
    and denominator together are off by u * sum w |v - out|; the result is rounded once more, u |out|.  Scores are sums of 128 products in 32
    bits, off by at most 2^-17 sum |q k| / sqrt(128) each (a weight by as much, relative), and some steps of 2^-24 in the exponent, its scale of up
    to |score| and the sums over keys.  fp16 weights below 2^-14 of the largest are steps of 2^-24, off by 2^-25."""
    tokens, heads, _ = q_bits.shape
    u = HALF_STEP[dt]
    out, tol, mine = np.zeros((tokens, heads, 128)), np.zeros((tokens, heads, 128)), np.zeros(tokens, dtype=bool)
    q = orc.widen(q_bits, dt).astype(np.float64)
    for b, n in enumerate(lens):
        k, there = sequence_rows(k_pool, table[b], n)
        v, _ = sequence_rows(v_pool, table[b], n)
        for t in range(starts[b], starts[b + 1]):
            mine[t] = True
            p = n - starts[b + 1] + t
            keys = [c for c in range(min(p + 1, n)) if there[c] and (window <= 0 or c > p - window or c < sinks)]
            if not keys:
                continue
            for h in range(heads):
                kk, vv = k[keys, h // group], v[keys, h // group]
                products = kk * q[t, h]
                s = products.sum(-1) / math.sqrt(128)
                w = np.exp(s - s.max())
                w /= w.sum()
                o = w @ vv
                spread = np.abs(vv - o)
                out[t, h] = o
                slack = 2.0 ** -17 * (np.abs(products).sum(-1) / math.sqrt(128)) + 2.0 ** -22 * (np.abs(s) + np.abs(s).max() + 4)
                tol[t, h] = (u + slack) * w @ spread + u * np.abs(o) + 2.0 ** -22 * (w @ np.abs(vv)) * (1 + len(keys) / 64)
                if dt == DT_FLOAT16:
                    tol[t, h] += 2.0 ** -25 * spread.sum(0) * w.max() + 2.0 ** -25
                tol[t, h] *= 1 + 2.0 ** -6  # second order
    return out, tol, mine
