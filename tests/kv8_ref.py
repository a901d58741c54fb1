"""Plain 64-bit implementation of the 8-bit key/value cache (numpy), which the tests of kv8_append,
kv8_read and attn_fwd_kv8 compare with: the definitions, one token and one row at a time where that
is quick enough, and the error bound of the attention.
"""
import math

import numpy as np


def decode_table():
    """The values of the 256 e4m3 codes: sign, 4 bits of exponent (bias 7), 3 of mantissa; 0x7f is NaN."""
    t = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.nan if (c & 0x7f) == 0x7f else (m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        t[c] = -v if c & 0x80 else v
    return t


TABLE = decode_table()


def round_e4m3(x):
    """Nearest e4m3 value, ties to even, magnitudes above 448 (infinities too) to 448, NaN kept."""
    x = np.asarray(x, dtype=np.float64)
    c = np.clip(x, -448, 448)
    _, e = np.frexp(c)
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    return np.rint(c / step) * step


def scale_for(amax):
    for e in range(-40, 40):
        if amax <= 448 * 2.0 ** e:
            return 2.0 ** e
    return 2.0 ** 40


class Cache:
    """values = codes' values (float64, [n_blocks, Hkv, P, D]); scales [n_blocks, Hkv]."""

    def __init__(self, codes, scales):
        self.values = TABLE[np.asarray(codes)]
        self.scales = np.array(scales, dtype=np.float64)

    def append(self, x, table, lens, new):
        """x [total, Hkv, D]: the last new[b] of lens[b] tokens of every sequence b, in order."""
        P, t = self.values.shape[2], 0
        for b, (n, m) in enumerate(zip(lens, new)):
            p = n - m
            while p < n:
                blk, lo = table[b][p // P], p % P
                c = min(P - lo, n - p)
                for h in range(x.shape[1]):
                    part = np.asarray(x[t:t + c, h], dtype=np.float64)
                    fin = np.abs(part[np.isfinite(part)])
                    s = scale_for(fin.max() if fin.size else 0.0)
                    if lo:
                        s = max(s, self.scales[blk, h])
                        if s > self.scales[blk, h]:
                            self.values[blk, h, :lo] = round_e4m3(self.values[blk, h, :lo] * (self.scales[blk, h] / s))
                    self.values[blk, h, lo:lo + c] = round_e4m3(part / s)
                    self.scales[blk, h] = s
                p, t = p + c, t + c

    def tokens(self, table_row, n):
        """The first n tokens of a sequence, [n, Hkv, D]."""
        P = self.values.shape[2]
        out = np.zeros((n, self.values.shape[1], self.values.shape[3]))
        for p in range(0, n, P):
            blk, c = table_row[p // P], min(P, n - p)
            out[p:p + c] = (self.values[blk, :, :c] * self.scales[blk][:, None, None]).transpose(1, 0, 2)
        return out

    def token_scales(self, table_row, n):
        P = self.values.shape[2]
        return np.stack([self.scales[table_row[p // P]] for p in range(n)]) if n else np.zeros((0, self.scales.shape[1]))


def attend(q, K, V, table, lens, new, scale, causal, gate=None, unit=2.0 ** -8):
    """(o, bound) [total, Hq, D]: exact outputs, and how far off a kernel may be that
      * sums a score's D products in 32 bits (2^-22 each and of the sum, which a tensor core may truncate),
      * rounds the weights to fp16 (2^-11 relative; 2^-25 absolute below 2^-14, of the largest being >= 1),
      * takes exponentials within 2^-21 and sums in 32 bits, and rounds the result to `unit`.
    unit: half a step of the output type (bf16 2^-8, fp16 2^-11)."""
    total, Hq, D = q.shape
    Hkv = K.values.shape[1]
    o, bound, t = np.zeros(q.shape), np.zeros(q.shape), 0
    for b, (n, m) in enumerate(zip(lens, new)):
        k, v = K.tokens(table[b], n), V.tokens(table[b], n)
        sv = V.token_scales(table[b], n)
        for i in range(m):
            see = min(n, max(0, n - m + i + 1)) if causal else n
            for hq in range(Hq):
                h = hq // (Hq // Hkv)
                if see:
                    kk, vv = k[:see, h], v[:see, h]
                    qq = np.asarray(q[t, hq], dtype=np.float64)
                    with np.errstate(invalid="ignore", over="ignore"):
                        x = scale * (kk @ qq)
                        p = np.exp(x - np.nanmax(x)) if not np.all(np.isnan(x)) else x
                        w = p / p.sum()
                        o[t, hq] = w @ vv
                        size = w @ np.abs(vv)
                        dx = (D + 4) * 2.0 ** -22 * scale * (np.abs(kk) @ np.abs(qq)).max()
                        # the weights in the kernel are of exp(x) * scale of V: 2^-25 of the largest of those
                        largest = int(np.argmax(np.log(np.maximum(w, 1e-300)) + np.log(sv[:see, h])))
                        small = 2.0 ** -25 * (np.abs(vv) / sv[:see, h][:, None]).sum(0) * sv[largest, h] * w[largest]
                        bound[t, hq] = (2 * (dx + 2.0 ** -20 + see * 2.0 ** -24) + 2.0 ** -11) * size + small
                if gate is not None:
                    with np.errstate(over="ignore"):
                        s = 1 / (1 + np.exp(-np.asarray(gate[t, hq], dtype=np.float64)))
                    o[t, hq] *= s
                    bound[t, hq] = bound[t, hq] * s + 2.0 ** -18 * np.abs(o[t, hq])
                bound[t, hq] += unit * np.abs(o[t, hq]) * (1 + 2.0 ** -6) + 2.0 ** -24 * unit
            t += 1
    return o, bound
