"""The 8-bit cache format in numpy: what the tests hold the kernels to.

A block (16 rows of one page, one KV head, K or V) holds E4M3 codes times
2^e.  All arithmetic here is in 64 bits on F32 inputs, where scaling by powers
of two and the rounding to 4 significant bits are exact, so the kernels' cells
have to equal these bit for bit.
"""
from __future__ import annotations

import numpy as np

EXP_MIN = -100
D = 128
PAGE = 16


def block_exponent(x) -> int:
    """The least e >= EXP_MIN with max|finite x| <= 448 * 2^e."""
    x = np.asarray(x, np.float64)
    amax = np.max(np.abs(x[np.isfinite(x)]), initial=0.0)
    if amax == 0.0:
        return EXP_MIN
    m, e = np.frexp(amax)  # m in [0.5, 1), 448 = 0.875 * 2^9
    return max(int(e) - 9 + (1 if m > 0.875 else 0), EXP_MIN)


def round_e4m3(y):
    """Nearest E4M3 number (ties to even) of |y| <= 448; not finite: NaN."""
    y = np.asarray(y, np.float64)
    ok = np.isfinite(y)
    z = np.where(ok, y, 0.0)
    _, e = np.frexp(z)
    step = np.ldexp(1.0, np.maximum(e - 4, -9))
    return np.where(ok, np.rint(z / step) * step, np.nan)


class SlotModel:
    """One slot's K or V of one layer: rows [L][G][D] as the cache holds them."""

    def __init__(self, G: int):
        self.G = G
        self.values = np.zeros((0, G, D))
        self.exp = np.zeros((0, G), np.int64)

    def write(self, pos0: int, rows) -> None:
        """rows [n][G][D] at positions pos0 ..: one call, cut at page borders."""
        rows = np.asarray(rows, np.float64)
        end = pos0 + rows.shape[0]
        full = -(-end // PAGE) * PAGE
        if full > self.values.shape[0]:
            more = full - self.values.shape[0]
            self.values = np.concatenate([self.values, np.zeros((more, self.G, D))])
            self.exp = np.concatenate([self.exp, np.full((more // PAGE, self.G), EXP_MIN)])
        for p in range(pos0 // PAGE, (end - 1) // PAGE + 1):
            lo, hi = max(pos0, p * PAGE), min(end, (p + 1) * PAGE)
            new = rows[lo - pos0:hi - pos0]
            for g in range(self.G):
                e = block_exponent(new[:, g])
                if lo % PAGE:
                    e = max(e, int(self.exp[p, g]))
                    if e > self.exp[p, g]:
                        others = [r for r in range(p * PAGE, (p + 1) * PAGE) if not lo <= r < hi]
                        self.values[others, g] = round_e4m3(np.ldexp(self.values[others, g], -e)) * 2.0 ** e
                self.exp[p, g] = e
                self.values[lo:hi, g] = round_e4m3(np.ldexp(new[:, g], -e)) * 2.0 ** e

    def fork(self, n: int) -> "SlotModel":
        m = SlotModel(self.G)
        pages = -(-n // PAGE)
        m.values = self.values[:pages * PAGE].copy()
        m.exp = self.exp[:pages].copy()
        return m


def attention(q, k, v, first, scale=1.0 / np.sqrt(float(D))):
    """q [T][H][D] (rotated), rows k, v [L][G][D]; row i of q sees rows [0, first + i].
    Float64 result [T][H][D] and the largest sum_d |q_d k_d| * scale of any pair seen."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    T, H, _ = q.shape
    G = k.shape[1]
    out = np.zeros((T, H, D))
    big = 0.0
    seen = np.arange(k.shape[0])[None] <= first + np.arange(T)[:, None]
    last = first + T
    for h in range(H):
        g = h // (H // G)
        s = (q[:, h] @ k[:last, g].T) * scale
        s = np.where(seen[:, :last], s, -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        out[:, h] = (p @ v[:last, g]) / p.sum(1, keepdims=True)
        big = max(big, float((np.abs(q[:, h]) @ np.abs(k[:last, g]).T).max()) * scale)
    return out, big


def attention_tolerance(big: float, rows: int, vmax: float) -> float:
    """Absolute bound on an output of the F32 kernels.

    A logit is off by at most big * (2^-22 + 2^-19): q is held in two F16 parts
    (2^-11 each, 2^-22 together), and its 128 products are summed in F32 in at
    most 16 steps of 2^-23 relative to sum |q k|.  A weight p is then off by that
    (relative), by 2^-21 for the exponential and its argument's rounding per unit
    of the logit range (at most `big` each side: 2 * big * 2^-23), and by 2^-22
    for its two F16 parts.  Both the weighted sum and the sum of weights are
    off by that, plus one rounding of 2^-23 for each page and merge step."""
    logit = big * (2.0 ** -22 + 2.0 ** -19) + 2 * big * 2.0 ** -23
    weight = logit + 2.0 ** -21 + 2.0 ** -22
    return vmax * (2 * weight + (rows / PAGE + 64) * 2.0 ** -23)
