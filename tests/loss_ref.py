"""The loss over an int8 linear layer in 64 bits (numpy), and how far a 32-bit evaluation may be from it."""
import numpy as np

import scaled_ref as ref

U32 = ref.U32

# m, k, n: up to 64 rows through their logits, then every tile of both passes; a class, odd sizes, sums over nothing
CASES = [(1, 64, 1), (1, 1, 2), (5, 120, 1203), (16, 4096, 700), (17, 128, 5000), (64, 333, 9001), (3, 0, 10), (100, 0, 70),
         (65, 64, 64), (65, 128, 1000), (66, 130, 129), (100, 333, 5003), (200, 127, 63), (300, 999, 1001), (256, 256, 256),
         (700, 1024, 3000), (1000, 512, 8000), (600, 2048, 4999), (2050, 400, 13000), (1030, 1030, 16500), (513, 64, 700),
         (130, 3000, 40), (875, 451, 15691), (2541, 768, 6285), (4872, 408, 2945)]


class Loss:
    """Of rows q [m, k] int8 with scales t, weights w, s, bias and targets; `ignored`: a target of none."""

    def __init__(self, q, t, w, s, bias, target, ignored=-100):
        self.w, self.s = w.astype(np.float64), s.astype(np.float64)
        self.l, self.e = ref.linear(q, t, w, s, bias)
        l, m = self.l, self.l.max(1, keepdims=True)
        self.has = target != ignored
        at = np.where(self.has, target, 0)
        rows = np.arange(len(at))
        x = np.exp(l - m)
        total = x.sum(1, keepdims=True)
        self.p = x / total
        self.d = (l - m) - np.log(total)
        mine = self.d[rows, at]
        self.loss = np.where(self.has, -mine, 0.0)
        self.at, self.rows = at, rows
        # exp: its argument's rounding (|l - m| each time), 2 of its own; a sum's joins, 4 each: 13 within a wave, 6
        # over a group's threads and the parts they take in turn
        joins = 13 + 4 * (8 + l.shape[1] / 1024)
        self.e_lse = (self.p * (self.e + np.abs(l - m) * 2 * U32)).sum(1) + (joins + 4) * U32 + 2 * U32 * np.log(total[:, 0])
        self.bound = self.e_lse + self.e[rows, at] + U32 * (2 * np.abs(self.loss) + 2 * np.abs(l[rows, at] - m[:, 0]))
        self.bound = np.where(self.has, self.bound, 0.0)

    def mean(self):
        n = self.has.sum()
        return self.loss.sum() / n, self.bound.sum() / n + 2 * U32 * abs(self.loss.sum() / n)

    def reach(self):
        """What a row's terms are normalised to, over the largest |s|: 1 - p of the target, or the logits' own
        rounding (steps of 2^-24 of m, a few of them) where that is more. float16 halves are then steps of 2^-24 of
        values of 2^14 .. 2^15, 2^-38 of this at most, which _grad counts."""
        m = self.l.max(1)
        rest = -np.expm1(self.d[self.rows, self.at])
        return np.maximum(rest, 2.0**-22 * np.clip(np.abs(m), 1.0, 2.0**20))

    def grad(self, g, half):
        """(dx, bound) for the gradients g [m] of the rows' losses."""
        g = np.where(self.has, g, 0.0)
        one = np.zeros_like(self.p)
        one[self.rows, self.at] = 1.0
        rest = -np.expm1(self.d[self.rows, self.at])
        v = self.p.copy()
        v[self.rows, self.at] = -rest
        terms = v * self.s * g[:, None]
        # the exponent's error: both logits', the sum's, two additions'; and of exp itself
        off = self.e + self.e_lse[:, None] + (4 * np.abs(self.d) + 4 * np.abs(self.l - self.l.max(1, keepdims=True)) + 8) * U32
        more = (np.abs(self.p * off * self.s) * np.abs(g)[:, None]) @ np.abs(self.w).T
        top = self.reach() * np.abs(self.s).max() * np.abs(g)
        dx, bound = ref._grad([(terms, self.w)], top, half, more)
        return dx, bound + 4 * U32 * np.abs(dx)     # the normalisers' division and g's
