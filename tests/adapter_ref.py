"""Low-rank adapters beside an int8 linear layer in 64 bits (numpy), and how far a 32-bit evaluation may be."""
import numpy as np

import scaled_ref as ref

U32 = ref.U32

# m, k, n, rank, adapters. The second half: sizes found by search, the cheapest that reach a kernel
# (test_layer_operators_host.py checks that all are). The first: decode batches (rows rounded in the kernel, in slices, joined), every tile, odd sizes,
# ranks from 1 to the largest, fewer and more adapters than rows
CASES = [(1, 64, 48, 1, 1), (1, 4096, 1000, 16, 3), (3, 120, 72, 5, 2), (5, 8192, 600, 8, 4), (16, 1000, 333, 16, 40),
         (2, 17000, 90, 7, 2), (17, 4096, 700, 16, 9), (33, 640, 4096, 33, 5), (48, 4096, 4300, 16, 32),
         (64, 14336, 500, 128, 3), (64, 100, 9000, 3, 64), (9, 0, 40, 4, 2), (70, 0, 40, 4, 2), (65, 64, 64, 16, 2), (66, 130, 129, 17, 3),
         (200, 127, 63, 5, 4), (300, 999, 1001, 5, 3), (400, 4096, 900, 8, 2), (256, 256, 256, 64, 1), (700, 1024, 3000, 16, 7),
         (1000, 512, 2500, 20, 5), (513, 2048, 4500, 128, 2), (2050, 400, 2300, 12, 6), (1030, 1030, 5000, 32, 3),
         (3000, 256, 300, 16, 100), (130, 3000, 40, 9, 1),
         (2621, 428, 2717, 128, 3), (1214, 479, 6299, 64, 1), (3864, 398, 2013, 20, 9), (3544, 1097, 82, 64, 9), (4907, 2338, 21, 20, 3),
         (2786, 1856, 70, 16, 3), (3138, 4564, 20, 32, 1), (1176, 3509, 167, 64, 9), (4594, 2824, 113, 1, 1), (1218, 87, 24, 128, 9),
         (1480, 87, 27, 128, 3), (5122, 65, 27, 128, 9), (797, 109, 61, 128, 1), (1571, 85, 45, 128, 3), (1, 63, 5390, 7, 9), (1, 88, 4586, 32, 1),
         (1, 61, 6923, 7, 9), (17, 66, 4380, 50, 1), (58, 66, 4234, 32, 3), (1, 68, 8238, 16, 9), (1, 65, 9839, 32, 9), (1, 166, 11406, 16, 1),
         (19, 80, 8501, 64, 3), (44, 71, 9402, 128, 9), (1, 65, 17170, 16, 1), (1, 79, 13932, 1, 1), (1, 87, 13403, 50, 9),
         (17, 85, 13993, 32, 9), (33, 97, 12457, 128, 1), (55, 87, 13783, 32, 3)]


class Adapted:
    """x the rows' values for the adapters, q and t their int8 form; w, s, bias the layer; down, up, c, which."""

    def __init__(self, x, q, t, w, s, bias, down, up, c, which, unit):
        self.x, self.w, self.s, self.c = (np.asarray(a, np.float64) for a in (x, w, s, c))
        self.down, self.up = down.astype(np.float64), up.astype(np.float64)
        self.which, self.unit, self.base = which, unit, (q, t, w, s, bias)
        self.u, self.eu = self._first(self.x, self.down)

    def rows(self, a):
        return np.nonzero(self.which == a)[0]

    def _first(self, x, p):
        """c x . p_a^T and its error: 32 products and additions at a time, then those, of lanes and waves."""
        m, k = x.shape
        u, e = np.zeros((m, p.shape[1])), np.zeros((m, p.shape[1]))
        for a in range(p.shape[0]):
            i = self.rows(a)
            u[i] = self.c * x[i] @ p[a].T
            e[i] = abs(self.c) * (np.abs(x[i]) @ np.abs(p[a]).T) * (k / 32 + 64) * 2 * U32
        return u, e

    def _second(self, u, eu, p):
        """u . p_a (p_a [r, cols]) and its error: u in two 16-bit halves of `unit` (float16 ones in steps of 2^-38 of
        the row's largest), rank products."""
        m, r = u.shape
        y, e = np.zeros((m, p.shape[2])), np.zeros((m, p.shape[2]))
        top = np.abs(u).max(1, keepdims=True, initial=0.0)
        off = eu + self.unit * np.abs(u) + 2.0**-38 * top
        for a in range(p.shape[0]):
            i = self.rows(a)
            y[i] = u[i] @ p[a]
            e[i] = off[i] @ np.abs(p[a]) + (np.abs(u[i]) @ np.abs(p[a])) * (r + 8) * 2 * U32
        return y, e

    def forward(self):
        y, b = ref.linear(*self.base)
        d, e = self._second(self.u, self.eu, self.up.transpose(0, 2, 1))
        return y + d, b + e + U32 * np.abs(y + d)

    def grad(self, dy, half):
        """(dx, ddown, dup), each with its bound."""
        dy = dy.astype(np.float64)
        h, eh = self._first(dy, self.up.transpose(0, 2, 1))
        dx, b = ref.linear_grad(dy, self.w, self.s, half)
        d, e = self._second(h, eh, self.down)
        m = len(dy)
        depth = m / 4 + 64      # 4 rows' products at a time
        dd, ed = np.zeros_like(self.down), np.zeros_like(self.down)
        du, eu = np.zeros_like(self.up), np.zeros_like(self.up)
        for a in range(len(self.down)):
            i = self.rows(a)
            dd[a] = h[i].T @ self.x[i]
            ed[a] = (eh[i] + np.abs(h[i]) * depth * 2 * U32).T @ np.abs(self.x[i])
            du[a] = dy[i].T @ self.u[i]
            eu[a] = np.abs(dy[i]).T @ (self.eu[i] + np.abs(self.u[i]) * depth * 2 * U32)
        return (dx + d, b + e + U32 * np.abs(dx + d)), (dd, ed), (du, eu)
