"""The paged 4-bit cache and attention over it, restated plainly: numpy, row
by row, 64-bit sums. Test infrastructure for tests/test_kv4.py."""

import numpy as np

F16MAX = np.float32(65504.0)


def tile_bytes(dk, dv):
    return 16 * (dk // 2 + dv // 2 + 8)


def quantize(x):
    """Rows x [..., d] float32 to (codes, scale, minimum), each step one f32
    operation."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        lo, hi = x.min(-1), x.max(-1)
        s = np.minimum((hi - lo) / np.float32(15.0), F16MAX).astype(np.float16)
        m = np.clip(lo, -F16MAX, F16MAX).astype(np.float16)
        c = np.clip(np.rint((x - m.astype(np.float32)[..., None]) / s.astype(np.float32)[..., None]), 0, 15)
    bad = ~np.isfinite(x).all(-1)
    c[(s == 0) | bad] = 0
    s[bad] = np.nan
    m[bad] = np.nan
    return c.astype(np.uint8), s, m


class Cache:
    """Values as the format holds them, by (page, head, slot)."""

    def __init__(self, pages, heads, page, dk, dv):
        self.k = np.full((pages, heads, page, dk), np.nan)
        self.v = np.full((pages, heads, page, dv), np.nan)
        self.page, self.pages = page, pages

    def place(self, table, s, pos):
        if pos < 0 or pos // self.page >= table.shape[1]:
            return None
        p = int(table[s, pos // self.page])
        return (p, pos % self.page) if 0 <= p < self.pages else None

    def append(self, k, v, table, lens, start):
        kq, vq = [m.astype(np.float64)[..., None] + s.astype(np.float64)[..., None] * c
                  for c, s, m in (quantize(k), quantize(v))]
        for s in range(len(lens)):
            n = start[s + 1] - start[s]
            for i in range(n):
                at = self.place(table, s, int(lens[s]) - n + i)
                if at:
                    self.k[at[0], :, at[1]] = kq[start[s] + i]
                    self.v[at[0], :, at[1]] = vq[start[s] + i]

    def read(self, table, lens, start, rows):
        k = np.zeros((rows,) + self.k.shape[1:2] + self.k.shape[3:])
        v = np.zeros((rows,) + self.v.shape[1:2] + self.v.shape[3:])
        for s in range(len(lens)):
            n = start[s + 1] - start[s]
            for i in range(n):
                at = self.place(table, s, int(lens[s]) - n + i)
                if at:
                    k[start[s] + i], v[start[s] + i] = self.k[at[0], :, at[1]], self.v[at[0], :, at[1]]
        return k, v

    def attend(self, q, table, lens, start, scale, window, sink):
        """(out, b, top): b bounds scale * sum |q| |k| as the codes make it,
        top the values' magnitude, per row and head, for tolerances."""
        rows, hq, dk = q.shape
        H = self.k.shape[1]
        out = np.zeros((rows, hq, self.v.shape[-1]))
        b, top = np.zeros((rows, hq, 1)), np.zeros((rows, hq, 1))
        for s in range(len(lens)):
            n = start[s + 1] - start[s]
            places = [self.place(table, s, j) for j in range(max(int(lens[s]), 0))]
            exists = np.array([p is not None for p in places], bool)
            where = np.array([p or (0, 0) for p in places]).reshape(-1, 2)
            key = np.arange(len(places))
            for i in range(n):
                pos = int(lens[s]) - n + i
                seen = exists & (key <= pos) & ((key > pos - window) | (key < sink) | (window <= 0))
                if not seen.any():
                    continue
                pg, sl = where[seen].T
                r = start[s] + i
                for g in range(hq):
                    h = g // (hq // H)
                    kk, vv = self.k[pg, h, sl], self.v[pg, h, sl]
                    x = kk @ q[r, g].astype(np.float64) * scale
                    with np.errstate(all="ignore"):
                        p = np.exp(x - x.max())
                        out[r, g] = (p / p.sum()) @ vv
                    b[r, g] = abs(scale) * np.abs(q[r, g].astype(np.float64)).sum() * 2 * np.abs(kk).max()
                    top[r, g] = 2 * np.abs(vv).max()
        return out, b, top
