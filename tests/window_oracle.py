"""Attention over a window and the first rows in float64, with paged_oracle's batches and bounds."""
import numpy as np

import paged_oracle as O


class Batch(O.Batch):
    def attention(self, scale=None, window=1, sinks=0):
        """(out, lse, bound of out's error, bound of lse's): paged_oracle's, over the rows that a token sees."""
        D, G, u = self.D, self.H // self.HKV, 2.0 ** -24
        scale = D ** -0.5 if scale is None else scale
        q = O.f64(self.q)
        out = np.full((self.T, self.H, D), np.nan)
        lse, eo, el = np.full((self.T, self.H), np.nan), np.full_like(out, np.nan), np.full((self.T, self.H), np.nan)
        for t, b, i in self.tokens():
            p = self.P + i
            seen = lambda j: j > p - window or j < sinks  # noqa: E731
            at = [(self.prefix_pages[j // self.page], j % self.page) for j in range(self.P) if seen(j)]
            at += [(self.table[b, j // self.page], j % self.page) for j in range(i + 1)
                   if j // self.page < self.table.shape[1] and seen(self.P + j)]
            at = [(g, r) for g, r in at if 0 <= g < self.kc.shape[0]]
            n = len(at)
            if n:
                g, r = zip(*at)
                k, v = O.f64(self.kc[list(g), list(r)]), O.f64(self.vc[list(g), list(r)])
            for h in range(self.H):
                if n == 0:
                    out[t, h], lse[t, h], eo[t, h], el[t, h] = 0, -np.inf, 0, 0
                    continue
                kh, vh = k[:, h // G], v[:, h // G]
                s = scale * (kh @ q[t, h])
                a = abs(scale) * (np.abs(kh) @ np.abs(q[t, h])).max()
                m = s.max()
                w = np.exp(s - m)
                l = w.sum()
                out[t, h], lse[t, h] = w @ vh / l, m + np.log(l)
                f32 = self.qt is O.torch.float32
                ds = (D + 2 + (8 if f32 else 0)) * u * a + 6 * u * (np.abs(s).max() + abs(m)) + 4 * u
                dw = 0.0 if f32 else O.HALF_STEP[self.kvt]
                spread = np.abs(w) @ np.abs(vh) / l
                eo[t, h] = O.HALF_STEP[self.qt] * np.abs(out[t, h]) + spread * (2 * ds + 2 * dw + 2 * (n + 8) * u) + 2.0 ** -25
                el[t, h] = ds + (n + 8) * u + dw + 2 * u * abs(lse[t, h])
        return out, lse, eo, el

    def slide(self, window, sinks):
        """Takes the pages that no new token sees out of the table, and poisons what stands in them and in every row that
        none sees."""
        for b, n in enumerate(self.lens):
            first = self.P + n - self.new[b] if self.new[b] else self.P + n
            for pg in range(-(-n // self.page)):
                rows = range(pg * self.page, min(n, (pg + 1) * self.page))
                unseen = [r for r in rows if not (self.P + r > first - window or self.P + r < sinks)]
                for r in unseen:
                    self.kc[self.table[b, pg], r % self.page] = self.r.choice([np.nan, np.inf, -np.inf])
                    self.vc[self.table[b, pg], r % self.page] = self.r.choice([np.nan, np.inf, -np.inf])
                if len(unseen) == len(rows):
                    self.table[b, pg] = -1
