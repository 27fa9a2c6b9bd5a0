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
        f32 = self.qt is O.torch.float32
        for b in range(len(self.lens)):
            t0, n = int(self.start[b]), self.new[b]
            if n == 0:
                continue
            index = self.lens[b] - n + np.arange(n)
            rows = [(j, self.prefix_pages[j // self.page], j % self.page) for j in range(self.P)]
            rows += [(self.P + j, self.table[b, j // self.page], j % self.page) for j in range(max(self.lens[b], 0))
                     if j // self.page < self.table.shape[1]]
            rows = [r for r in rows if 0 <= r[1] < self.kc.shape[0]]
            j = np.array([r[0] for r in rows], np.int64)
            k, v = (O.f64(c[[r[1] for r in rows], [r[2] for r in rows]]) if rows else np.zeros((0, self.HKV, D))
                    for c in (self.kc, self.vc))
            p = (self.P + index)[:, None]
            seen = ((j < self.P) | (j <= p)) & ((j > p - window) | (j < sinks))
            count = seen.sum(1)
            # rows that none sees may hold anything
            k, v = (np.where(seen.any(0)[:, None, None], c, 0.0) for c in (k, v))
            for h in range(self.H):
                kh, vh, qh = k[:, h // G], v[:, h // G], q[t0:t0 + n, h]
                s = np.where(seen, scale * (qh @ kh.T), -np.inf)
                a = np.where(seen, abs(scale) * (np.abs(qh) @ np.abs(kh).T), 0.0).max(1, initial=0.0)
                m = s.max(1, initial=-np.inf)
                some = count > 0
                m0 = np.where(some, m, 0.0)
                w = np.exp(s - m0[:, None])
                l = w.sum(1)
                l1 = np.where(some, l, 1.0)
                o = w @ vh / l1[:, None]
                out[t0:t0 + n, h] = o
                with np.errstate(divide="ignore"):
                    lse[t0:t0 + n, h] = np.where(some, m0 + np.log(l1), -np.inf)
                top = np.where(seen, np.abs(s), 0.0).max(1, initial=0.0)
                ds = (D + 2 + (8 if f32 else 0)) * u * a + 6 * u * (top + np.abs(m0)) + 4 * u
                dw = 0.0 if f32 else O.HALF_STEP[self.kvt]
                spread = w @ np.abs(vh) / l1[:, None]
                e = O.HALF_STEP[self.qt] * np.abs(o) + spread * (2 * ds + 2 * dw + 2 * (count + 8) * u)[:, None] + 2.0 ** -25
                eo[t0:t0 + n, h] = np.where(some[:, None], e, 0.0)
                el[t0:t0 + n, h] = np.where(some, ds + (count + 8) * u + dw + 2 * u * np.abs(m0 + np.log(l1)), 0.0)
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
