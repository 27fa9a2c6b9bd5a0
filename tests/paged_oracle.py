"""Plain float64 forms of the operators of include/bpdq_serve.h, and random batches for their tests.
Host only (numpy); every unseen row of a cache holds NaN or infinity."""
import numpy as np
import torch

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def f64(t):
    return t.detach().cpu().double().numpy()


class Batch:
    """Sequences with `new` new tokens and `lens` rows of their own each, behind `prefix` shared rows."""

    def __init__(self, seed, new, lens, prefix, H, HKV, D, q="f32", kv="f16", page=16, heads_first=True, pad=0,
                 decode=False, sigma=1.0):
        r = self.r = np.random.default_rng(seed)
        self.new, self.lens, self.P, self.H, self.HKV, self.D, self.page = new, lens, prefix, H, HKV, D, page
        self.qt, self.kvt, B = DT[q], DT[kv], len(lens)
        self.T = sum(new) + pad
        self.start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        per = [-(-l // page) for l in lens]
        npre, W = -(-prefix // page), max(per + [1])
        n_pages = npre + sum(per) + 2
        order = r.permutation(n_pages)
        self.prefix_pages = order[:npre].astype(np.int32)
        self.table = np.full((B, W), -1, np.int32)
        at = npre
        for b, k in enumerate(per):
            self.table[b, :k] = order[at:at + k]
            at += k
        shape = (n_pages, HKV, page, D) if heads_first else (n_pages, page, HKV, D)
        bad = np.where(r.random(shape) < 0.5, np.nan, np.inf)
        mk = lambda: torch.from_numpy(bad).to(self.kvt)  # noqa: E731
        self.kc, self.vc = mk(), mk()
        if heads_first:
            self.kc, self.vc = self.kc.transpose(1, 2), self.vc.transpose(1, 2)
        val = lambda *s: torch.from_numpy(r.standard_normal(s) * sigma)  # noqa: E731
        for i in range(prefix):
            self.kc[self.prefix_pages[i // page], i % page] = val(HKV, D).to(self.kvt)
            self.vc[self.prefix_pages[i // page], i % page] = val(HKV, D).to(self.kvt)
        for b in range(B):
            for i in range(lens[b]):
                self.kc[self.table[b, i // page], i % page] = val(HKV, D).to(self.kvt)
                self.vc[self.table[b, i // page], i % page] = val(HKV, D).to(self.kvt)
        self.q = val(self.T, H, D).to(self.qt)
        self.decode = decode
        assert not decode or (all(n == 1 for n in new) and not pad)

    def tokens(self):
        """(token, sequence, index in its own part)"""
        return [(int(self.start[b]) + j, b, self.lens[b] - self.new[b] + j) for b in range(len(self.lens))
                for j in range(self.new[b])]

    def rows(self, pages, n):
        """k, v [n][HKV][D] of the first n rows; rows of pages outside the cache are left out."""
        keep = [i for i in range(max(n, 0)) if 0 <= pages[i // self.page] < self.kc.shape[0]]
        pick = lambda c: np.stack([f64(c[pages[i // self.page], i % self.page]) for i in keep]) if keep else \
            np.zeros((0, self.HKV, self.D))  # noqa: E731
        return pick(self.kc), pick(self.vc)

    def device(self, dev):
        """PagedCache, PagedBatch and q on the device, the layout kept."""
        from bpd_substrate_amd import serve

        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
        lay = lambda c: (c.transpose(1, 2).contiguous().to(dev).transpose(1, 2) if not c.is_contiguous() else c.to(dev))  # noqa: E731
        self.cache = serve.PagedCache(lay(self.kc), lay(self.vc))
        self.batch = serve.PagedBatch(t(self.table), t(np.asarray(self.lens, np.int32)),
                                      q_start=None if self.decode else t(self.start), n_tokens=self.T,
                                      prefix=t(self.prefix_pages) if self.P else None, prefix_len=self.P)
        return self.cache, self.batch, self.q.to(dev)

    def attention(self, scale=None):
        """(out, lse, bound of out's error, bound of lse's) in float64; rows of no sequence NaN.

        Bounds: a score is a sum of D products in fp32 (u = 2^-24 of the absolute sum per operation, D + 2
        of them; fp32 queries split into parts keep 2^-21 of it), its exponential's argument and the
        exponential carry some units more, the weights are rounded to the cache's type before
        the second product (half a step each) when q has that type, sums run over N terms in fp32, and the
        result is rounded once."""
        D, G, u = self.D, self.H // self.HKV, 2.0 ** -24
        scale = D ** -0.5 if scale is None else scale
        q = f64(self.q)
        out = np.full((self.T, self.H, D), np.nan)
        lse, eo, el = np.full((self.T, self.H), np.nan), np.full_like(out, np.nan), np.full((self.T, self.H), np.nan)
        pk, pv = self.rows(self.prefix_pages, self.P)
        own = [self.rows(self.table[b], self.lens[b]) for b in range(len(self.lens))]
        for t, b, i in self.tokens():
            ok, ov = self.rows(self.table[b], i + 1) if (self.table[b] < 0).any() else (own[b][0][:max(i + 1, 0)],
                                                                                       own[b][1][:max(i + 1, 0)])
            k, v = np.concatenate([pk, ok]), np.concatenate([pv, ov])
            n = len(k)
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
                ds = (D + 2 + (8 if self.qt is torch.float32 else 0)) * u * a + 6 * u * (np.abs(s).max() + abs(m)) + 4 * u
                dw = 0.0 if self.qt is torch.float32 else HALF_STEP[self.kvt]
                spread = np.abs(w) @ np.abs(vh) / l
                eo[t, h] = HALF_STEP[self.qt] * np.abs(out[t, h]) + spread * (2 * ds + 2 * dw + 2 * (n + 8) * u) + 2.0 ** -25
                el[t, h] = ds + (n + 8) * u + dw + 2 * u * abs(lse[t, h])
        return out, lse, eo, el


def rope(x, pos, rot, neox, base=10000.0, factors=None):
    """x [heads][D] float64 rotated at position pos, in float64 with the angle reduced in extended precision."""
    y = x.copy()
    f = factors if factors is not None else np.ones(rot // 2)
    for j in range(rot // 2):
        a, b = (j, j + rot // 2) if neox else (2 * j, 2 * j + 1)
        ang = np.fmod(np.longdouble(pos) * np.longdouble(base ** (-2.0 * j / rot) / f[j]), 2 * np.longdouble(np.pi))
        c, s = float(np.cos(ang)), float(np.sin(ang))
        y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, a] * s + x[:, b] * c
    return y


def rope_bound(x, rot, neox, dtype, ref):
    """Rounding once to dtype, and in fp32 the angle (pi 2^-25 half revolutions, and what a position of
    2^20 leaves in binary64), sine and cosine (2 units) and three operations on |a| + |b|."""
    m = np.zeros_like(x)
    for j in range(rot // 2):
        a, b = (j, j + rot // 2) if neox else (2 * j, 2 * j + 1)
        m[:, a] = m[:, b] = np.abs(x[:, a]) + np.abs(x[:, b])
    least = 2.0 ** -25 if dtype is torch.float16 else 2.0 ** -134   # half the smallest step
    return HALF_STEP[dtype] * np.abs(ref) + 8 * 2.0 ** -24 * m * (1 + HALF_STEP[dtype]) + least


def check_sample(x, token, logprob, kept, u, t=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row's result against the definition.  Weights are multiples of 2^-44 (vocab up to 2^18) of the
    largest, each off by 2^-45, and before that by (3 y + 4) 2^-53 of itself, y = (max - l) / t: three
    roundings of y and four of the exponential's parts.  As exp(-y) y <= 1 / e, that is at most 2^-45 + 2^-52 +
    2^-51 of itself; a border between cumulated sums may fall on either side within `slack`, nothing else
    may differ."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    V = len(x)
    if V == 0 or x.max() == -np.inf:
        assert (token, kept) == (-1, 0) and np.isnan(logprob)
        return
    order = np.lexsort((np.arange(V), -x))
    order = order[x[order] > -np.inf]
    top = x[order[0]]
    if not t > 0:
        assert (token, kept, logprob) == (order[0], 1, 0.0), (token, order[0], kept, logprob)
        return
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.nan_to_num(np.exp((x[order] - top) / t)))
    slack = len(order) * 2.0 ** -44 + 2.0 ** -50 * w.sum()
    n = len(order) if not 0 < top_k < len(order) else top_k
    lo = hi = n
    if top_p < 1:
        c = np.cumsum(w[:n])
        need = max(top_p, 0.0) * c[-1]
        lo = min(n, int(np.searchsorted(c, need - slack)) + 1)
        hi = min(n, int(np.searchsorted(c, need + slack)) + 1)
    if min_p > 0:
        m = min(min_p, 1.0)
        near = (3 * -np.log(m) + 4) * 2.0 ** -53     # where w is about min_p, y is about -log(min_p)
        lo, hi = min(lo, max(1, int((w >= m * (1 + near)).sum()))), min(hi, max(1, int((w >= m * (1 - near)).sum())))
    assert lo <= kept <= hi, (kept, lo, hi)
    left = np.sort(order[:kept])
    place = {int(i): j for j, i in enumerate(order)}
    wi = np.array([w[place[int(i)]] for i in left])
    c = np.cumsum(wi)
    j = int(np.searchsorted(left, token))
    assert j < len(left) and left[j] == token, f"token {token} is not among the {kept} left"
    at = min(max(u, 0.0), 1.0) * c[-1]
    assert (c[j - 1] if j else 0.0) <= at + slack and at <= c[j] + slack, (token, c[j - 1] if j else 0, at, c[j])
    want = np.log(wi[j] / c[-1])
    off = 2.0 ** -44 / max(wi[j], 2.0 ** -44) + slack / c[-1] + 2.0 ** -24 * abs(want) + 2.0 ** -50
    assert abs(logprob - want) <= off, (logprob, want, off)
