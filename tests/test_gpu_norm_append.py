"""bpd_norm_rope_append_paged_gpu against a plain float64 form."""
import numpy as np
import pytest
import torch

import paged_oracle as O
from bpd_substrate_amd import serve

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def normed(x, w, eps):
    """x [heads][D], w [D] or [heads][D] or None: (normed, bound of its error in binary32 before the rotation).

    D products and sums, the mean and eps: (D + 4) u of the sum; half of that in its root, which with the division has
    3 u more; two products."""
    if w is None:
        return x, np.zeros_like(x)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    return y, ((x.shape[-1] + 4) / 2 + 5) * U * np.abs(y)


def rotated(y, err, pos, rot, neox, dtype):
    """(rotated, bound): the rotation's bound, and the errors of both elements of a pair."""
    ref = O.rope(y, pos, rot, neox)
    e = err.copy()
    for j in range(rot // 2):
        a, b = (j, j + rot // 2) if neox else (2 * j, 2 * j + 1)
        e[:, a] = e[:, b] = err[:, a] + err[:, b]
    return ref, O.rope_bound(y, rot, neox, dtype, ref) + e * (1 + O.HALF_STEP[dtype])


def run(dev, seed, new, lens, P, H, HKV, D, x, kv, page, heads_first, pad, rot, neox, w, which="qk", per_head=False,
        decode=False, in_place=False, eps=1e-6, scale=1.0):
    b = O.Batch(seed, new, lens, P, H, HKV, D, "f32", kv, page, heads_first, pad, decode)
    r, xt, wt = b.r, O.DT[x], O.DT[w]
    row = torch.from_numpy(r.standard_normal((b.T, H + 2 * HKV, D)) * scale).to(xt)
    q, k, v = row[:, :H], row[:, H:H + HKV], row[:, H + HKV:]
    mk = lambda h: torch.from_numpy(1 + 0.3 * r.standard_normal((h, D) if per_head else D)).to(wt)  # noqa: E731
    qw, kw = mk(H) if "q" in which else None, mk(HKV) if "k" in which else None
    cache, batch, _ = b.device(dev)
    rowd = row.to(dev)
    qd, kd, vd = rowd[:, :H], rowd[:, H:H + HKV], rowd[:, H + HKV:]
    rope = serve.Rope(rot, neox=neox, device=dev) if rot else None
    at = lambda t: None if t is None else t.to(dev)  # noqa: E731
    before_k, before_v = cache.k.clone(), cache.v.clone()
    qo = qd if in_place else torch.full((b.T, H, D), 7.0, dtype=xt, device=dev)
    got = serve.rope_append(cache, batch, qd, kd, vd, rope=rope, q_out=qo, q_norm=at(qw), k_norm=at(kw), eps=eps)
    assert got is qo
    got, kc, vc = O.f64(got), O.f64(cache.k), O.f64(cache.v)
    want_k, want_v = O.f64(before_k), O.f64(before_v)
    untouched = np.ones(kc.shape[:2], bool)
    free = np.ones(b.T, bool)
    for t, s, i in b.tokens():
        free[t] = False
        f = lambda z, ww, dt: rotated(*normed(O.f64(z[t]), None if ww is None else O.f64(ww), eps), P + i, rot, neox, dt)  # noqa: E731,B023
        ref, bound = f(q, qw, xt)
        assert (np.abs(got[t] - ref) <= bound).all(), (t, (np.abs(got[t] - ref) - bound).max())
        if i < 0:
            continue
        page_, row_ = b.table[s, i // page], i % page
        ref, bound = f(k, kw, b.kvt)
        assert (np.abs(kc[page_, row_] - ref) <= bound).all(), (t, (np.abs(kc[page_, row_] - ref) - bound).max())
        assert np.array_equal(vc[page_, row_], O.f64(v[t].to(b.kvt)))
        untouched[page_, row_] = False
    assert np.array_equal(kc[untouched], want_k[untouched], equal_nan=True)
    assert np.array_equal(vc[untouched], want_v[untouched], equal_nan=True)
    if not in_place:
        assert (got[free] == 7.0).all()


CASES = [  # new, lens, P, H, HKV, D, x, kv, page, heads_first, pad, rot, neox, weights
    ([1], [1], 0, 1, 1, 8, "f32", "f16", 1, True, 0, 8, False, "f32"),
    ([1, 1], [70, 9], 5, 4, 2, 64, "f16", "f16", 16, True, 0, 64, True, "f16"),
    ([3, 0, 5], [30, 4, 5], 0, 8, 2, 128, "bf16", "bf16", 16, False, 2, 128, True, "f32"),
    ([3, 0, 5], [30, 4, 5], 77, 8, 2, 128, "f32", "bf16", 16, False, 2, 64, True, "f32"),
    ([7], [20], 0, 5, 5, 96, "f16", "f16", 21, True, 0, 48, True, "f32"),
    ([7], [20], 3, 5, 1, 80, "f16", "bf16", 21, True, 0, 40, True, "f16"),       # halves of 20: no whole vectors
    ([7], [20], 3, 5, 1, 80, "bf16", "f16", 21, True, 0, 40, False, "bf16"),
    ([4], [400], 0, 20, 10, 256, "f32", "f16", 64, True, 0, 256, True, "f32"),
    ([4], [400], 0, 3, 1, 200, "f16", "f16", 64, True, 0, 6, True, "f32"),        # a few elements turn
    ([4], [400], 0, 3, 1, 200, "bf16", "bf16", 64, False, 0, 0, False, "bf16"),   # none do
    ([5], [3], 9, 2, 2, 64, "f32", "f16", 16, True, 0, 64, False, "f32"),         # more new tokens than rows
]
MANY = [  # more tokens than take four waves each: two waves, and one where a token has few heads
    ([600, 1, 505], [600, 9, 700], 5, 16, 2, 128, "bf16", "bf16", 16, True, 3, 64, True, "f32"),
    ([1100], [1100], 0, 15, 3, 80, "f16", "f16", 21, False, 0, 40, True, "f16"),
    ([700, 400], [800, 400], 0, 7, 1, 64, "f32", "f16", 16, True, 1, 64, False, "f32"),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", range(len(MANY)))
def test_many_tokens(dev, case, in_place):
    run(dev, 795 + case, *MANY[case], per_head=case == 1, in_place=in_place)


@pytest.mark.parametrize("case", range(len(CASES)))
def test_norm_and_append(dev, case):
    run(dev, 700 + case, *CASES[case])


@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("case", [1, 5, 6])
def test_one_of_both_is_normed(dev, case, which):
    run(dev, 720 + case, *CASES[case], which=which)


@pytest.mark.parametrize("case", [1, 2, 5, 7])
def test_weights_of_each_head(dev, case):
    run(dev, 740 + case, *CASES[case], per_head=True)


@pytest.mark.parametrize("case", [1, 3, 5, 6, 8])
def test_in_place(dev, case):
    run(dev, 760 + case, *CASES[case], in_place=True)


@pytest.mark.parametrize("case", [0, 1])
def test_one_token_each(dev, case):
    run(dev, 780 + case, *CASES[case], decode=True)


@pytest.mark.parametrize("scale,eps", [(1e-18, 1e-6), (1e-6, 1e-6), (1e15, 1e-6), (1.0, 0.0), (1.0, 10.0)])
def test_small_and_large_heads(dev, scale, eps):
    run(dev, 790, [3], [9], 0, 4, 2, 64, "f32", "bf16", 16, True, 0, 64, True, "f32", scale=scale, eps=eps)


def test_a_head_of_zeros_and_one_that_is_no_number(dev):
    """Zeros stay zeros (eps holds the division up), and a NaN stays in its head."""
    cache = serve.PagedCache.empty(2, 16, 2, 64, torch.float16, device=dev)
    lens = torch.tensor([4], dtype=torch.int32, device=dev)
    batch = serve.PagedBatch(torch.zeros(1, 1, dtype=torch.int32, device=dev), lens)
    w = torch.ones(64, device=dev)
    q, k = torch.zeros(1, 4, 64, device=dev), torch.zeros(1, 2, 64, device=dev)
    q[0, 1] = 1.0
    q[0, 2, 5] = float("nan")
    out = serve.rope_append(cache, batch, q, k, k, rope=serve.Rope(64, device=dev), q_norm=w, k_norm=w)
    assert (out[0, 0] == 0).all() and torch.isfinite(out[0, 1]).all() and torch.isnan(out[0, 2]).all()
    assert (out[0, 3] == 0).all() and (cache.k[0, 3] == 0).all()


def test_q_or_k_alone_and_given_positions(dev):
    b = O.Batch(5, [3, 2], [30, 4], 0, 4, 2, 64, "f16", "f16", 16)
    cache, batch, _ = b.device(dev)
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn(5, h, 64, generator=g).half().to(dev) for h in (4, 2))
    w = torch.ones(64, device=dev)
    rope = serve.Rope(64, neox=True, device=dev)
    pos = torch.tensor([28, 28, 29, 2, 3], dtype=torch.int32, device=dev)
    both = serve.rope_append(cache, batch, q, k, k, rope=rope, q_norm=w, k_norm=w, pos=pos)
    kept = cache.k.clone()
    assert torch.equal(serve.rope_append(cache, batch, q, None, None, rope=rope, q_norm=w, k_norm=w, pos=pos), both)
    cache.k.zero_()
    assert serve.rope_append(cache, batch, None, k, k, rope=rope, q_norm=w, k_norm=w, pos=pos) is None
    t, r = b.table, lambda i: i % 16
    for s, i in ((0, 27), (0, 28), (0, 29), (1, 2), (1, 3)):
        assert torch.equal(cache.k[int(t[s, i // 16]), r(i)], kept[int(t[s, i // 16]), r(i)])
