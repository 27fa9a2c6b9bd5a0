"""bpd_sample_gpu against the definition in float64 (paged_oracle.check_sample)."""
import numpy as np
import pytest
import torch

import paged_oracle as O
from bpd_substrate_amd import serve

pytestmark = pytest.mark.gpu


def run(dev, x, u, t=None, k=None, p=None, m=None):
    B = x.shape[0]
    f = lambda a, dt: None if a is None else torch.tensor(np.broadcast_to(a, B).copy(), dtype=dt, device=dev)  # noqa: E731
    u, t, p, m = (f(a, torch.float32) for a in (u, t, p, m))
    k = f(k, torch.int32)
    tok, lp, kept = (a.cpu().numpy() for a in serve.sample(x, u, temperature=t, top_k=k, top_p=p, min_p=m))
    get = lambda a, i, off: off if a is None else float(a[i])  # noqa: E731
    rows = O.f64(x)
    for i in range(B):
        O.check_sample(rows[i], int(tok[i]), float(lp[i]), int(kept[i]), float(u[i]), get(t, i, 1.0),
                       int(get(k, i, 0)), get(p, i, 1.0), get(m, i, 0.0))
    return tok, lp, kept


def logits(seed, B, V, dtype=torch.float32, sigma=2.0):
    r = np.random.default_rng(seed)
    x = r.standard_normal((B, V)) * sigma
    for b in range(B):
        at = r.integers(0, V, min(V, 20))
        x[b, at] += 5 + 3 * r.standard_normal(len(at))
    return torch.from_numpy(x).to(dtype)


FILTERS = [{}, {"t": 0.7}, {"k": 1}, {"k": 5}, {"k": 50, "t": 1.3}, {"p": 0.9}, {"p": 0.1}, {"p": 0.9, "k": 30, "t": 0.6},
           {"m": 0.05}, {"m": 0.05, "p": 0.95, "k": 40}, {"t": 0.0}, {"t": 0.0, "k": 3, "p": 0.5}, {"p": 0.0}, {"m": 1.0},
           {"m": 2.0}, {"k": 10 ** 9}, {"k": -4}, {"p": 2.0}, {"t": 100.0, "p": 0.999}, {"t": 1e-3}, {"p": -1.0}]


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 4097, 32000])
@pytest.mark.parametrize("f", range(len(FILTERS)))
def test_filters(dev, V, f):
    r = np.random.default_rng(f * 100 + V)
    run(dev, logits(V + f, 6, V).to(dev), r.random(6).astype(np.float32), **FILTERS[f])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [37, 50257, 128256, 131075, 300001])
def test_types_and_sizes(dev, dtype, V):
    """16-bit logits have long runs of equal values: ties at every cut."""
    r = np.random.default_rng(V)
    B = 7
    run(dev, logits(V, B, V, dtype).to(dev), r.random(B).astype(np.float32), t=r.uniform(0.4, 1.5, B), k=r.integers(0, 90, B),
        p=r.uniform(0.3, 1.2, B), m=r.uniform(-0.05, 0.1, B))


@pytest.mark.parametrize("f", [{}, {"k": 7}, {"p": 0.5}, {"k": 10, "p": 0.5}, {"m": 0.5}, {"p": 0.999}, {"k": 999}])
@pytest.mark.parametrize("levels", [1, 2, 3])
def test_equal_logits_go_by_index(dev, f, levels):
    r = np.random.default_rng(levels)
    x = torch.from_numpy(r.integers(0, levels, (5, 3001)).astype(np.float32)).to(dev)
    u = np.array([0.0, 0.2, 0.5, 0.9, 1 - 2.0 ** -24], np.float32)
    run(dev, x, u, **f)


@pytest.mark.parametrize("f", [{}, {"k": 3}, {"p": 0.7}, {"m": 0.1}, {"t": 0.0}, {"k": 700, "p": 0.99}])
def test_special_values(dev, f):
    V, inf, nan = 700, float("inf"), float("nan")
    x = logits(5, 12, V).clone()
    x[0] = nan
    x[1] = -inf
    x[2, ::2] = nan
    x[3, 5:] = -inf
    x[4, [3, 77, 300]] = inf
    x[5] = torch.finfo(torch.float32).min           # a mask of the type's lowest value in every place
    x[6, 10:] = torch.finfo(torch.float32).min
    x[7] = -0.0
    x[7, ::3] = 0.0
    x[8, 699] = 1e38
    x[9, :] = nan
    x[9, 698] = -3.0
    x[10] = torch.linspace(-3e38, 3e38, V)
    x[11, 0] = 1e4
    u = np.linspace(0, 1, 12, endpoint=False).astype(np.float32)
    run(dev, x.to(dev), u, **f)


@pytest.mark.parametrize("t", [1e-38, 1e-20, 1e-12, 1e-5, 1e10, 1e38, float("inf")])
@pytest.mark.parametrize("V", [700, 40000])
def test_extreme_temperatures(dev, t, V):
    """Some rows' ranges have no binary32 distance, some temperatures leave the largest logit alone."""
    x = logits(8, 5, V).clone()
    x[0] = x[0] * 1e4
    x[1] = torch.from_numpy(np.linspace(-3e38, 3e38, V))
    x[2] = x[2] * 1e-30
    x[3, ::2] = -float("inf")
    for f in ({}, {"p": 0.9}, {"k": 20, "p": 0.99}, {"m": 0.2}):
        run(dev, x.to(dev), np.array([0.1, 0.4, 0.5, 0.9, 0.99], np.float32), t=t, **f)


@pytest.mark.parametrize("V", [5000, 40000])
def test_more_equal_logits_than_are_listed(dev, V):
    x = torch.zeros(4, V)
    x[1, 7] = 1.0
    x[2, ::2] = -5.0
    x[3, V // 2] = 12.0
    for f in ({"k": 10}, {"p": 0.5}, {"k": 4500, "p": 0.3}, {"m": 0.9}, {"k": 4999, "m": 0.5, "p": 0.9}, {}):
        run(dev, x.to(dev), np.array([0.2, 0.6, 0.0, 0.97], np.float32), **f)


def test_random_numbers_at_the_borders(dev):
    x = torch.zeros(6, 8)
    tok, _, _ = run(dev, x.to(dev), np.array([0.0, 0.125, 0.124999, 0.875, 1 - 2.0 ** -24, 0.5], np.float32))
    assert tok.tolist() == [0, 1, 0, 7, 7, 4]
    # outside [0, 1): the nearest token, never one out of range
    tok, _, _ = serve.sample(x.to(dev), torch.tensor([-1.0, 1.0, 5.0, float("nan"), 0.0, 0.0], device=dev))
    assert tok.tolist() == [0, 7, 7, 0, 0, 0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("off,stride", [(1, 1003), (3, 1001), (0, 1500), (5, 1000)])
def test_rows_at_any_place(dev, dtype, off, stride):
    """Rows that begin at no 16-byte border, neighbours of NaN around them."""
    B, V = 5, 990
    flat = torch.full((off + B * stride + 20,), float("nan"), dtype=dtype, device=dev)
    x = torch.as_strided(flat, (B, V), (stride, 1), off)
    x.copy_(logits(3, B, V, dtype))
    run(dev, x, np.linspace(0.05, 0.95, B).astype(np.float32), t=0.9, p=0.95)


def test_draws_follow_the_weights(dev):
    """Over 4,096 equally spaced random numbers each token comes up as often as its weight says, to one."""
    B, V = 4096, 50
    x = logits(8, 1, V).to(dev)
    u = ((torch.arange(B, device=dev) + 0.5) / B).float()
    tok, lp, _ = serve.sample(x.expand(B, V).contiguous(), u)
    w = torch.softmax(x[0].double().cpu(), 0)
    n = torch.bincount(tok.cpu().long(), minlength=V)
    assert ((n - B * w).abs() <= 1.0 + 1e-6 * B).all()


def test_sample_large_offsets(dev):
    """Rows beyond 2^31 elements."""
    B, V = 5, 1000
    stride = (1 << 29) + 8
    flat = torch.empty(stride * (B - 1) + V, dtype=torch.float16, device=dev)
    x = torch.as_strided(flat, (B, V), (stride, 1))
    x.copy_(logits(4, B, V, torch.float16))
    run(dev, x, np.linspace(0.05, 0.95, B).astype(np.float32), k=40)


def test_sample_captured(dev):
    B, V = 9, 33000
    x, u = torch.zeros(B, V, device=dev), torch.zeros(B, device=dev)
    p = torch.full((B,), 0.95, device=dev)
    k = torch.full((B,), 60, dtype=torch.int32, device=dev)
    serve.sample(x, u, top_p=p, top_k=k)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        out = serve.sample(x, u, top_p=p, top_k=k)
    for i in range(4):
        x.copy_(logits(20 + i, B, V))
        u.copy_(torch.rand(B, generator=torch.Generator(device=dev).manual_seed(i), device=dev))
        want = [a.clone() for a in serve.sample(x, u, top_p=p, top_k=k)]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_no_rows_and_no_vocabulary(dev):
    t, lp, k = serve.sample(torch.zeros(0, 10, device=dev), torch.zeros(0, device=dev))
    assert t.shape == lp.shape == k.shape == (0,)
    t, lp, k = serve.sample(torch.zeros(3, 0, device=dev), torch.zeros(3, device=dev))
    assert t.tolist() == [-1] * 3 and k.tolist() == [0] * 3 and lp.isnan().all()


@pytest.mark.parametrize("V", [16384, 16385, 32768, 32769, 40000])
@pytest.mark.parametrize("k", [None, 40, 4096, 4097])
def test_sizes_where_the_launches_change(dev, V, k):
    run(dev, logits(V, 3, V).to(dev), np.array([0.1, 0.5, 0.9], np.float32), k=k, p=0.9)


def test_equal_largest_threads(dev):
    """The largest logits all next to each other, so few threads hold them; and every thread's largest equal."""
    V = 32000
    x = logits(6, 4, V)
    x[0, :200] += 30
    x[1, 31900:] += 30
    x[2, ::4] = 9.0
    x[3, ::32] = 9.0
    for k in (1, 50, 500):
        run(dev, x.to(dev), np.array([0.1, 0.5, 0.9, 0.99], np.float32), k=k, p=0.95)
