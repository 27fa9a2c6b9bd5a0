"""bpd_attn_window_paged_gpu against a plain float64 form (window_oracle)."""
import numpy as np
import pytest
import torch

import paged_oracle as O
from bpd_substrate_amd import serve
from window_oracle import Batch

pytestmark = pytest.mark.gpu


def check(b, dev, window, sinks, scale=None):
    cache, batch, q = b.device(dev)
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=dev)
    got, lse = serve.attention(cache, batch, q, scale=scale, out=out, return_lse=True, window=window, sinks=sinks)
    ref, rlse, eo, el = b.attention(scale, window, sinks)
    got, lse = O.f64(got), O.f64(lse)
    none = np.isnan(ref[:, 0, 0])
    assert (got[none] == 7.0).all(), "rows of no sequence were written"
    assert np.isfinite(got[~none]).all()
    over = np.abs(got - ref)[~none] - eo[~none]
    assert over.max(initial=-1) <= 0, (over.max(), np.unravel_index(over.argmax(), over.shape))
    empty = rlse == -np.inf
    assert np.array_equal(lse[~none] == -np.inf, empty[~none])
    m = ~none[:, None] & ~empty
    assert (np.abs(lse[m] - rlse[m]) <= el[m]).all(), (np.abs(lse[m] - rlse[m]) - el[m]).max()


# new tokens, own rows, prefix, H, HKV, D, q, kv, page, heads_first, padding rows; window, sinks
CASES = [
    (([1], [1], 0, 1, 1, 8, "f16", "f16", 1, True, 0), (1, 0)),
    (([1], [0], 0, 2, 2, 64, "f16", "f16", 16, True, 0), (5, 3)),                     # nothing to see
    (([1], [0], 5, 2, 1, 64, "f32", "bf16", 16, True, 0), (3, 1)),                    # the prefix alone
    (([1, 1, 1], [300, 1, 17], 0, 8, 2, 64, "f16", "f16", 16, True, 0), (64, 4)),
    (([1, 1, 1], [300, 33, 97], 0, 8, 2, 64, "f16", "f16", 16, True, 0), (1, 0)),     # itself alone
    (([1] * 5, [33, 64, 1, 129, 95], 77, 8, 8, 128, "bf16", "bf16", 16, False, 0), (100, 10)),   # windows into the prefix
    (([1] * 3, [40, 500, 7], 130, 32, 8, 128, "f32", "f16", 32, False, 0), (60, 140)),           # sinks behind the prefix
    (([1] * 3, [40, 500, 7], 130, 32, 8, 128, "f32", "bf16", 64, True, 0), (31, 33)),
    (([1] * 2, [100, 31], 61, 5, 1, 80, "f16", "f16", 21, True, 0), (50, 2)),         # pages that end inside every unit
    (([1] * 2, [100, 31], 61, 12, 4, 96, "f32", "f16", 3, False, 0), (37, 65)),
    (([1] * 2, [150, 31], 200, 6, 2, 256, "bf16", "bf16", 64, True, 0), (33, 5)),
    (([1] * 2, [700, 66], 0, 40, 1, 64, "f16", "f16", 16, True, 0), (65, 1)),         # more than 16 heads a kv head
    (([3, 0, 20, 1], [10, 4, 20, 90], 0, 4, 2, 64, "f16", "f16", 16, True, 3), (7, 2)),
    (([3, 0, 70, 1], [10, 0, 170, 90], 50, 8, 2, 128, "bf16", "bf16", 64, True, 2), (64, 0)),
    (([130], [330], 33, 4, 4, 128, "f32", "f16", 16, False, 0), (100, 40)),
    (([150, 9], [400, 9], 90, 4, 2, 96, "f16", "f16", 48, False, 1), (128, 3)),
    (([150], [700], 0, 4, 2, 64, "bf16", "bf16", 16, True, 0), (200, 64)),
    (([5, 5], [3, 5], 0, 2, 2, 64, "f16", "f16", 16, True, 0), (2, 1)),               # more new tokens than rows
    (([40, 33], [45, 200], 64, 4, 2, 256, "f32", "bf16", 32, True, 0), (30, 65)),
    (([200], [200], 0, 2, 1, 64, "f16", "f16", 16, True, 0), (1000, 5)),              # a window beyond everything
    (([200], [300], 70, 2, 1, 64, "f16", "f16", 16, True, 0), (2 ** 31 - 1, 0)),
    (([9], [300], 70, 2, 1, 64, "f16", "f16", 16, True, 0), (4, 2 ** 31 - 1)),        # every row a sink
]


# the same for batches that k_attn_plan lays out, whose tiles k_attn_tile takes
TILES = [
    (([900], [1100], 0, 32, 8, 64, "f16", "f16", 16, True, 0), (2000, 0)),
    (([800, 300, 1, 0, 400], [900, 700, 60, 9, 700], 77, 32, 8, 64, "bf16", "bf16", 16, False, 3), (700, 100)),
    (([600, 500], [600, 900], 130, 32, 8, 128, "bf16", "bf16", 64, True, 0), (401, 140)),
    (([500, 611], [700, 800], 61, 40, 8, 96, "f16", "f16", 21, True, 1), (377, 4)),     # pages that end inside every unit
    (([450, 550], [760, 900], 40, 32, 8, 128, "f32", "bf16", 32, True, 0), (700, 0)),
    (([500, 490], [800, 900], 0, 32, 8, 80, "f32", "f16", 16, False, 0), (900, 33)),
    (([300, 500], [700, 900], 50, 32, 4, 256, "f16", "f16", 16, True, 0), (840, 7)),
]
# one token each, too many rows for a workgroup: units dealt to all waves, and a join
DEALT = [
    (([1] * 2, [2700, 1200], 0, 8, 2, 128, "bf16", "bf16", 64, True, 0), (2400, 4)),
    (([1] * 3, [2600, 40, 1000], 90, 8, 2, 64, "f16", "f16", 16, True, 0), (2500, 95)),
    (([1] * 3, [900, 700, 33], 61, 12, 4, 96, "f32", "f16", 21, False, 0), (700, 3)),
    (([1] * 2, [900, 120], 200, 6, 2, 256, "bf16", "bf16", 64, True, 0), (650, 5)),
    (([1] * 2, [800, 300], 30, 6, 2, 128, "f32", "bf16", 32, True, 0), (700, 0)),
]


def many(B, n, longest, H, HKV, D, q, kv, page, P=0):
    """Lengths of 0 to `longest`, with up to n new tokens each."""
    r = np.random.default_rng(B + D)
    lens = [int(x) for x in r.integers(0, longest + 1, B - 1)] + [longest]
    new = [1 if n == 1 else min(int(x), k) for x, k in zip(r.integers(0, n + 1, B), lens)]
    return new, lens, P, H, HKV, D, q, kv, page, True, 0 if n == 1 else 2


# many sequences of few rows: two waves to a workgroup, or one
CROWDS = [
    (many(120, 1, 60, 8, 8, 64, "f16", "f16", 16), (40, 3), 2),
    (many(260, 1, 70, 16, 8, 128, "bf16", "bf16", 16), (64, 4), 1),
    (many(120, 1, 90, 20, 5, 96, "f32", "f16", 21, 30), (50, 33), 2),
    (many(300, 1, 50, 20, 5, 80, "f32", "bf16", 8), (45, 0), 1),
    (many(100, 1, 40, 8, 4, 256, "bf16", "bf16", 32), (33, 1), 2),
    (many(200, 1, 40, 8, 4, 256, "f16", "f16", 8), (100, 5), 1),
    (many(130, 5, 70, 16, 4, 128, "f16", "f16", 16), (60, 4), 2),
    (many(300, 4, 50, 8, 4, 64, "f32", "bf16", 21, 20), (30, 25), 1),
]


@pytest.mark.parametrize("case", range(len(CROWDS)))
def test_many_sequences(dev, case):
    args, win, _ = CROWDS[case]
    check(Batch(860 + case, *args, decode=max(args[0]) == 1), dev, *win)


@pytest.mark.parametrize("slide", [False, True])
@pytest.mark.parametrize("case", range(len(TILES)))
def test_tiles(dev, case, slide):
    args, win = TILES[case]
    b = Batch(800 + case, *args)
    if slide:
        b.slide(*win)
    check(b, dev, *win)


@pytest.mark.parametrize("slide", [False, True])
@pytest.mark.parametrize("case", range(len(DEALT)))
def test_dealt_units(dev, case, slide):
    args, win = DEALT[case]
    b = Batch(820 + case, *args, decode=True)
    if slide:
        b.slide(*win)
    check(b, dev, *win)


@pytest.mark.parametrize("case", range(len(CASES)))
def test_window(dev, case):
    args, win = CASES[case]
    check(Batch(300 + case, *args), dev, *win)


@pytest.mark.parametrize("case", [c for c in range(len(CASES)) if set(CASES[c][0][0]) == {1} and not CASES[c][0][10]])
def test_one_token_each(dev, case):
    args, win = CASES[case]
    check(Batch(400 + case, *args, decode=True), dev, *win)


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("case", [3, 6, 8, 9, 10])
def test_pages_behind_the_window_are_not_read(dev, case, decode):
    """Their entries are -1, and infinities and NaN stand in every row that no token sees."""
    args, (window, sinks) = CASES[case]
    b = Batch(500 + case, *args, decode=decode)
    b.slide(window, sinks)
    check(b, dev, window, sinks)


@pytest.mark.parametrize("case", [12, 13, 14, 15, 16, 18])
def test_chunks_beside_poisoned_rows(dev, case):
    args, (window, sinks) = CASES[case]
    b = Batch(600 + case, *args)
    b.slide(window, sinks)
    check(b, dev, window, sinks)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("P", [0, 70])
@pytest.mark.parametrize("n,H,HKV", [(100, 2, 1), (1000, 32, 8)])     # 16 rows to a workgroup, and tiles
def test_a_bad_row_reaches_the_tokens_that_see_it_alone(dev, bad, P, n, H, HKV):
    """One row of infinities or NaN in v: tokens whose window holds it are not finite, the others as without it."""
    S, own, at = 3, n + 60, n - 10
    W = 40 if n == 100 else 900
    b = Batch(7, [n], [own], P, H, HKV, 64, "f16", "f16", 16)
    ref = b.attention(None, W, S)
    b.vc[b.table[0, at // 16], at % 16] = bad
    cache, batch, q = b.device(dev)
    got = O.f64(serve.attention(cache, batch, q, window=W, sinks=S))
    i = own - n + np.arange(n)
    sees = (at <= i) & (at > i - W)
    assert sees.any() and not sees.all()
    assert (~np.isfinite(got[sees])).all()
    assert (np.abs(got - ref[0])[~sees] <= ref[2][~sees]).all()


def test_scales(dev):
    for s in (0.0, -0.3, 3.0):
        check(Batch(8, [1, 20], [90, 120], 30, 4, 2, 64, "f16", "f16", 16), dev, 50, 5, s)


def test_a_window_of_everything_is_the_attention_without(dev):
    """Each is within the bound of the same exact value, as their sums may be split in other places: their difference is
    within twice that."""
    for decode in (True, False):
        b = Batch(9, [1, 1, 1], [90, 1, 300], 0, 8, 2, 128, "bf16", "bf16", 16, decode=decode)
        cache, batch, q = b.device(dev)
        a, la = serve.attention(cache, batch, q, return_lse=True)
        w, lw = serve.attention(cache, batch, q, return_lse=True, window=1000)
        _, _, eo, el = b.attention(None, 1000, 0)
        assert (np.abs(O.f64(a) - O.f64(w)) <= 2 * eo).all() and (np.abs(O.f64(la) - O.f64(lw)) <= 2 * el).all()


@pytest.mark.parametrize("lens", [[2 ** 31 - 1, 5], [-3, 70], [1000, 10]])
@pytest.mark.parametrize("decode", [True, False])
def test_lengths_of_any_kind_stay_inside(dev, lens, decode):
    b = Batch(10, [1, 1], [70, 70], 40, 4, 2, 64, "f16", "f16", 16, decode=decode)
    cache, batch, q = b.device(dev)
    batch.lens.copy_(torch.tensor(lens, dtype=torch.int32))
    out = serve.attention(cache, batch, q, window=30, sinks=4)
    torch.cuda.synchronize()
    assert out.shape == q.shape


@pytest.mark.parametrize("offsets", [[0, 90, 3, 40, 60], [-5, 2 ** 31 - 1, -2 ** 31, 7, 10 ** 6], [60, 50, 40, 2, 0]])
@pytest.mark.parametrize("D,HKV,lens", [(64, 2, 200), (256, 16, 3000)])
def test_offsets_of_any_kind_stay_inside(dev, offsets, D, HKV, lens):
    """Rows of the output that they do not name stay as they were, the others are some sequence's."""
    cache = serve.PagedCache.empty(50, 64, HKV, D, torch.float16, device=dev)
    cache.v.fill_(1.0)
    table = torch.arange(50, dtype=torch.int32, device=dev).repeat(4, 1)
    batch = serve.PagedBatch(table, torch.full((4,), lens, dtype=torch.int32, device=dev),
                             q_start=torch.tensor(offsets, dtype=torch.int64).clamp(-2 ** 31, 2 ** 31 - 1).int().to(dev), n_tokens=64)
    q = torch.randn(64, 2 * HKV, D, device=dev).half()
    wide = torch.full((66, 2 * HKV, D), 7.0, dtype=torch.float16, device=dev)
    out = wide[1:65]
    serve.attention(cache, batch, q, window=2000, sinks=3, out=out)
    torch.cuda.synchronize()
    assert (wide[0] == 7.0).all() and (wide[65] == 7.0).all()
    assert ((out == 7.0) | (out == 1.0) | (out == 0.0)).all()


def test_many_sequences_of_few_tokens(dev):
    """More than a wave's search looks at in one step."""
    n = [i % 3 for i in range(700)]
    check(Batch(13, n, [i % 40 + k for i, k in enumerate(n)], 0, 4, 1, 64, "f16", "f16", 16), dev, 20, 2)


def test_pages_of_any_kind_are_absent(dev):
    b = Batch(11, [1, 30], [200, 150], 40, 4, 2, 64, "f16", "f16", 16)
    b.table[0, 11], b.table[1, 4], b.prefix_pages[0] = -5, 2 ** 31 - 1, 10 ** 6
    check(b, dev, 100, 20)


def test_a_replayed_graph_follows_the_lengths(dev):
    b = Batch(12, [1] * 4, [120, 60, 200, 90], 20, 4, 2, 64, "f16", "f16", 16, decode=True)
    cache, batch, q = b.device(dev)
    f = lambda: serve.attention(cache, batch, q, window=48, sinks=6, return_lse=True)  # noqa: E731
    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        out, lse = f()
    for lens in ([120, 60, 200, 90], [100, 1, 7, 33], [113, 59, 160, 64]):
        batch.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want, wl = f()
        assert torch.equal(out, want) and torch.equal(lse, wl)
        torch.cuda.synchronize()


@pytest.mark.parametrize("decode", [True, False])
def test_pages_beyond_32_bits(dev, decode):
    """Pages 2^30 - 8 elements apart: the third begins at byte 2^32 - 32.  The append with norms writes its rows there, the
    attention reads them, as with pages side by side."""
    far, HKV, D, page = (1 << 30) - 8, 2, 64, 16
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 17 GB")
    new = [1, 1] if decode else [20, 3]
    lens, T = [45, 9], sum(new)
    buf = [torch.empty(3 * far + 4096, dtype=torch.float16, device=dev) for _ in range(2)]
    wide = [x.as_strided((4, page, HKV, D), (far, D, page * D, 1)) for x in buf]
    near = [torch.zeros(4, HKV, page, D, dtype=torch.float16, device=dev).transpose(1, 2) for _ in range(2)]
    g = torch.Generator(device=dev).manual_seed(1)
    for a, b in zip(wide, near):
        b.copy_(torch.randn(b.shape, generator=g, device=dev))
        a.copy_(b)
    table = torch.tensor([[3, 0, 2], [1, -1, -1]], dtype=torch.int32, device=dev)   # no page is two sequences'
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    start = None if decode else torch.tensor([0, new[0], T], dtype=torch.int32, device=dev)
    x = torch.randn(T, 8, D, generator=g, device=dev).half()
    w, rope = torch.ones(D, device=dev), serve.Rope(D, device=dev)
    got = []
    for k, v in (wide, near):
        cache, batch = serve.PagedCache(k, v), serve.PagedBatch(table, n, q_start=start, n_tokens=T)
        q = serve.rope_append(cache, batch, x[:, :4], x[:, 4:6], x[:, 6:], rope=rope, q_norm=w, k_norm=w)
        got.append((serve.attention(cache, batch, q, window=30, sinks=2), k.contiguous(), v.contiguous()))
    assert all(torch.equal(a, b) for a, b in zip(*got))
