"""bpd_rope_append_paged_gpu and bpd_attn_paged_gpu against plain float64 forms (paged_oracle)."""
import numpy as np
import pytest
import torch

import paged_oracle as O
from bpd_substrate_amd import serve

pytestmark = pytest.mark.gpu


def check_attention(b, dev, scale=None):
    cache, batch, q = b.device(dev)
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=dev)
    got, lse = serve.attention(cache, batch, q, scale=scale, out=out, return_lse=True)
    ref, rlse, eo, el = b.attention(scale)
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


# new tokens, own rows, prefix, H, HKV, D, q, kv, page, heads_first, padding rows
ATTN = [
    ([1], [1], 0, 1, 1, 8, "f16", "f16", 1, True, 0),            # one key
    ([1], [0], 0, 2, 2, 64, "f16", "f16", 16, True, 0),          # a row with nothing to see
    ([1], [0], 5, 2, 1, 64, "f32", "bf16", 16, True, 0),         # the prefix alone
    ([1, 1, 1], [300, 0, 17], 0, 8, 2, 64, "f16", "f16", 16, True, 0),
    ([1] * 5, [33, 64, 1, 129, 95], 77, 8, 8, 128, "bf16", "bf16", 16, False, 0),
    ([1] * 3, [40, 500, 7], 130, 32, 8, 128, "f32", "f16", 32, False, 0),
    ([1] * 3, [40, 500, 7], 130, 32, 8, 128, "f32", "bf16", 64, True, 0),
    ([1] * 2, [100, 31], 61, 5, 1, 80, "f16", "f16", 21, True, 0),     # odd page: ends inside every tile
    ([1] * 2, [100, 31], 61, 12, 4, 96, "f32", "f16", 3, False, 0),
    ([1] * 2, [150, 31], 200, 6, 2, 256, "bf16", "bf16", 64, True, 0),
    ([1] * 2, [150, 31], 200, 3, 3, 200, "f32", "f16", 7, True, 0),
    ([1] * 70, [9] * 70, 100, 4, 1, 64, "f16", "f16", 16, True, 0),    # many rows behind a prefix
    ([1] * 2, [70, 66], 70, 40, 1, 64, "f16", "f16", 16, True, 0),     # more than 16 heads a kv head
    ([3, 0, 20, 1], [10, 4, 20, 90], 0, 4, 2, 64, "f16", "f16", 16, True, 3),
    ([3, 0, 70, 1], [10, 0, 170, 90], 50, 8, 2, 128, "bf16", "bf16", 64, True, 2),
    ([130], [130], 33, 4, 4, 128, "f32", "f16", 16, False, 0),         # a whole prompt, causal from its start
    ([150, 9], [400, 9], 90, 4, 2, 96, "f16", "f16", 48, False, 1),
    ([5, 5], [3, 5], 0, 2, 2, 64, "f16", "f16", 16, True, 0),          # more new tokens than rows: the first see none
    ([40, 33], [45, 200], 64, 4, 2, 256, "f32", "bf16", 32, True, 0),
    ([1, 40], [45, 200], 64, 2, 2, 8, "f16", "f16", 32, True, 0),
]


@pytest.mark.parametrize("case", range(len(ATTN)))
def test_attention(dev, case):
    new, lens, P, H, HKV, D, q, kv, page, hf, pad = ATTN[case]
    check_attention(O.Batch(100 + case, new, lens, P, H, HKV, D, q, kv, page, hf, pad), dev)


@pytest.mark.parametrize("case", [1, 2, 4, 5, 9, 11, 12])
def test_attention_one_token_form(dev, case):
    new, lens, P, H, HKV, D, q, kv, page, hf, pad = ATTN[case]
    check_attention(O.Batch(100 + case, new, lens, P, H, HKV, D, q, kv, page, hf, pad, decode=True), dev)


@pytest.mark.parametrize("q,scale,sigma", [("f32", 3.0, 1.0), ("f16", -0.5, 2.0), ("f32", 0.0, 1.0), ("f16", 1e-3, 20.0)])
def test_attention_scale(dev, q, scale, sigma):
    check_attention(O.Batch(31, [1, 7], [90, 150], 64, 4, 2, 64, q, "f16", 16, sigma=sigma), dev, scale)


def test_attention_long_split(dev):
    """One long sequence and one short: the long one's keys are split over many workgroups and joined."""
    check_attention(O.Batch(41, [1, 1], [5000, 3], 3000, 4, 2, 64, "f16", "f16", 16, decode=True), dev)


def test_attention_bad_pages_are_absent(dev):
    b = O.Batch(51, [1, 2], [90, 40], 48, 4, 2, 64, "f16", "f16", 16)
    b.table[0, 1], b.table[0, 3], b.prefix_pages[1] = -7, b.kc.shape[0], 2 ** 30
    check_attention(b, dev)


def test_attention_length_beyond_table_is_clamped(dev):
    b = O.Batch(52, [1, 1], [64, 40], 0, 4, 2, 64, "f16", "f16", 16, decode=True)
    b.table = np.ascontiguousarray(b.table[:, :4])
    cache, batch, q = b.device(dev)
    want = serve.attention(cache, batch, q)
    batch.lens.copy_(torch.tensor([2 ** 30, 40], dtype=torch.int32))
    got = serve.attention(cache, batch, q)
    assert torch.equal(got, want)
    batch.lens.copy_(torch.tensor([-5, -(2 ** 31)], dtype=torch.int32))
    assert (serve.attention(cache, batch, q) == 0).all()


@pytest.mark.parametrize("q", ["f16", "f32"])
def test_attention_later_rows_with_infinities_stay_unseen(dev, q):
    """A later token's key and value may be infinite or NaN: earlier tokens of the same call do not see them."""
    b = O.Batch(53, [40], [100], 32, 4, 2, 64, q, "f16", 16)
    ref, _, eo, _ = b.attention()
    i = 61 + 20                     # the row of new token 21
    b.vc[b.table[0, i // 16], i % 16] = float("inf")
    b.kc[b.table[0, i // 16], i % 16] = float("nan")
    cache, batch, qd = b.device(dev)
    got = O.f64(serve.attention(cache, batch, qd))
    assert (np.abs(got - ref)[:21] <= eo[:21]).all()
    assert np.isnan(got[21:]).all()
    b.vc[b.table[0, i // 16], i % 16] = float("nan")
    b.kc[b.table[0, i // 16], i % 16] = 0.0
    cache, batch, qd = b.device(dev)
    got = O.f64(serve.attention(cache, batch, qd))
    assert (np.abs(got - ref)[:21] <= eo[:21]).all()
    assert np.isnan(got[21:]).all()


def test_attention_same_bits_every_time_and_in_any_company(dev):
    """A sequence's bits do not change between calls."""
    b = O.Batch(54, [1] * 9, [700, 20, 333, 1, 64, 900, 5, 5, 128], 900, 8, 2, 128, "f16", "f16", 16, decode=True)
    cache, batch, q = b.device(dev)
    first = serve.attention(cache, batch, q, return_lse=True)
    for _ in range(3):
        again = serve.attention(cache, batch, q, return_lse=True)
        assert all(torch.equal(x, y) for x, y in zip(first, again))


def test_attention_far_pages(dev):
    """Rows whose offset passes 2^31 elements, and 2^32 bytes."""
    n = (1 << 31) // (64 * 64) + 3
    k = torch.empty(n, 64, 1, 64, dtype=torch.float16, device=dev)
    v = torch.empty_like(k)
    g = torch.Generator(device=dev).manual_seed(3)
    pages = [n - 1, 0, n - 2]
    for p in pages:
        k[p] = torch.randn(64, 1, 64, generator=g, device=dev).half()
        v[p] = torch.randn(64, 1, 64, generator=g, device=dev).half()
    q = torch.randn(1, 4, 64, generator=g, device=dev).half()
    table = torch.tensor([pages], dtype=torch.int32, device=dev)
    lens = torch.tensor([150], dtype=torch.int32, device=dev)
    far = serve.attention(serve.PagedCache(k, v), serve.PagedBatch(table, lens), q)
    near_k, near_v = k[pages].clone(), v[pages].clone()
    near = serve.attention(serve.PagedCache(near_k, near_v),
                           serve.PagedBatch(torch.tensor([[0, 1, 2]], dtype=torch.int32, device=dev), lens), q)
    assert torch.equal(far, near)
    rot = serve.Rope(64, device=dev)
    x = torch.randn(1, 1, 64, generator=g, device=dev)
    lens.fill_(65 + 64)
    serve.rope_append(serve.PagedCache(k, v), serve.PagedBatch(table, lens), None, x, x, rope=rot)
    assert torch.equal(v[n - 2, 0], x[0].half())


def test_attention_strided_rows_and_another_stream(dev):
    b = O.Batch(55, [1] * 4, [70, 20, 33, 1], 40, 8, 2, 64, "f16", "f16", 16, decode=True)
    cache, batch, q = b.device(dev)
    want = serve.attention(cache, batch, q)
    row = torch.zeros(4, 12, 64, dtype=q.dtype, device=dev)
    row[:, 2:10] = q
    wide = torch.full((4, 20, 64), 3.0, dtype=q.dtype, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        serve.attention(cache, batch, row[:, 2:10], out=wide[:, 5:13])
    s.synchronize()
    assert torch.equal(wide[:, 5:13], want)
    assert (wide[:, :5] == 3.0).all() and (wide[:, 13:] == 3.0).all()


def test_library_workspace_serves_callers_without_one(dev):
    from bpd_substrate_amd import gpu
    b = O.Batch(56, [1] * 4, [700, 20, 33, 1], 400, 8, 2, 64, "f16", "f16", 16, decode=True)
    cache, batch, q = b.device(dev)
    want = serve.attention(cache, batch, q)
    out = torch.zeros_like(q)
    gpu._use_torch_stream()
    gpu.call("bpd_attn_paged_gpu", cache._p, batch._p, q, 8 * 64, out, 8 * 64, None, 1, 8, 0.125, None, 0)
    assert torch.equal(out, want)


def test_empty_batches_and_a_cache_without_pages(dev):
    cache = serve.PagedCache.empty(0, 16, 2, 64, device=dev)
    t = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
    out, lse = serve.attention(cache, serve.PagedBatch(t(3, 2), t(3) + 20), torch.ones(3, 4, 64, dtype=torch.float16, device=dev),
                               return_lse=True)
    assert (out == 0).all() and (lse == -float("inf")).all()
    none = serve.PagedBatch(t(0, 2), t(0))
    assert serve.attention(cache, none, torch.ones(0, 4, 64, dtype=torch.float16, device=dev)).shape == (0, 4, 64)
    full = serve.PagedCache.empty(2, 16, 2, 64, device=dev)
    assert serve.attention(full, serve.PagedBatch(t(2, 0), t(2) + 5), torch.ones(2, 4, 64, dtype=torch.float16, device=dev)).sum() == 0
    ragged = serve.PagedBatch(t(2, 1), t(2), q_start=t(3), n_tokens=4)      # four rows of no sequence
    o = torch.full((4, 4, 64), 5.0, dtype=torch.float16, device=dev)
    serve.attention(full, ragged, torch.ones(4, 4, 64, dtype=torch.float16, device=dev), out=o)
    assert (o == 5.0).all()
    q = torch.ones(4, 4, 64, dtype=torch.float32, device=dev)
    o = torch.full((4, 4, 64), 5.0, device=dev)
    serve.rope_append(full, ragged, q, q[:, :2], q[:, :2], rope=serve.Rope(64, device=dev), q_out=o)
    assert (o == 5.0).all() and (full.k == 0).all()


@pytest.mark.parametrize("q_start", [[0, 40, 8, 60], [60, 30, 10, 0], [-5, 20, -2 ** 31, 2 ** 31 - 1], [7, 2 ** 31 - 1, 3, 5],
                                     [-2 ** 31, -2 ** 31, 60, 60], [0, 0, 0, 0]])
@pytest.mark.parametrize("P", [0, 70])
def test_offsets_that_decrease_stay_inside(dev, q_start, P):
    """Which rows such a batch writes is open; the guards around out, lse and the cache are not."""
    b = O.Batch(71, [20, 20, 20], [30, 90, 20], P, 4, 2, 64, "f16", "f16", 16)
    cache, batch, q = b.device(dev)
    batch.q_start.copy_(torch.tensor(q_start, dtype=torch.int32))
    wide = torch.full((62, 4, 64), 7.0, dtype=torch.float16, device=dev)
    bits = lambda: cache.k.contiguous().view(torch.int16).clone()  # noqa: E731
    pages, table = bits(), batch.table.clone()
    serve.attention(cache, batch, q, out=wide[1:61])
    assert (wide[0] == 7).all() and (wide[61] == 7).all() and torch.equal(bits(), pages)
    x = torch.randn(60, 2, 64, dtype=torch.float16, device=dev)
    serve.rope_append(cache, batch, q, x, x, rope=serve.Rope(64, device=dev), q_out=wide[1:61])
    assert (wide[0] == 7).all() and (wide[61] == 7).all() and torch.equal(batch.table, table)


def test_attention_own_keys_beyond_the_last_cache(dev):
    """Own keys and values of more than 256 MB, as the formula's size goes: they are read past the last-level cache."""
    check_attention(O.Batch(60, [1] * 9, [8200, 1, 8192, 8191, 33, 0, 8200, 8000, 8100], 40, 8, 8, 128, "f16", "f16", 64,
                            decode=True), dev)


def test_attention_many_heads_and_one_kv_head_of_many(dev):
    check_attention(O.Batch(57, [1, 1], [70, 3], 40, 64, 64, 64, "f16", "f16", 16, decode=True), dev)
    check_attention(O.Batch(58, [1, 1], [70, 3], 40, 16, 1, 128, "bf16", "bf16", 16, decode=True), dev)
    check_attention(O.Batch(59, [2, 1], [70, 3], 40, 130, 1, 64, "f16", "f16", 16), dev)


# ---------------------------------------------------------------- append

# new tokens, own rows, prefix, H, HKV, D, x, kv, page, heads_first, padding, rot, neox
APPEND = [
    ([1], [1], 0, 1, 1, 8, "f32", "f16", 1, True, 0, 8, False),
    ([1, 1, 1], [40, 17, 1], 100, 8, 2, 128, "f32", "f16", 16, True, 0, 128, False),
    ([5, 0, 33, 1], [40, 17, 33, 9], 7, 4, 2, 64, "bf16", "bf16", 21, False, 4, 64, True),
    ([5, 70], [5, 170], 0, 6, 3, 96, "f16", "f16", 16, True, 0, 48, True),
    ([5, 7], [5, 17], 3, 2, 1, 80, "f16", "bf16", 16, False, 0, 40, True),    # halves of 20: no whole vectors
    ([5, 7], [5, 17], 3, 2, 1, 80, "f16", "f16", 16, False, 2, 20, False),
    ([9], [9], 0, 2, 2, 256, "f32", "bf16", 8, True, 0, 256, True),
    ([9], [9], 0, 2, 2, 40, "bf16", "f16", 8, True, 0, 2, True),
]


def check_append(b, dev, rot, neox, fused, factors=None, pos=None, base=10000.0):
    cache, batch, q = b.device(dev)
    r = np.random.default_rng(9)
    H, K, D, T = b.H, b.HKV, b.D, b.T
    row = torch.from_numpy(r.standard_normal((T, H + 2 * K, D))).to(b.qt).to(dev)
    q, k, v = row[:, :H], row[:, H:H + K], row[:, H + K:]
    if not fused:
        q, k, v = (x.contiguous() for x in (q, k, v))
    before_k, before_v = cache.k.clone(), cache.v.clone()
    q_out = torch.full((T, H, D), 7.0, dtype=b.qt, device=dev)
    rope = serve.Rope(rot, base=base, factors=factors, neox=neox, device=dev)
    p = None if pos is None else torch.tensor(pos, dtype=torch.int32, device=dev)
    serve.rope_append(cache, batch, q, k, v, rope=rope, pos=p, q_out=q_out)
    kc, vc, qo = cache.k.cpu(), cache.v.cpu(), O.f64(q_out)
    ek, ev = before_k.cpu(), before_v.cpu()
    seen = np.zeros(T, bool)
    for t, s, i in b.tokens():
        seen[t] = True
        at = b.P + i if pos is None else pos[t]
        x = O.f64(q[t])
        ref = O.rope(x, at, rot, neox, base, factors)
        assert (np.abs(qo[t] - ref) <= O.rope_bound(x, rot, neox, b.qt, ref)).all(), (t, np.abs(qo[t] - ref).max())
        page = b.table[s, i // b.page] if 0 <= i < b.table.shape[1] * b.page else -1
        if not 0 <= page < kc.shape[0]:
            continue
        x = O.f64(k[t])
        ref = O.rope(x, at, rot, neox, base, factors)
        got = O.f64(kc[page, i % b.page])
        assert (np.abs(got - ref) <= O.rope_bound(x, rot, neox, b.kvt, ref)).all(), (t, np.abs(got - ref).max())
        assert torch.equal(vc[page, i % b.page], v[t].to(b.kvt).cpu())
        ek[page, i % b.page], ev[page, i % b.page] = kc[page, i % b.page], vc[page, i % b.page]
    assert (qo[~seen] == 7.0).all(), "rows of no sequence were written"
    bits = lambda x: x.contiguous().view(torch.int16)  # noqa: E731
    assert torch.equal(bits(kc), bits(ek)) and torch.equal(bits(vc), bits(ev)), "other rows of the cache changed"


@pytest.mark.parametrize("case", range(len(APPEND)))
@pytest.mark.parametrize("fused", [False, True])
def test_append(dev, case, fused):
    new, lens, P, H, HKV, D, x, kv, page, hf, pad, rot, neox = APPEND[case]
    check_append(O.Batch(200 + case, new, lens, P, H, HKV, D, x, kv, page, hf, pad), dev, rot, neox, fused)


def test_append_far_positions_and_factors(dev):
    b = O.Batch(61, [4], [20], 0, 2, 2, 64, "f32", "f16", 16)
    check_append(b, dev, 64, False, False, pos=[0, 131071, 1 << 20, 999983], base=500000.0)
    check_append(b, dev, 64, True, False, pos=[1, 2, 70000, 3], factors=np.linspace(1.0, 8.0, 32))


def test_append_absent_rows_are_not_written(dev):
    """Pages outside the cache, indexes below zero or beyond the table: q is rotated, nothing is written."""
    b = O.Batch(62, [3, 4], [50, 2], 0, 2, 2, 64, "f16", "f16", 16)     # b: two tokens before its first row
    b.table[0, 3] = b.kc.shape[0]
    check_append(b, dev, 64, False, False)
    b.table[0, 3] = -2 ** 31
    check_append(b, dev, 64, False, False)


def test_append_in_place_without_rope_and_parts(dev):
    b = O.Batch(63, [3], [20], 0, 4, 2, 64, "f32", "f16", 16)
    cache, batch, q = b.device(dev)
    rope = serve.Rope(64, device=dev)
    x = torch.randn(3, 2, 64, device=dev)
    want = serve.rope_append(cache, batch, q, None, None, rope=rope)
    kc = cache.k.clone()
    inplace = q.clone()
    assert serve.rope_append(cache, batch, inplace, x, x, rope=rope, q_out=inplace) is inplace
    assert torch.equal(inplace, want)
    assert not torch.equal(kc.view(torch.int16), cache.k.contiguous().view(torch.int16))
    assert serve.rope_append(cache, batch, None, x, x) is None
    i = torch.arange(17, 20)
    at = torch.from_numpy(b.table[0])[i // 16].long()
    assert torch.equal(cache.k[at, i % 16], x.half())


# ---------------------------------------------------------------- together

def test_decode_steps_together_in_a_graph(dev):
    """Steps of a served batch: append, attention over prefix and pages, a head, sampling; captured once and
    replayed with lengths, inputs and random numbers changed in place, eager work between; every replay
    equals the same calls made eagerly, and the attention the plain form."""
    B, H, HKV, D, P, V = 5, 8, 2, 64, 50, 1000
    lens0 = [3, 30, 15, 16, 64]
    steps = 4
    b = O.Batch(71, [1] * B, [l + steps for l in lens0], P, H, HKV, D, "f32", "f16", 16, decode=True)
    cache, batch, _ = b.device(dev)
    g = torch.Generator(device=dev).manual_seed(5)
    rope, head = serve.Rope(D, device=dev), torch.randn(H * D, V, generator=g, device=dev)
    row, u = torch.zeros(B, H + 2 * HKV, D, device=dev), torch.zeros(B, device=dev)
    t, tp = torch.full((B,), 0.8, device=dev), torch.full((B,), 0.9, device=dev)

    def step():
        q = serve.rope_append(cache, batch, row[:, :H], row[:, H:H + HKV], row[:, H + HKV:], rope=rope)
        out = serve.attention(cache, batch, q)
        logits = (out.reshape(B, 1, H * D) * head.t().reshape(1, V, H * D)).sum(-1)
        return (out, logits) + serve.sample(logits, u, temperature=t, top_p=tp)

    def feed(i):
        r = torch.Generator(device=dev).manual_seed(100 + i)
        row.copy_(torch.randn(row.shape, generator=r, device=dev))
        u.copy_(torch.rand(B, generator=r, device=dev))
        batch.lens.copy_(torch.tensor([l + i + 1 for l in lens0], dtype=torch.int32))

    feed(0)
    step()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        captured = step()
    kept = [cache.k.clone(), cache.v.clone()]
    for i in range(steps):
        feed(i)
        cache.k.copy_(kept[0]), cache.v.copy_(kept[1])
        eager = [x.clone() for x in step()]
        after = [cache.k.clone(), cache.v.clone()]
        cache.k.copy_(kept[0]), cache.v.copy_(kept[1])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(eager, captured):
            assert torch.equal(x, y), f"step {i}"
        assert torch.equal(after[0].view(torch.int16), cache.k.view(torch.int16))
        kept = after
        # the step against the plain form on the cache as it is now
        b.lens = [l + i + 1 for l in lens0]
        lay = lambda c: c.cpu().transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
        b.kc, b.vc = lay(cache.k), lay(cache.v)
        b.q = serve.rope_append(cache, batch, row[:, :H], None, None, rope=rope).cpu()
        ref, _, eo, _ = b.attention()
        assert (np.abs(O.f64(captured[0]) - ref) <= eo).all()
        for j in range(B):
            O.check_sample(O.f64(captured[1])[j], int(captured[2][j]), float(captured[3][j]), int(captured[4][j]),
                           float(u[j]), float(t[j]), top_p=float(tp[j]))


def test_two_graphs_of_one_stream_replayed_side_by_side(dev):
    """Calls captured on one stream do not share a workspace: their graphs run on two streams at once."""
    bs = [O.Batch(80 + i, [1] * 6, [900, 20, 333, 1, 64, 500], 700, 8, 2, 64, "f16", "f16", 16, decode=True)
          for i in range(2)]
    dv = [b.device(dev) for b in bs]
    want = [serve.attention(*d) for d in dv]
    cap = torch.cuda.Stream()
    graphs, outs = [], []
    torch.cuda.synchronize()
    for d in dv:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=cap):
            outs.append(serve.attention(*d))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w), rep


def test_calls_of_two_threads_on_streams_of_their_own(dev):
    import threading
    bs = [O.Batch(90 + i, [1] * 6, [900, 20, 333, 1, 64, 500], 300, 8, 2, 64, "f16", "f16", 16, decode=True)
          for i in range(2)]
    dv = [b.device(dev) for b in bs]
    want = [serve.attention(*d) for d in dv]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(50):
                got = serve.attention(*dv[i])
                st.synchronize()
                if not torch.equal(got, want[i]):
                    wrong.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not wrong
