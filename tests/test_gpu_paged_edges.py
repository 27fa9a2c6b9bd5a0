"""Edges of bpd_rope_append_paged_gpu and bpd_attn_paged_gpu that their other tests do not reach."""
import numpy as np
import pytest
import torch

import paged_oracle as O
from bpd_substrate_amd import serve
from test_gpu_paged import check_attention

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


# ---------------------------------------------------------------- offsets beyond the tokens

@pytest.mark.parametrize("start,same", [([0, 2, 50], [0, 2, 5]), ([0, 2, 2 ** 31 - 1], [0, 2, 5]),
                                        ([0, 9, 9], [0, 5, 5]), ([-7, 2, 5], [0, 2, 5]), ([-2 ** 31, 2, 6], [0, 2, 5])])
@pytest.mark.parametrize("x", ["f32", "f16"])
def test_offsets_are_clamped_alike_by_append_and_attention(dev, start, same, x):
    """q_start below 0 counts as 0 and above n_tokens as n_tokens, for the row that a token's key goes to as for the
    rows that it sees."""
    got = []
    for s in (start, same):
        b = O.Batch(11, [2, 3], [10, 20], 7, 4, 2, 64, x, "f16", 16)
        cache, batch, q = b.device(dev)
        batch.q_start.copy_(torch.tensor(s, dtype=torch.int32))
        g = torch.Generator(device=dev).manual_seed(3)
        k, v = (torch.randn(5, 2, 64, generator=g, device=dev).to(q.dtype) for _ in range(2))
        before = cache.k.clone()
        r = serve.rope_append(cache, batch, q, k, v, rope=serve.Rope(64, device=dev))
        assert not torch.equal(before.view(torch.int16), cache.k.contiguous().view(torch.int16))
        out, lse = serve.attention(cache, batch, r, return_lse=True)
        got.append((cache.k.contiguous().view(torch.int16), cache.v.contiguous().view(torch.int16), r, out, lse))
    for a, b in zip(*got):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- tiny scores, queries of infinities

@pytest.mark.parametrize("kv", ["f16", "bf16"])
@pytest.mark.parametrize("decode", [False, True])
@pytest.mark.parametrize("exponent,scale", [(-110, 1e-20), (-126, 1e-38), (0, 2.0 ** -126), (-60, 2.0 ** -100)])
def test_scores_that_vanish(dev, kv, decode, exponent, scale):
    """Queries and scales so small that every score is next to 0: the mean of the values seen, none of the rows that are
    not there."""
    b = O.Batch(23, [1, 1] if decode else [1, 40], [21, 90], 70, 4, 2, 64, "f32", kv, 16, decode=decode)
    b.table[1, 2] = -1
    b.q = torch.ldexp(b.q, torch.tensor(exponent))
    check_attention(b, dev, scale)


@pytest.mark.parametrize("bad", [INF, -INF, NAN])
@pytest.mark.parametrize("q", ["f32", "f16"])
@pytest.mark.parametrize("form", ["chunks", "chunks without a prefix", "a chunk of its own tiles", "one token",
                                  "one token behind a prefix", "rows split over many workgroups"])
def test_a_query_of_infinities_that_sees_no_row(dev, bad, q, form):
    """Every page outside the cache: zeros and -infinity, whatever the query holds."""
    one = form.startswith("one")
    new, lens, P = {"chunks": ([1, 40], [20, 90], 70), "chunks without a prefix": ([1, 40], [20, 90], 0),
                    "a chunk of its own tiles": ([1, 150], [20, 190], 70), "one token": ([1, 1], [20, 90], 0),
                    "one token behind a prefix": ([1, 1], [20, 90], 70),
                    "rows split over many workgroups": ([1, 2], [20, 2500], 3000)}[form]
    b = O.Batch(21, new, lens, P, 4, 2, 64, q, "f16", 16, decode=one)
    b.table[:] = -1
    b.prefix_pages[:] = b.kc.shape[0]
    b.q[:, :, 3] = bad
    cache, batch, qd = b.device(dev)
    out, lse = serve.attention(cache, batch, qd, return_lse=True)
    assert (out == 0).all() and (lse == -INF).all()


@pytest.mark.parametrize("bad", [INF, NAN])
def test_a_query_of_infinities_leaves_the_others_alone(dev, bad):
    """Rows of one tile whose neighbour's scores are NaN, pages missing in between.  Their bits may change (the rows
    of a wave move their reference exponents together), their bounds do not."""
    b = O.Batch(22, [1, 40], [20, 90], 70, 4, 2, 64, "f16", "f16", 16)
    b.table[1, 2], b.prefix_pages[1] = -1, 2 ** 30
    cache, batch, qd = b.device(dev)
    ref, rlse, eo, el = b.attention()
    qd[5] = bad
    out, lse = (O.f64(x) for x in serve.attention(cache, batch, qd, return_lse=True))
    keep = np.arange(len(qd)) != 5
    assert (np.abs(out - ref) <= eo)[keep].all() and (np.abs(lse - rlse) <= el)[keep].all()
    assert np.isnan(out[5]).all() and np.isnan(lse[5]).all()


# ---------------------------------------------------------------- caches laid out otherwise, other sequences beside

@pytest.mark.parametrize("page", [100, 20, 4])
@pytest.mark.parametrize("q", ["f32", "f16"])
@pytest.mark.parametrize("decode", [False, True])
def test_contiguous_caches_are_pages_by_strides(dev, page, q, decode):
    """The decode step's cache, [max_seq][n_head_kv * head_dim] binary16 for each sequence: one page of a sequence,
    or one per 20 or 4 rows of it."""
    b = O.Batch(41, [1, 1, 1] if decode else [1, 9, 1], [100, 37, 1], 0, 8, 2, 64, q, "f16", 100, heads_first=False,
                decode=decode)
    rows = [c[torch.from_numpy(b.table[:, 0]).long()].reshape(3, 100, 2 * 64) for c in (b.kc, b.vc)]
    b.kc, b.vc = (c.view(3 * 100 // page, page, 2, 64) for c in rows)
    b.page, b.table = page, np.arange(3 * 100 // page, dtype=np.int32).reshape(3, -1)
    check_attention(b, dev)


@pytest.mark.parametrize("decode", [False, True])
@pytest.mark.parametrize("q", ["f32", "f16"])
def test_a_sequence_alone_and_in_company(dev, q, decode):
    """Other sequences change how one's keys are split, and with that its bits: not more than twice its bound."""
    new = [1] * 9 if decode else [1, 40, 3, 1, 90, 1, 1, 2, 1]
    b = O.Batch(42, new, [700, 120, 333, 1, 164, 900, 5, 5, 128], 300, 8, 2, 64, q, "f16", 16, decode=decode)
    cache, batch, qd = b.device(dev)
    _, _, eo, el = b.attention()
    out, lse = (O.f64(x) for x in serve.attention(cache, batch, qd, return_lse=True))
    for s in range(9):
        at = slice(int(b.start[s]), int(b.start[s + 1]))
        n = b.new[s]
        start = None if decode else torch.tensor([0, n], dtype=torch.int32, device=dev)
        one = serve.PagedBatch(batch.table[s:s + 1], batch.lens[s:s + 1], q_start=start, n_tokens=n,
                               prefix=batch.prefix, prefix_len=300)
        o, l = (O.f64(x) for x in serve.attention(cache, one, qd[at], return_lse=True))
        assert (np.abs(o - out[at]) <= 2 * eo[at]).all() and (np.abs(l - lse[at]) <= 2 * el[at]).all()
