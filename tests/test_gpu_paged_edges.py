"""Edges of bpd_rope_append_paged_gpu and bpd_attn_paged_gpu that their other tests do not reach."""
import pytest
import torch

import paged_oracle as O
from bpd_substrate_amd import serve
from test_gpu_paged import check_attention

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- offsets beyond the tokens

@pytest.mark.parametrize("start,same", [([0, 2, 50], [0, 2, 5]), ([0, 2, 2 ** 31 - 1], [0, 2, 5]), ([0, 9, 9], [0, 5, 5]),
                                        ([-7, 2, 5], [0, 2, 5]), ([-2 ** 31, 2, 6], [0, 2, 5])])
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
