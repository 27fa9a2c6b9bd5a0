"""Sizes at which the 32-bit indexes of the paged kernels end (no kernel is launched; no GPU)."""
import ctypes

import pytest

from bpd_substrate_amd import _native
from test_serve_host import append, attn, batch, cache, err

TOP = (1 << 31) - 1024


@pytest.fixture
def L():
    lib = _native.load_hip()
    lib.bpd_gpu_last_error()
    return lib


# rows of the table (pages of one row), of the prefix and new tokens, which add up to `total`
SPLITS = [lambda total: dict(table_width=total - 1, prefix_len=0, n_seqs=1, n_tokens=1),
          lambda total: dict(table_width=3, prefix_len=total - 4, n_seqs=1, n_tokens=1),
          lambda total: dict(table_width=1 << 30, prefix_len=total - (1 << 30) - 2, n_seqs=2, n_tokens=2)]


@pytest.mark.parametrize("split", SPLITS)
@pytest.mark.parametrize("f", [attn, append])
def test_rows_whose_units_would_pass_2_31_are_refused(L, f, split):
    """A sum of rows and what rounds it up to units of 64, and the units asked for ahead, stay below 2^31."""
    c = cache(page_size=1, page_stride=64)
    for total in (TOP, TOP + 1, (1 << 31) - 65, (1 << 31) - 64, (1 << 31) - 2, (1 << 31) - 1):
        b = split(total)
        f(L, c, batch(table_stride=b["table_width"], prefix=0x8000, **b), n=0) if f is attn else \
            f(L, c, batch(table_stride=b["table_width"], prefix=0x8000, **b), pos=0x3)
        err(L, 2, "2^31 - 1024")
    b = split(TOP - 1)
    b = batch(table_stride=b["table_width"], prefix=0x8000, **b)
    if f is attn:
        f(L, c, b, n=0)
        err(L, 2, "ws_bytes")                    # all sizes were taken
        assert L.bpd_attn_paged_workspace(ctypes.addressof(c), ctypes.addressof(b), 4) > 0
    else:
        f(L, c, b, pos=0x3)
        err(L, 3, "pos")


@pytest.mark.parametrize("f", [attn, append])
def test_sequences_beyond_the_search_are_refused(L, f):
    """count_le looks through q_start's n_seqs + 1 values in 32 bits, 63 more for its rounding."""
    for n in ((1 << 30) + 1, (1 << 31) - 1):
        f(L, cache(), batch(n_seqs=n, q_start=0x9000, n_tokens=5))
        err(L, 7, "n_seqs is above 2^30")
