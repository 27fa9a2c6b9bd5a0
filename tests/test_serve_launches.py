"""What the entry points of include/bpdq_serve.h launch, against what their kernels hold in LDS.  No GPU."""

import pytest

from launches import Recorder

A = 0x100000  # never read: aligned as a torch tensor is
SLICES = 256  # of a row, whose sums k_draw keeps in LDS


@pytest.fixture(scope="module")
def launched(tmp_path_factory):
    return Recorder(str(tmp_path_factory.mktemp("launches")))


def sample_launches(launched, B, V, type=0):
    none = [None] * 4
    return launched("bpd_sample_gpu", A, type, V, B, V, *none, 2 * A, 3 * A, None, None, 4 * A, 1 << 40)


def slice_of(launched, B, V):
    """(slices of a row, elements of one): the first from the grid, the second from what the workspace holds."""
    S, rest = divmod(sample_launches(launched, B, V)[0].grid[0], B)
    assert rest == 0
    n, up16 = B * S, lambda x: (x + 15) // 16 * 16
    lists = launched.lib.bpd_sample_workspace(B, V) - up16(12 * n) - up16(16 * n) - up16(24 * B) - 8192 * n
    return S, lists // (2 * n)


VOCAB = [32769, 50257, 128256, 300001, 524287, 524288, 524289, (1 << 20) - 1, 1 << 20, (1 << 20) + 3, 1 << 21,
         (1 << 21) + 1, 3 << 20, (1 << 22) - 1, 1 << 22]


@pytest.mark.parametrize("V", VOCAB)
def test_slices_of_a_row_fit_the_draw(launched, V):
    """Every slice has a place among the row's sums, and each thread of its workgroup of 512 marks its up to 32
    elements in one word."""
    for B in [*range(1, 9), 63, 64, 256, 1024]:
        S, n = slice_of(launched, B, V)
        assert S <= SLICES, (B, V, S)
        assert 2048 <= n <= 16384 and n & (n - 1) == 0 and S == -(-V // n), (B, V, S, n)


def test_rows_that_a_workgroup_holds_take_one_launch(launched):
    for V in (1, 1000, 32768):
        (one,) = sample_launches(launched, 3, V)
        assert one.kernel == "k_sample_row" and one.grid[0] == 3
    assert [l.kernel for l in sample_launches(launched, 3, 32769)] == ["k_max", "k_hist", "k_cut", "k_pick", "k_draw"]
