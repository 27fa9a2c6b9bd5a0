"""Which form the windowed attention takes where few workgroups would have many rows, or one sequence most of them.
No GPU."""
import pytest

from launches import Recorder
from test_step_launches import window

TILES, DEALT, ONE = ["k_attn_plan", "k_attn_tile", "k_attn_join"], ["k_attn_wave", "k_attn_join"], ["k_attn_head"]


@pytest.fixture(scope="module")
def launched(tmp_path_factory):
    return Recorder(str(tmp_path_factory.mktemp("launches")))


def kernels(launched, new, rows, H, HKV, D, q, kv, page, decode=False, win=None):
    need, got = window(launched, (new, [rows] * len(new), 0, H, HKV, D, q, kv, page, True, 0), (win or rows - 4, 4), decode)
    names = [l.kernel for l in got]
    assert (need > 0) == (names != ONE)
    return names


@pytest.mark.parametrize("new", [[1], [4], [16]])
@pytest.mark.parametrize("shape,short", [((32, 8, 128, "bf16", "bf16", 64), 1028), ((4, 1, 128, "bf16", "bf16", 64), 1028),
                                         ((40, 8, 64, "f16", "f16", 16), 1028), ((16, 2, 256, "bf16", "bf16", 64), 516),
                                         ((32, 8, 128, "f32", "f16", 64), 1028), ((20, 5, 96, "f32", "f16", 21), 1028),
                                         ((32, 8, 128, "bf16", "bf16", 21), 1028)])
def test_a_few_tokens_of_one_sequence(launched, shape, short, new):
    """By 16 rows to a workgroup there are up to 40 of them on 256 CUs: from some thousand rows on they go to all."""
    assert kernels(launched, new, short, *shape) == ONE
    for rows in (7000, 32772, 131076):
        assert kernels(launched, new, rows, *shape) == TILES


def test_a_window_is_what_counts(launched):
    """Long sequences, of which a token sees little."""
    assert kernels(launched, [4], 131076, 32, 8, 128, "bf16", "bf16", 64, win=512) == ONE
    assert kernels(launched, [1] * 64, 131076, 32, 8, 128, "bf16", "bf16", 64, win=4096) == ONE


def test_many_sequences_of_which_one_may_be_long(launched):
    """64 sequences fill the chip, but the host does not know that they are alike."""
    for new in ([1] * 64, [2] * 64):
        assert kernels(launched, new, 8192, 32, 8, 128, "bf16", "bf16", 64) == ONE
        assert kernels(launched, new, 8196, 32, 8, 128, "bf16", "bf16", 64) == TILES


@pytest.mark.parametrize("B,shape", [(16, (32, 8, 128, "bf16", "bf16", 64)), (64, (32, 8, 128, "f16", "f16", 16)), (64, (40, 8, 64, "f16", "f16", 16)),
                                     (64, (16, 2, 256, "bf16", "bf16", 64)), (200, (8, 8, 64, "f32", "bf16", 16))])
def test_one_token_each_of_many_sequences(launched, B, shape):
    assert kernels(launched, [1] * B, 2052, *shape, decode=True) == ONE
    assert kernels(launched, [1] * B, 4096, *shape, decode=True) == ONE
    for rows in (4100, 131072):
        assert kernels(launched, [1] * B, rows, *shape, decode=True) == DEALT
    assert kernels(launched, [1] * B, 131072, *shape, decode=True, win=2048) == ONE


def test_so_many_sequences_that_one_may_be_long(launched):
    """The others keep the chip busy beside it, and tiles or dealt units would need a workspace of gigabytes."""
    for rows in (8196, 131072):
        assert kernels(launched, [1] * 65, rows, 32, 8, 128, "bf16", "bf16", 64) == ONE
        assert kernels(launched, [1] * 64, rows, 32, 8, 128, "bf16", "bf16", 64) == TILES
        assert kernels(launched, [1] * 513, rows, 32, 8, 128, "bf16", "bf16", 64, decode=True) == ONE
        assert kernels(launched, [1] * 512, rows, 32, 8, 128, "bf16", "bf16", 64, decode=True) == DEALT
