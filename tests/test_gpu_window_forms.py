"""The forms of the windowed attention that need a workspace (tiles that are planned, units dealt to all waves), where
few tokens stand before many rows, against window_oracle."""
import pytest

from test_gpu_window import check
from window_oracle import Batch

pytestmark = pytest.mark.gpu


def needs_workspace(b, dev, window, sinks):
    cache, batch, q = b.device(dev)
    return batch._workspace(cache, q.dtype, q.shape[1], window, sinks) > 0


# new tokens, own rows, prefix, H, HKV, D, q, kv, page, heads_first, padding rows; window, sinks
FEW = [
    (([1], [9000], 0, 8, 2, 128, "bf16", "bf16", 64, True, 0), (8500, 4)),
    (([4], [8301], 61, 10, 2, 64, "f16", "f16", 16, False, 1), (7000, 70)),
    (([4, 0, 1], [6300, 20, 700], 0, 12, 4, 96, "f32", "f16", 21, False, 0), (5000, 3)),
    (([2, 3], [40, 4600], 100, 6, 2, 256, "bf16", "bf16", 32, True, 0), (4100, 0)),
    (([1, 1], [7000, 6999], 0, 4, 2, 80, "f32", "bf16", 16, True, 2), (2 ** 31 - 1, 0)),
]


@pytest.mark.parametrize("slide", [False, True])
@pytest.mark.parametrize("case", range(len(FEW)))
def test_few_tokens_before_many_rows(dev, case, slide):
    args, win = FEW[case]
    b = Batch(900 + case, *args)
    if slide:
        b.slide(*win)
    assert needs_workspace(b, dev, *win)
    check(b, dev, *win)


# one token each, of sequences of which one is long: its units go to all waves
LONG = [
    (([1] * 17, [30] * 9 + [4800] + [1, 2, 64, 0, 700, 33, 32], 0, 16, 8, 128, "bf16", "bf16", 64, True, 0), (4500, 4)),
    (([1] * 65, [40] * 64 + [4300], 50, 4, 2, 64, "f32", "f16", 16, False, 0), (4200, 60)),
    (([1] * 65, [4700] + [3] * 64, 0, 4, 2, 256, "f16", "f16", 32, True, 0), (2 ** 31 - 1, 0)),
]


@pytest.mark.parametrize("slide", [False, True])
@pytest.mark.parametrize("case", range(len(LONG)))
def test_one_long_sequence_among_many(dev, case, slide):
    args, win = LONG[case]
    b = Batch(920 + case, *args, decode=True)
    if slide:
        b.slide(*win)
    assert needs_workspace(b, dev, *win)
    check(b, dev, *win)
