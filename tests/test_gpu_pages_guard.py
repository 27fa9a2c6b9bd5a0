"""The page pool's calls on pools of any content, each of its tensors and outputs between words of one buffer that have to
stay as they are."""
import ctypes

import numpy as np
import pytest
import torch

from bpd_substrate_amd import gpu, serve

pytestmark = pytest.mark.gpu

BIG = 2 ** 31 - 1
MARK = 0x5A5A5A5


class Between:
    """int32 tensors in one buffer, `gap` marked words before, between and behind them, and behind each row of a table."""

    def __init__(self, dev, gap, **shapes):
        self.at, n = {}, gap
        for name, shape in shapes.items():
            pitch = shape[-1] + gap if len(shape) == 2 and name.startswith("table") else shape[-1]
            rows = shape[0] if len(shape) == 2 else 1
            self.at[name] = (n, shape, pitch)
            n += rows * pitch + gap
        self.buf = torch.full((n,), MARK, dtype=torch.int32, device=dev)
        self.free = torch.ones(n, dtype=torch.bool, device=dev)   # words that no tensor has
        for name in shapes:
            self.of(self.free, name).fill_(False)

    def of(self, buf, name):
        n, shape, pitch = self.at[name]
        return buf.as_strided(shape, (pitch, 1) if len(shape) == 2 else (1,), n)

    def __getitem__(self, name):
        return self.of(self.buf, name)

    def check(self, what):
        torch.cuda.synchronize()
        bad = (self.free & (self.buf != MARK)).nonzero().flatten().tolist()
        assert not bad, (what, bad[:10], self.at)


R, W, N, PAGE, T = 5, 4, 6, 4, 7


def run(dev, lens, n_free, gone, free, table, new, rows, keep, gap):
    B = len(new)
    x = Between(dev, gap, table=(R, W), lens=(R,), gone=(R, 2), free=(N,), n_free=(2,), table_out=(B, W), lens_out=(B,),
                q_start=(B + 1,), slots=(T,), pos=(T,), refused=(B,))
    i32 = lambda v: torch.tensor(np.asarray(v, np.int64), dtype=torch.int32, device=dev)  # noqa: E731
    for name, v in (("table", table), ("lens", lens), ("gone", gone), ("free", free), ("n_free", [n_free, 0])):
        x[name].copy_(i32(v))
    pool = serve.PagePool(x["table"], x["lens"], x["free"], x["n_free"], PAGE, gone=x["gone"])
    new, keep, rows = i32(new), i32(keep), None if rows is None else i32(rows)
    rp = None if rows is None else rows.data_ptr()
    for tables in (True, False):
        gpu.call("bpd_pages_extend_gpu", ctypes.addressof(pool.c), rp, new.data_ptr(), B, T, 3,
                 x["table_out"].data_ptr() if tables else None, x["table_out"].stride(0), x["lens_out"].data_ptr(),
                 x["q_start"].data_ptr(), x["slots"].data_ptr(), x["pos"].data_ptr(), x["refused"].data_ptr())
        x.check("extend")
        assert 0 <= int(pool.n_free[0]) <= N and int(pool.n_free[1]) == 0
        assert -1 <= int(x["slots"].min()) and int(x["slots"].max()) < N * PAGE
        start = x["q_start"].tolist()
        assert start[0] == 0 and start == sorted(start) and start[-1] <= T
        pool.release(keep, rows=rows, window=3, sinks=1)
        x.check("release")
        pool.release(window=1)
        x.check("release by window")
        assert 0 <= int(pool.n_free[0]) <= N and int(pool.n_free[1]) == 0
        assert 0 <= int(pool.lens.min()) and int(pool.lens.max()) <= W * PAGE


CONTENT = [
    ([BIG, -5, 7, 0, 16], 99, [[3, 2], [-4, BIG], [1, 2], [0, 0], [0, 4]]),
    ([-BIG - 1, 3, BIG, 1, 15], -3, [[BIG, -1], [0, 0], [2, 1], [-BIG - 1, BIG], [3, 9]]),
    ([12, 12, 12, 12, 12], BIG, [[0, 3], [5, 9], [0, 1], [1, 3], [2, 2]]),
    ([0, 0, 0, 0, 0], 6, [[0, 0]] * 5),
]


@pytest.mark.parametrize("gap", [1, 64])
@pytest.mark.parametrize("case", range(len(CONTENT)))
def test_pools_of_any_content_stay_inside(dev, case, gap):
    lens, n_free, gone = CONTENT[case]
    for table, free in (([[BIG] * W] * R, [5, -1, BIG, 2, 0, 0]), ([[-BIG - 1, -1, 5, 6]] * R, [0, 1, 2, 3, 4, 5])):
        for new, rows, keep in (([3, 2, 1], [2, 0, 1], [1, BIG, -2]), ([BIG, 1, -7], [4, 4, -1], [BIG, 0, 5]),
                                ([7, 0, 0], [BIG, 3, 5], [0, 0, 0]), ([1, 1, 1, 1, 1], None, [16, 0, -1, BIG, 3]),
                                ([0, 16, 2], [1, 3, 3], [13, 13, 13])):
            run(dev, lens, n_free, gone, free, table, new, rows, keep, gap)
