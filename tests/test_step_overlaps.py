"""Numbers that a call reads of a sequence while it writes another's length are not the pool's own lengths.  No GPU."""
import pytest
import torch

from bpd_substrate_amd import gpu, serve
from test_step_host import i32
from test_step_sizes import sent  # noqa: F401


@pytest.mark.parametrize("call", ["extend", "release"])
def test_the_pools_lengths_by_row(sent, call):  # noqa: F811
    p = serve.PagePool.empty(10, 16, 4, 5, windowed=True, device="cpu")
    f = (lambda x, rows: p.extend(x, 8, rows=rows)) if call == "extend" else (lambda x, rows: p.release(x, rows=rows))
    for x in (p.lens, p.lens[:2], p.lens[3:]):
        with pytest.raises(gpu.BpdqError, match="lies in the pool's lens"):
            f(x, i32(x.shape[0]))
    assert not sent
    f(p.lens, None)                 # a sequence's own
    f(p.lens[i32(2).long()], i32(2))   # a copy
    f(p.lens[4:], i32(0))
    state = torch.zeros(12, dtype=torch.int32)   # lengths and numbers side by side
    p = serve.PagePool(p.table, state[4:8], p.free, p.n_free, 16)
    f(state[:4], i32(4))
    f(state[8:], i32(4))
    assert len(sent) == 5
