import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
HERE = os.path.dirname(os.path.abspath(__file__))
if HERE not in sys.path:
    sys.path.insert(0, HERE)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (gfx950) GPU; runs through libbpdq_hip.so")


@pytest.fixture(scope="session")
def dev():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")
    return torch.device("cuda:0")


# Tests that capture a torch sum.  torch splits it over workgroups that count themselves in memory cleared by
# hipMemsetAsync, which becomes a memset node of the graph, and on replays after the first such nodes have left the
# counts as they were: no workgroup was the last, and the sum of the replay before stayed.  They get the same sum from
# additions alone.
SUMS_IN_GRAPHS = {"test_decode_steps_together_in_a_graph"}


@pytest.fixture(autouse=True)
def _sums_of_additions(request, monkeypatch):
    if getattr(request.node, "originalname", None) not in SUMS_IN_GRAPHS:
        return
    import torch

    plain = torch.Tensor.sum

    def by_halves(x, *args, **kw):
        if args != (-1,) or kw or not x.is_cuda:
            return plain(x, *args, **kw)
        while x.shape[-1] > 1:
            n = x.shape[-1]
            h = x[..., :n // 2] + x[..., n // 2:n // 2 * 2]
            x = h if n % 2 == 0 else torch.cat([h[..., :-1], h[..., -1:] + x[..., -1:]], -1)
        return x[..., 0]

    monkeypatch.setattr(torch.Tensor, "sum", by_halves)
