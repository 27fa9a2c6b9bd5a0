"""Filters of bpd_sample_gpu beyond their usual range."""
import pytest
import torch

from bpd_substrate_amd import serve

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.mark.parametrize("V", [2, 9, 3001, 5000, 32768, 32769, 60000])
@pytest.mark.parametrize("f", [{}, {"k": 10}, {"p": 0.7}, {"k": 4097}, {"k": 3, "p": 0.5, "t": 0.3}])
def test_min_p_above_1_leaves_the_first_of_the_largest(dev, V, f):
    """No weight is above 1, so the largest logit alone is left: of equal ones the first, as they rank by index.  At 1
    all that equal the largest stay."""
    x = torch.zeros(5, V)
    x[1, ::2] = -3.0                   # half of them the largest, from index 1 on
    x[2] = torch.linspace(-4, 0, V)    # one, the last
    x[3, V // 2:] = INF
    x[4, 1:] = -INF
    ties = (x == x.amax(1, keepdim=True))
    first = ties.float().argmax(1).tolist()
    u = torch.full((5,), 0.999, device=dev)
    full = lambda v, dt=torch.float32: None if v is None else torch.full((5,), v, dtype=dt, device=dev)  # noqa: E731
    for dtype in (torch.float32, torch.float16):
        for m in (2.0, 1.0 + 2.0 ** -23, INF):
            tok, lp, kept = serve.sample(x.to(dtype).to(dev), u, temperature=full(f.get("t")), min_p=full(m),
                                         top_k=full(f.get("k"), torch.int32), top_p=full(f.get("p")))
            assert kept.tolist() == [1] * 5 and lp.tolist() == [0.0] * 5
            assert tok[[0, 1, 3, 4]].tolist() == [first[i] for i in (0, 1, 3, 4)]
            assert x.to(dtype)[2, tok[2]] == x.to(dtype)[2].max() and (tok[2] == 0 or x.to(dtype)[2, tok[2] - 1] < 0)
    if not f:
        tok, _, kept = serve.sample(x.to(dev), u, min_p=full(1.0))
        assert kept.tolist() == ties.sum(1).tolist()
        assert all(ties[i, t] for i, t in enumerate(tok.tolist()))
