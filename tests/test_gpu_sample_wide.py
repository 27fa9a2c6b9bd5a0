"""bpd_sample_gpu on rows of more than 2^19 logits, up to the largest vocab, against the definition in float64."""
import math

import numpy as np
import pytest
import torch

import paged_oracle as O
from bpd_substrate_amd import serve

pytestmark = pytest.mark.gpu


def check_row(x, token, logprob, kept, u, t=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Weights are multiples of s = 2^-(62 - bits) of the largest, bits = ceil(log2 V), each off by s / 2 and by 2^-50
    of itself: a cumulated sum over V of them by V s / 2 + 2^-50 of the sum, which is how far a border may lie."""
    x = np.asarray(x, np.float64)
    V = len(x)
    if not t > 0:
        assert (token, kept, logprob) == (int(x.argmax()), 1, 0.0)
        return
    order = np.argsort(-x, kind="stable")
    w = np.exp((x[order] - x[order[0]]) / t)
    s = 2.0 ** -(62 - math.ceil(math.log2(V)))
    slack = V * s / 2 + 2.0 ** -50 * w.sum()
    lo = hi = top_k if 0 < top_k < V else V
    if top_p < 1:
        c = np.cumsum(w[:lo])
        need = top_p * c[-1]
        lo, hi = (min(hi, int(np.searchsorted(c, need + d)) + 1) for d in (-slack, slack))
    if min_p > 0:
        near = (3 * -math.log(min_p) + 4) * 2.0 ** -53
        lo, hi = (min(n, int((w >= min_p * (1 + d)).sum())) for n, d in ((lo, near), (hi, -near)))
    assert lo <= kept <= hi, (kept, lo, hi)
    y = np.zeros(V)
    y[order[:kept]] = w[:kept]
    c = np.cumsum(y)
    at = u * c[-1]
    assert y[token] > 0 and c[token] - y[token] <= at + slack and at <= c[token] + slack, (token, at, c[token])
    want = math.log(y[token] / c[-1])
    assert abs(logprob - want) <= s / y[token] + slack / c[-1] + 2.0 ** -24 * abs(want) + 2.0 ** -50, (logprob, want)


def rows(seed, B, V, dtype):
    """Wide rows whose largest logits stand at the end, in the middle, at the start, or everywhere."""
    r = np.random.default_rng(seed)
    x = r.standard_normal((B, V)).astype(np.float32) * 2
    for b in range(B):
        at = [slice(V - 6, V), slice(V * 5 // 8, V * 5 // 8 + 6), slice(0, 6), slice(0, 0)][b % 4]
        x[b, at] += 22
    return torch.from_numpy(x).to(dtype)


@pytest.mark.parametrize("V", [(1 << 19) + 1, (1 << 20) + 3, 1 << 22])
@pytest.mark.parametrize("B", [1, 4])
@pytest.mark.parametrize("f", [{}, {"top_p": 0.9}, {"min_p": 0.02}, {"top_p": 0.95, "min_p": 0.001}, {"top_k": 40},
                               {"t": 0.0}])
def test_wide_rows(dev, V, B, f):
    dtype = torch.float16 if V == (1 << 20) + 3 else torch.float32
    x = rows(V + B, B, V, dtype)
    u = torch.linspace(0.13, 0.97, B)
    full = lambda v, dt=torch.float32: torch.full((B,), v, dtype=dt, device=dev)  # noqa: E731
    got = serve.sample(x.to(dev), u.to(dev), temperature=full(f["t"]) if "t" in f else None,
                       top_k=full(f["top_k"], torch.int32) if "top_k" in f else None,
                       top_p=full(f["top_p"]) if "top_p" in f else None,
                       min_p=full(f["min_p"]) if "min_p" in f else None)
    tok, lp, kept = (a.cpu().numpy() for a in got)
    f = {k: float(np.float32(v)) if k in ("top_p", "min_p") else v for k, v in f.items()}
    for b in range(B):
        check_row(O.f64(x[b]), int(tok[b]), float(lp[b]), int(kept[b]), float(u[b]), **f)
