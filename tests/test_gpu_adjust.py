"""bpd_adjust_logits_gpu against a plain float64 form."""
import numpy as np
import pytest
import torch

import paged_oracle as O
from bpd_substrate_amd import serve

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def plain(x, tokens=None, lens=None, prompt=None, rep=None, freq=None, pres=None, bias=None, mask=None, mask_row=None):
    """(logits, bound) in float64: a rounding of binary32 for each operation that a token meets, of the largest that
    stands in it."""
    x = x.copy()
    B, V = x.shape
    err = np.zeros_like(x)
    for b in range(B):
        if tokens is not None:
            n = tokens.shape[1] if lens is None else min(max(int(lens[b]), 0), tokens.shape[1])
            p = 0 if prompt is None else min(max(int(prompt[b]), 0), n)
            row = tokens[b, :n]
            for t in set(int(t) for t in row if 0 <= t < V):
                r = 1.0 if rep is None else float(rep[b])
                x[b, t] = x[b, t] / r if x[b, t] > 0 else x[b, t] * r
                c = int((row[p:] == t).sum())
                err[b, t] += U * abs(x[b, t])
                if c:
                    f, s = (0.0 if z is None else float(z[b]) for z in (freq, pres))
                    top = abs(x[b, t]) + abs(f) * c + abs(s)
                    x[b, t] -= f * c + s
                    err[b, t] += 3 * U * top
        if bias is not None:
            start, word, value = bias
            last = {int(word[i]): float(value[i]) for i in range(max(int(start[b]), 0), min(int(start[b + 1]), len(word)))}
            for t, v in last.items():
                if 0 <= t < V:
                    x[b, t] += v
                    err[b, t] += U * (abs(x[b, t]) if np.isfinite(x[b, t]) else 0)
        if mask is not None:
            m = b if mask_row is None else int(mask_row[b])
            if 0 <= m < len(mask):
                bits = np.unpackbits(np.ascontiguousarray(mask[m]).view(np.uint8), bitorder="little")[:V]
                x[b, bits == 0] = -np.inf
                err[b, bits == 0] = 0
    return x, err


def make(seed, B, V, dtype, hist=0, bias=0, masks=0, allow=0.5, lens=True):
    r = np.random.default_rng(seed)
    x = torch.from_numpy(3 * r.standard_normal((B, V))).to(dtype)
    k = {}
    f32 = lambda *s: r.uniform(*s).astype(np.float32)  # noqa: E731
    if hist:
        k["tokens"] = (V * r.random((B, hist)) ** 3).astype(np.int32)
        if lens:
            k["lens"] = r.integers(0, hist + 1, B).astype(np.int32)
            k["prompt"] = np.array([r.integers(0, n + 1) for n in k["lens"]], np.int32)
        k["rep"], k["freq"], k["pres"] = f32(0.8, 1.5, B), f32(-0.5, 0.5, B), f32(0, 0.5, B)
    if bias:
        per = r.integers(0, bias + 1, B)
        start = np.concatenate([[0], np.cumsum(per)]).astype(np.int32)
        k["bias"] = (start, r.integers(0, V, start[-1]).astype(np.int32), (5 * r.standard_normal(start[-1])).astype(np.float32))
    if masks:
        N = -(-V // 32)
        bits = np.packbits(r.random((masks, N * 32)) < allow, axis=1, bitorder="little")
        k["mask"] = np.ascontiguousarray(bits).view(np.int32)
        k["mask_row"] = r.integers(-1, masks + 1, B).astype(np.int32)
    return x, k


NAMES = dict(rep="repetition", freq="frequency", pres="presence")


def device(k, dev):
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    return {NAMES.get(n, n): tuple(t(x) for x in v) if n == "bias" else t(v) for n, v in k.items()}


def check(dev, x, k, out_dtype=None, in_place=False):
    xd = x.to(dev)
    got = serve.adjust_logits(xd, **device(k, dev), out=xd if in_place else None, dtype=None if in_place else out_dtype)
    dt = out_dtype or x.dtype
    assert got.dtype is dt and (not in_place or got is xd)
    ref, err = plain(O.f64(x), **k)
    got = O.f64(got)
    inf = ~np.isfinite(ref)
    assert np.array_equal(got[inf], ref[inf], equal_nan=True)
    step = np.abs(ref[~inf]) * O.HALF_STEP[dt] + (2.0 ** -25 if dt is torch.float16 else 2.0 ** -134)
    bound = err[~inf] * (1 + O.HALF_STEP[dt]) + (step if dt is not torch.float32 else 0)
    bad = np.abs(got[~inf] - ref[~inf]) - bound
    assert bad.max(initial=-1) <= 0, bad.max()
    if not in_place:
        assert torch.equal(xd.cpu(), x)


SIZES = [(1, 1), (1, 7), (3, 33), (2, 1000), (2, 1024), (1, 8193), (5, 32001), (2, 128256), (70, 4099), (1, 1 << 22)]
TYPES = [("f32", None), ("f16", None), ("bf16", None), ("f16", "f32"), ("bf16", "f32")]


@pytest.mark.parametrize("B,V", SIZES)
@pytest.mark.parametrize("t,o", TYPES)
def test_all_rules(dev, B, V, t, o):
    x, k = make(B * V, B, V, O.DT[t], hist=300, bias=20, masks=3)
    check(dev, x, k, O.DT[o] if o else None)


@pytest.mark.parametrize("rules", [dict(hist=50), dict(hist=50, lens=False), dict(bias=9), dict(masks=2), dict(hist=5, masks=1),
                                   dict(bias=3, masks=1, allow=0.01), dict()])
@pytest.mark.parametrize("in_place", [False, True])
def test_some_rules(dev, rules, in_place):
    for t in ("f32", "bf16"):
        x, k = make(len(rules), 4, 5003, O.DT[t], **rules)
        check(dev, x, k, in_place=in_place)


def test_long_histories_of_one_token(dev):
    """100,000 times the same token, in the prompt and behind it."""
    x, k = make(1, 2, 9000, torch.float32, hist=100000, lens=False)
    k["tokens"][0], k["tokens"][1, ::2] = 8999, 4
    k["prompt"] = np.array([10, 99999], np.int32)
    check(dev, x, k)


def test_a_token_that_stands_twice_in_a_bias_list(dev):
    """The last entry counts, however many there are."""
    V = 3000
    x = torch.zeros(2, V)
    word = np.array([5, 7, 5, 9, 5, 7] + [11] * 2000 + [5], np.int32)
    value = np.arange(1, len(word) + 1).astype(np.float32)
    k = dict(bias=(np.array([0, 5, len(word)], np.int32), word, value))
    check(dev, x, k)
    check(dev, x, k, in_place=True)


def test_tokens_outside_the_vocabulary_and_offsets_outside_the_list(dev):
    x, k = make(3, 3, 2000, torch.float32, hist=40, bias=10, masks=2)
    k["tokens"][:, ::3] = np.array([-1, 2000, 2 ** 31 - 1])[:, None]
    start, word, value = k["bias"]
    word[::2] = -7
    k["bias"] = (np.array([-5, 3, 6, 2 ** 31 - 1], np.int32), word, value)
    k["mask_row"] = np.array([-2 ** 31, 1, 2 ** 31 - 1], np.int32)
    k["lens"], k["prompt"] = np.array([-3, 2 ** 31 - 1, 40], np.int32), np.array([7, 2 ** 31 - 1, -9], np.int32)
    check(dev, x, k)


def test_infinities_nan_and_masked_places(dev):
    """A masked place is -infinity whatever stood there; elsewhere infinities and NaN follow the arithmetic."""
    V = 64
    x = torch.zeros(2, V)
    x[:, 0], x[:, 1], x[:, 2] = float("nan"), float("inf"), -float("inf")
    x[:, 40], x[:, 41], x[:, 42] = float("nan"), float("inf"), -float("inf")
    mask = np.array([[-1, 0], [0, -1]], np.int32)
    tokens = np.array([[0, 1, 2, 3, 40, 41, 42]] * 2, np.int32)
    one = np.array([1.5, 1.5], np.float32)
    k = dict(tokens=tokens, rep=one, freq=one, mask=mask)
    got = serve.adjust_logits(x.to(dev), **device(k, dev)).cpu()
    for b, lo in ((0, 0), (1, 32)):
        other = 32 - lo
        assert (got[b, other:other + 32] == -float("inf")).all()
    assert torch.isnan(got[0, 0]) and got[0, 1] == float("inf") and got[0, 2] == -float("inf") and got[0, 3] == -1.5
    assert torch.isnan(got[1, 40]) and got[1, 41] == float("inf") and got[1, 42] == -float("inf")


def test_strided_rows_and_what_lies_between(dev):
    for pad_in, pad_out in ((1, 0), (3, 5), (8, 16)):
        x, k = make(5, 6, 1027, torch.float16, hist=30, bias=4, masks=2)
        wide = torch.full((6, 1027 + pad_in), 3.0, dtype=torch.float16, device=dev)
        wide[:, :1027] = x.to(dev)
        to = torch.full((6, 1027 + pad_out), 9.0, device=dev)
        serve.adjust_logits(wide[:, :1027], **device(k, dev), out=to[:, :1027])
        want = serve.adjust_logits(x.to(dev), **device(k, dev), dtype=torch.float32)
        assert torch.equal(to[:, :1027], want) and (to[:, 1027:] == 9.0).all() and (wide[:, 1027:] == 3.0).all()
        y = torch.empty(6 * 1027 + 1, dtype=torch.float16, device=dev)[1:].view(6, 1027)   # rows at no 4-byte border
        y.copy_(x)
        serve.adjust_logits(y, **device(k, dev), out=y)
        assert torch.equal(y, serve.adjust_logits(x.to(dev), **device(k, dev)))


def test_a_row_that_nothing_is_left_of_samples_nothing(dev):
    x = torch.randn(2, 500, device=dev)
    mask = torch.zeros(1, 16, dtype=torch.int32, device=dev)
    y = serve.adjust_logits(x, mask=mask, mask_row=torch.tensor([0, -1], dtype=torch.int32, device=dev))
    token, logprob, kept = serve.sample(y, torch.full((2,), 0.5, device=dev))
    assert token[0] == -1 and torch.isnan(logprob[0]) and kept[0] == 0 and kept[1] == 500
