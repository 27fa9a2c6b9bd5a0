"""Refusals of the page pool, the normed append, the windowed attention and the adjusted logits, in the C interface and
in bpd_substrate_amd.serve (no kernel is launched; no GPU)."""
import ctypes

import pytest
import torch

from bpd_substrate_amd import _native, gpu, serve
from test_serve_host import BATCH, CACHE, batch, cache, err, make

E = gpu.BpdqError
A = ctypes.addressof


@pytest.fixture
def L():
    lib = _native.load_hip()
    lib.bpd_gpu_last_error()
    return lib


def pool(**kw):
    d = dict(table=0x1000, table_stride=5, table_width=5, lens=0x2000, gone=0x3000, free_pages=0x4000, n_free=0x5000,
             n_rows=4, n_pages=10, page_size=16)
    return serve._Pool(**{**d, **kw})


POOL = [(dict(n_rows=-1), 2, "n_rows"), (dict(n_pages=-1), 2, "n_pages"), (dict(page_size=0), 2, "page_size"),
        (dict(table_width=-1), 2, "table_width"), (dict(table_stride=4), 2, "table_stride"),
        (dict(n_rows=(1 << 14) + 1), 7, "n_rows is above 2^14"), (dict(n_pages=1 << 28), 2, "n_pages times page_size"),
        (dict(table_width=1 << 28, table_stride=1 << 28), 2, "a table's rows"), (dict(table=None), 1, "pool.table"),
        (dict(table=0x1002), 3, "pool.table"), (dict(lens=None), 1, "pool.lens"), (dict(n_free=None), 1, "pool.n_free"),
        (dict(free_pages=0x4001), 3, "pool.free_pages"), (dict(gone=0x3002), 3, "pool.gone"), (dict(n_rows=2), 2, "n_seqs")]


def extend(L, p, **kw):
    d = dict(rows=0x6000, new=0x7000, B=3, T=20, P=0, table=0x8000, stride=5, lens=0x9000, start=0xA000, slots=0xB000,
             pos=0xC000, refused=0xD000)
    d = {**d, **kw}
    L.bpd_pages_extend_gpu(None if p is None else A(p), d["rows"], d["new"], d["B"], d["T"], d["P"], d["table"], d["stride"],
                           d["lens"], d["start"], d["slots"], d["pos"], d["refused"])


def release(L, p, **kw):
    d = {**dict(rows=0x6000, keep=0x7000, B=3, window=0, sinks=0), **kw}
    L.bpd_pages_release_gpu(None if p is None else A(p), d["rows"], d["keep"], d["B"], d["window"], d["sinks"])


@pytest.mark.parametrize("f", [extend, release])
def test_pool_refusals(L, f):
    f(L, None)
    err(L, 1, "pool is NULL")
    for kw, code, text in POOL:
        f(L, pool(**kw))
        err(L, code, text)
    f(L, pool(), rows=0x6002)
    err(L, 3, "rows")
    f(L, pool(), B=-1)
    err(L, 2, "n_seqs")
    f(L, pool(), B=0)
    assert L.bpd_gpu_last_error() == 0


def test_extend_and_release_refusals(L):
    for kw, code, text in ((dict(T=-1), 2, "n_tokens is negative"), (dict(P=-1), 2, "prefix_len"),
                           (dict(T=(1 << 23) + 1), 7, "2^23"), (dict(P=(1 << 31) - 1024), 2, "2^31 - 1024"),
                           (dict(new=None), 1, "n_new"), (dict(new=0x7001), 3, "n_new"), (dict(lens=None), 1, "lens_out"),
                           (dict(start=None), 1, "q_start"), (dict(refused=None), 1, "refused"), (dict(slots=None), 1, "slots"),
                           (dict(pos=0xC002), 3, "pos"), (dict(table=0x8002), 3, "table_out"),
                           (dict(stride=4), 2, "table_out_stride")):
        extend(L, pool(), **kw)
        err(L, code, text)
    for p, kw, code, text in ((pool(), dict(window=-1), 2, "window"), (pool(), dict(sinks=-1), 2, "sinks"),
                              (pool(gone=None), dict(window=5), 1, "pool.gone"), (pool(), dict(keep=0x7002), 3, "keep")):
        release(L, p, **kw)
        err(L, code, text)


def norm_append(L, c, b, **kw):
    d = dict(qw=0x80000, qws=0, kw=0x90000, kws=0, wt=0, eps=1e-6, pos=None, q=0x30000, qs=256, k=0x60000, ks=128, v=0x70000,
             vs=128, out=0x40000, os=256, type=1, H=4, n=0)
    d = {**d, **kw}
    L.bpd_norm_rope_append_paged_gpu(A(c), A(b), d["qw"], d["qws"], d["kw"], d["kws"], d["wt"], d["eps"], None, d["pos"],
                                     d["q"], d["qs"], d["k"], d["ks"], d["v"], d["vs"], d["out"], d["os"], d["type"], d["H"])


def window(L, c, b, **kw):
    d = dict(q=0x30000, qs=256, out=0x40000, os=256, lse=None, type=1, H=4, W=10, S=2, ws=0x50000, n=1 << 40, pos=None)
    d = {**d, **kw}
    L.bpd_attn_window_paged_gpu(A(c), A(b), d["q"], d["qs"], d["out"], d["os"], d["lse"], d["type"], d["H"], 0.1, d["W"],
                                d["S"], d["ws"], d["n"])


@pytest.mark.parametrize("f", [norm_append, window])
def test_cache_and_batch_refusals(L, f):
    for kw, code, text in CACHE:
        f(L, cache(**kw), batch())
        err(L, code, text)
    for kw, code, text in BATCH:
        f(L, cache(), batch(**kw))
        err(L, code, text)


def test_norm_refusals(L):
    for kw, code, text in ((dict(wt=2), 2, "w_type"), (dict(wt=7), 2, "w_type"), (dict(eps=-1e-6), 2, "eps"),
                           (dict(eps=float("nan")), 2, "eps"), (dict(qws=8), 2, "q_norm_stride"), (dict(kws=-64), 2, "k_norm_stride"),
                           (dict(qws=68), 3, "q_norm_stride"), (dict(kws=1 << 30), 2, "k_norm_stride"),
                           (dict(qw=0x80004), 3, "q_norm"), (dict(kw=0x90008), 3, "k_norm"), (dict(q=0x30004), 3, "q is not"),
                           (dict(type=3), 2, "x_type"), (dict(out=0x30010), 2, "q_out overlaps q"), (dict(pos=0x3), 3, "pos"),
                           (dict(v=None), 2, "one of k and v")):
        norm_append(L, cache(), batch(), **kw)
        err(L, code, text)
    norm_append(L, cache(), batch(n_seqs=0, n_tokens=0, table=None, lens=None))
    assert L.bpd_gpu_last_error() == 0


def test_window_refusals(L):
    for kw, code, text in ((dict(W=0), 2, "window"), (dict(W=-5), 2, "window"), (dict(S=-1), 2, "sinks"), (dict(type=2), 2, "q_type"),
                           (dict(H=3), 2, "n_heads"), (dict(q=None), 1, "q is NULL"), (dict(out=0x30000), 2, "overlap"),
                           (dict(lse=0x42), 3, "lse"), (dict(H=1 << 17), 7, "n_heads is above")):
        window(L, cache(), batch(), **kw)
        err(L, code, text)
    chunk = batch(q_start=0x8000, n_tokens=4000, table_width=1000, table_stride=1000)
    far = dict(out=0x40000000, W=9000)
    window(L, cache(), chunk, n=0, **far)
    err(L, 2, "ws_bytes")
    window(L, cache(), chunk, ws=0x50008, **far)
    err(L, 3, "ws")
    need = lambda c, b, t=1, W=10, S=2, H=4: L.bpd_attn_window_paged_workspace(A(c), A(b), t, H, W, S)  # noqa: E731
    assert need(cache(), batch()) == 0 and need(cache(), batch(q_start=0x8000, n_tokens=50)) == 0
    assert need(cache(), chunk, W=9000) > 0
    wide = batch(table_width=1000, table_stride=1000)                         # few sequences, many rows: two launches
    assert need(cache(), wide, W=10) == 0 and need(cache(), wide, W=9000) > 0
    for a in (dict(W=0), dict(S=-1), dict(t=2), dict(H=3)):
        assert need(cache(), batch(), **a) == -1
        assert L.bpd_gpu_last_error() == 2


def adjust(L, r, **kw):
    d = {**dict(x=0x10000, type=1, xs=100, out=0x20000, ot=1, os=100, B=2, V=100), **kw}
    L.bpd_adjust_logits_gpu(d["x"], d["type"], d["xs"], d["out"], d["ot"], d["os"], d["B"], d["V"], None if r is None else A(r))


def rules(**kw):
    d = dict(tokens=0x1000, token_stride=9, token_width=9, lens=0x2000, prompt=0x3000, repetition=0x4000, frequency=0x5000,
             presence=0x6000, bias_start=0x7000, bias_token=0x8000, bias_value=0x9000, n_bias=5, mask=0xA000, mask_stride=4,
             n_masks=2, mask_row=0xB000)
    return serve._Rules(**{**d, **kw})


def test_adjust_refusals(L):
    adjust(L, None)
    err(L, 1, "rules is NULL")
    for kw, code, text in ((dict(type=3), 2, "type"), (dict(ot=2), 2, "out_type"), (dict(B=-1), 2, "n_rows"), (dict(V=-1), 2, "vocab"),
                           (dict(xs=99), 2, "row_stride"), (dict(os=99), 2, "out_stride"), (dict(x=None), 1, "logits"),
                           (dict(x=0x10001), 3, "logits"), (dict(out=None), 1, "out"), (dict(out=0x20001), 3, "out"),
                           (dict(V=(1 << 22) + 1, xs=1 << 23, os=1 << 23), 7, "2^22"), (dict(B=1 << 22), 7, "n_rows"),
                           (dict(B=1 << 20, V=32767, xs=32767, os=32767), 7, "n_rows"),
                           (dict(out=0x10000 + 200), 2, "overlaps"), (dict(out=0x10000, ot=0), 2, "overlaps"),
                           (dict(out=0x10000, xs=200), 2, "overlaps")):
        adjust(L, rules(), **kw)
        err(L, code, text)
    for kw, code, text in ((dict(token_width=-1), 2, "token_width"), (dict(token_stride=8), 2, "token_stride"),
                           (dict(n_bias=-1), 2, "n_bias"), (dict(n_masks=-1), 2, "n_masks"), (dict(mask_stride=3), 2, "mask_stride"),
                           *((dict([(n, 0x1002)]), 3, n) for n in ("tokens", "lens", "prompt", "repetition", "frequency", "presence",
                                                                   "bias_start", "bias_token", "bias_value", "mask", "mask_row")),
                           (dict(bias_token=None), 1, "bias_token"), (dict(bias_value=None), 1, "bias_value")):
        adjust(L, rules(**kw))
        err(L, code, text)
    adjust(L, rules(), B=0)
    adjust(L, rules(), V=0, xs=0, os=0)
    assert L.bpd_gpu_last_error() == 0


# ---------------------------------------------------------------- the tensor helpers, on CPU tensors

def i32(*s):
    return torch.zeros(*s, dtype=torch.int32)


def test_cpu_tensors_are_refused():
    c, b, q = make()
    p = serve.PagePool.empty(10, 16, 4, 5, device="cpu")
    w = torch.ones(64)
    for f in (lambda: serve.attention(c, b, q, window=4), lambda: p.extend(i32(2), 8), lambda: p.release(),
              lambda: serve.rope_append(c, b, q, q[:, :2], q[:, :2], q_norm=w, k_norm=w),
              lambda: serve.adjust_logits(torch.zeros(2, 5))):
        with pytest.raises(E, match="not on a GPU"):
            f()


def test_helper_refusals():
    c, b, q = make()
    k, w, f32, x = q[:, :2], torch.ones(64), torch.zeros, torch.zeros(2, 100)
    p = serve.PagePool.empty(10, 16, 4, 5, windowed=True, device="cpu")
    plain = serve.PagePool.empty(10, 16, 4, 5, device="cpu")
    pool_of = lambda **kw: serve.PagePool(**{**dict(table=i32(4, 5), lens=i32(4), free=i32(10), n_free=i32(2), page_size=16), **kw})  # noqa: E731
    for f, text in (
            (lambda: serve.attention(c, b, q, window=0), "window is below 1"),
            (lambda: serve.attention(c, b, q, window=4, sinks=-1), "sinks is negative"),
            (lambda: serve.attention(c, b, q, sinks=3), "sinks without a window"),
            (lambda: serve.rope_append(c, b, q, k, k, q_norm=torch.ones(63)), "q_norm is not a contiguous"),
            (lambda: serve.rope_append(c, b, q, k, k, k_norm=torch.ones(4, 64)), "k_norm is not a contiguous"),
            (lambda: serve.rope_append(c, b, q, k, k, q_norm=torch.ones(128)[::2]), "q_norm is not a contiguous"),
            (lambda: serve.rope_append(c, b, q, k, k, q_norm=w.bfloat16()), "q_norm is"),
            (lambda: serve.rope_append(c, b, q, k, k, q_norm=w, k_norm=w.half()), "and k_norm"),
            (lambda: pool_of(table=i32(4, 5).long()), "table is"),
            (lambda: pool_of(table=i32(5, 4).t()), "table's rows"),
            (lambda: pool_of(lens=i32(3)), "lens is"),
            (lambda: pool_of(n_free=i32(1)), "n_free is"),
            (lambda: pool_of(gone=i32(4)), "gone has"),
            (lambda: pool_of(gone=i32(4, 3)), "gone is"),
            (lambda: pool_of(free=i32(20)[::2]), "free is not contiguous"),
            (lambda: serve.PagePool.empty(10, 16, 4, 5, reserved=11, device="cpu"), "reserved"),
            (lambda: p.extend(None, 4), "new is None"),
            (lambda: p.extend(i32(2), -1), "n_tokens is negative"),
            (lambda: p.extend(i32(2), 4, rows=i32(3)), "new has 2 values and rows 3"),
            (lambda: p.extend(i32(2).long(), 4), "new is"),
            (lambda: p.release(window=0), "window 0 is below 1"),
            (lambda: p.release(window=3, sinks=-1), "negative"),
            (lambda: plain.release(window=3), "without gone"),
            (lambda: p.release(i32(2), rows=i32(3)), "keep has 2 values"),
            (lambda: serve.adjust_logits(x.double()), "logits are"),
            (lambda: serve.adjust_logits(x[0]), "dimensions"),
            (lambda: serve.adjust_logits(torch.zeros(100, 2).t()), "rows of logits"),
            (lambda: serve.adjust_logits(x, dtype=torch.float16), "dtype is"),
            (lambda: serve.adjust_logits(x, out=x.half()), "out is"),
            (lambda: serve.adjust_logits(x, out=torch.zeros(2, 99)), "out is"),
            (lambda: serve.adjust_logits(x, lens=i32(2)), "without tokens"),
            (lambda: serve.adjust_logits(x, presence=f32(2)), "penalties without tokens"),
            (lambda: serve.adjust_logits(x, mask_row=i32(2)), "mask_row without mask"),
            (lambda: serve.adjust_logits(x, tokens=i32(3, 4)), "tokens has 3 rows"),
            (lambda: serve.adjust_logits(x, tokens=i32(2, 4).long()), "tokens is"),
            (lambda: serve.adjust_logits(x, tokens=i32(4, 2).t()), "rows of tokens"),
            (lambda: serve.adjust_logits(x, tokens=i32(2, 4), lens=i32(3)), "lens is not"),
            (lambda: serve.adjust_logits(x, tokens=i32(2, 4), repetition=f32(2).half()), "repetition is not"),
            (lambda: serve.adjust_logits(x, mask=i32(2, 3)), "mask has 3 words"),
            (lambda: serve.adjust_logits(x, mask=i32(2, 4), mask_row=i32(2).long()), "mask_row is not"),
            (lambda: serve.adjust_logits(x, bias=(i32(2), i32(4), f32(4))), "bias has"),
            (lambda: serve.adjust_logits(x, bias=(i32(3), i32(4), f32(5))), "bias has"),
            (lambda: serve.adjust_logits(x, bias=(i32(3), i32(4), i32(4))), "bias's value is")):
        with pytest.raises(E, match=text):
            f()
