"""Refusals of include/bpdq_serve.h and bpd_substrate_amd.serve (no kernel is launched; no GPU)."""
import ctypes

import pytest
import torch

from bpd_substrate_amd import _native, gpu, serve

E = gpu.BpdqError


@pytest.fixture
def L():
    lib = _native.load_hip()
    lib.bpd_gpu_last_error()
    return lib


def err(L, code, text):
    assert L.bpd_gpu_last_error() == code, L.bpd_gpu_last_error_message()
    assert text in L.bpd_gpu_last_error_message().decode()


def cache(**kw):
    d = dict(k=0x10000, v=0x20000, type=1, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64, page_stride=2048,
             row_stride=64, head_stride=1024)
    return serve._Cache(**{**d, **kw})


def batch(**kw):
    d = dict(table=0x1000, table_stride=3, table_width=3, lens=0x2000, q_start=None, n_seqs=2, n_tokens=2, prefix=None,
             prefix_len=0)
    return serve._Batch(**{**d, **kw})


CACHE = [(dict(type=0), 2, "neither f16 nor bf16"), (dict(page_size=0), 2, "page_size"), (dict(n_pages=-1), 2, "n_pages"),
         (dict(head_dim=264), 2, "head_dim"), (dict(head_dim=12), 2, "head_dim"), (dict(head_dim=0), 2, "head_dim"),
         (dict(n_kv_heads=0), 2, "n_kv_heads"), (dict(row_stride=60), 3, "multiple of 8"), (dict(page_stride=-8), 2, "stride"),
         (dict(k=None), 1, "cache.k is NULL"), (dict(v=0x20008), 3, "cache.v is not 16-byte")]
BATCH = [(dict(n_seqs=-1), 2, "n_seqs"), (dict(n_tokens=3), 2, "without q_start"), (dict(table_stride=2), 2, "table_stride"),
         (dict(prefix_len=-1), 2, "prefix_len"), (dict(prefix_len=5), 1, "batch.prefix is NULL"), (dict(lens=None), 1, "lens"),
         (dict(table=0x1002), 3, "table"), (dict(table_width=1 << 28, table_stride=1 << 28), 2, "2^31"),
         (dict(n_tokens=-2), 2, "n_tokens"), (dict(q_start=0x2002), 3, "q_start")]


def attn(L, c, b, **kw):
    d = dict(q=0x30000, qs=256, out=0x40000, os=256, lse=None, type=1, H=4, ws=0x50000, n=1 << 40)
    d = {**d, **kw}
    a = lambda x: None if x is None else ctypes.addressof(x)  # noqa: E731
    L.bpd_attn_paged_gpu(a(c), a(b), d["q"], d["qs"], d["out"], d["os"], d["lse"], d["type"], d["H"], 0.1, d["ws"], d["n"])


def append(L, c, b, rope=None, **kw):
    d = dict(pos=None, q=0x30000, qs=256, k=0x60000, ks=128, v=0x70000, vs=128, out=0x40000, os=256, type=0, H=4)
    d = {**d, **kw}
    L.bpd_rope_append_paged_gpu(ctypes.addressof(c), ctypes.addressof(b), None if rope is None else ctypes.addressof(rope),
                                d["pos"], d["q"], d["qs"], d["k"], d["ks"], d["v"], d["vs"], d["out"], d["os"], d["type"],
                                d["H"])


@pytest.mark.parametrize("f", [attn, append])
def test_cache_and_batch_refusals(L, f):
    for kw, code, text in CACHE:
        f(L, cache(**kw), batch())
        err(L, code, text)
    for kw, code, text in BATCH:
        f(L, cache(), batch(**kw))
        err(L, code, text)
    attn(L, None, batch())
    err(L, 1, "cache is NULL")
    attn(L, cache(), None)
    err(L, 1, "batch is NULL")


def test_attention_refusals(L):
    for kw, code, text in ((dict(type=2), 2, "q_type"), (dict(H=3), 2, "n_heads"), (dict(H=0), 2, "n_heads"),
                           (dict(q=None), 1, "q is NULL"), (dict(out=0x40008), 3, "out is not 16-byte"),
                           (dict(qs=248), 2, "q_stride is shorter"), (dict(os=260), 3, "out_stride"),
                           (dict(lse=0x42), 3, "lse"), (dict(n=0), 2, "ws_bytes"), (dict(ws=0x50008), 3, "ws"),
                           (dict(H=1 << 17), 7, "n_heads is above"), (dict(out=0x30000), 2, "q and out overlap"),
                           (dict(out=0x30000 + 1008), 2, "overlap"), (dict(out=0x30000 - 1008), 2, "overlap"),
                           (dict(out=0x30000 + 512, qs=512, os=504), 2, "overlap"),
                           (dict(out=0x30000 + 496, qs=512, os=512), 2, "overlap"),
                           (dict(out=0x30000 + 528, qs=512, os=512), 2, "overlap"),
                           (dict(out=0x30000 + 512, qs=512, os=512, n=0), 2, "ws_bytes"),      # between q's rows
                           (dict(out=0x30000 + 1024, n=0), 2, "ws_bytes"), (dict(out=0x30000 - 1024, n=0), 2, "ws_bytes")):
        attn(L, cache(), batch(), **kw)
        err(L, code, text)
    assert L.bpd_attn_paged_workspace(ctypes.addressof(cache()), ctypes.addressof(batch()), 3) == -1
    err(L, 2, "n_heads")
    assert L.bpd_attn_paged_workspace(ctypes.addressof(cache()), ctypes.addressof(batch()), 4) > 0
    many = batch(n_seqs=1 << 20, n_tokens=1 << 20, table_width=1 << 20, table_stride=1 << 20)
    assert L.bpd_attn_paged_workspace(ctypes.addressof(cache()), ctypes.addressof(many), 4) == -1
    err(L, 7, "multiply to 2^31")
    for f, kw in ((attn, dict(out=0x100000000000)), (append, dict(out=0x100000000000))):
        f(L, cache(), batch(n_seqs=(1 << 23) + 1, n_tokens=(1 << 23) + 1), **kw)
        err(L, 7, "n_tokens is above 2^23")
    attn(L, cache(), batch(n_seqs=1 << 22, n_tokens=1 << 22), H=34, qs=2176, os=2176)
    err(L, 7, "heads of a kv head")
    assert L.bpd_sample_workspace(1, (1 << 22) + 1) == -1
    err(L, 7, "2^22")


def test_append_refusals(L):
    R = serve._Rope
    for rope, kw, code, text in ((None, dict(type=3), 2, "x_type"), (None, dict(v=None), 2, "one of k and v"),
                                 (None, dict(H=-1), 2, "n_heads"), (None, dict(q=0x30004), 3, "q is not"),
                                 (None, dict(ks=64), 2, "k_stride is shorter"), (None, dict(vs=130), 3, "v_stride"),
                                 (None, dict(pos=0x3), 3, "pos"), (R(None, 64, 0), {}, 1, "rope.turns"),
                                 (R(0x1000, 65, 0), {}, 2, "rot_dim"), (R(0x1000, 128, 0), {}, 2, "rot_dim"),
                                 (R(0x1000, 64, 2), {}, 2, "neox"), (R(0x1004, 64, 1), {}, 3, "rope.turns"),
                                 (None, dict(out=0x30010), 2, "q_out overlaps q"),
                                 (None, dict(out=0x30000, os=512), 2, "q_out overlaps q"),
                                 (None, dict(out=0x60000 - 1024), 2, "q_out overlaps k"),
                                 (None, dict(out=0x70000 + 512), 2, "q_out overlaps k or v")):
        append(L, cache(), batch(), rope, **kw)
        err(L, code, text)


def test_sample_refusals(L):
    def call(x=0x1000, type=0, stride=100, B=2, V=100, t=None, u=0x2000, tok=0x3000, ws=0x50000, n=1 << 40):
        L.bpd_sample_gpu(x, type, stride, B, V, t, None, None, None, u, tok, None, None, ws, n)
    for kw, code, text in ((dict(type=5), 2, "type"), (dict(B=-1), 2, "n_rows"), (dict(V=-1), 2, "vocab"),
                           (dict(stride=99), 2, "row_stride"), (dict(x=None), 1, "logits"), (dict(x=0x1002), 3, "logits"),
                           (dict(u=None), 1, "u is NULL"), (dict(tok=0x3001), 3, "token"), (dict(t=0x3), 3, "temperature"),
                           (dict(n=0), 2, "ws_bytes"), (dict(V=(1 << 22) + 1, stride=1 << 23), 7, "2^22"),
                           (dict(B=1 << 22), 7, "n_rows"), (dict(B=1 << 14, V=1 << 22, stride=1 << 22), 7, "n_rows")):
        call(**kw)
        err(L, code, text)


def test_empty_calls_are_no_ops(L):
    attn(L, cache(), batch(n_seqs=0, n_tokens=0, table=None, lens=None))
    append(L, cache(), batch(n_seqs=0, n_tokens=0, table=None, lens=None))
    append(L, cache(), batch(), q=None, H=0, k=None, v=None)
    L.bpd_sample_gpu(None, 0, 0, 0, 0, None, None, None, None, None, None, None, None, None, 0)
    assert L.bpd_gpu_last_error() == 0


# ---------------------------------------------------------------- the tensor helpers, on CPU tensors

def make(T=2, dtype=torch.float16):
    c = serve.PagedCache.empty(4, 16, 2, 64, dtype, device="cpu")
    b = serve.PagedBatch(torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32))
    return c, b, torch.zeros(T, 4, 64, dtype=dtype)


def test_cpu_tensors_are_refused():
    c, b, q = make()
    with pytest.raises(E, match="not on a GPU"):
        serve.attention(c, b, q)
    with pytest.raises(E, match="not on a GPU"):
        serve.rope_append(c, b, q, q[:, :2], q[:, :2], rope=serve.Rope(64, device="cpu"))
    with pytest.raises(E, match="not on a GPU"):
        serve.sample(torch.zeros(2, 5), torch.zeros(2))


def test_helper_refusals():
    c, b, q = make()
    k = q[:, :2]
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    for f, text in (
            (lambda: serve.attention(c, b, q.float().double()), "neither float32"),
            (lambda: serve.attention(c, b, q.bfloat16()), "neither float32"),
            (lambda: serve.attention(c, b, q[:1]), r"q is"),
            (lambda: serve.attention(c, b, q.transpose(0, 1)), r"q is"),
            (lambda: serve.attention(c, b, q.transpose(1, 2).contiguous().transpose(1, 2)), "not contiguous within"),
            (lambda: serve.attention(c, b, q[0].expand(2, 4, 64)), "overlap"),
            (lambda: serve.attention(c, b, q[:, :3]), "n_heads"),
            (lambda: serve.attention(c, b, q, out=q.float()), "out is"),
            (lambda: serve.attention(c, serve.PagedBatch(i32(2, 3), i32(2), prefix=i32(2), prefix_len=33), q), "more than its"),
            (lambda: serve.PagedBatch(i32(2, 3), i32(3)), "table has"),
            (lambda: serve.PagedBatch(i32(2, 3).long(), i32(2)), "table is"),
            (lambda: serve.PagedBatch(i32(3, 2).t(), i32(2)), "table's rows"),
            (lambda: serve.PagedBatch(i32(2, 3), i32(2), q_start=i32(2), n_tokens=2), "q_start has"),
            (lambda: serve.PagedBatch(i32(2, 3), i32(2), q_start=i32(3)), "needs n_tokens"),
            (lambda: serve.PagedBatch(i32(2, 3), i32(2), prefix_len=3), "without prefix"),
            (lambda: serve.PagedBatch(i32(2, 3), i32(4)[::2]), "not contiguous"),
            (lambda: serve.PagedCache(c.k, c.v[:2]), "differ"),
            (lambda: serve.PagedCache(c.k.float(), c.v.float()), "k is"),
            (lambda: serve.PagedCache(c.k.transpose(2, 3), c.v.transpose(2, 3)), "head_dim is not contiguous"),
            (lambda: serve.Rope(7), "rot_dim"),
            (lambda: serve.Rope(8, factors=[1.0] * 3, device="cpu"), "factors"),
            (lambda: serve.rope_append(c, b, q, k, None), "only one"),
            (lambda: serve.rope_append(c, b, None, None, None), "neither"),
            (lambda: serve.rope_append(c, b, q, k.float(), k.float()), "k is"),
            (lambda: serve.rope_append(c, b, q, k, k, pos=i32(3)), "pos has"),
            (lambda: serve.sample(torch.zeros(5), torch.zeros(2)), "dimensions"),
            (lambda: serve.sample(torch.zeros(2, 5, dtype=torch.float64), torch.zeros(2)), "logits are"),
            (lambda: serve.sample(torch.zeros(5, 2).t(), torch.zeros(2)), "rows of logits"),
            (lambda: serve.sample(torch.zeros(2, 5), torch.zeros(3)), "u is not"),
            (lambda: serve.sample(torch.zeros(2, 5), torch.zeros(2), top_k=torch.zeros(2)), "top_k is not")):
        with pytest.raises(E, match=text):
            f()
    with pytest.raises(TypeError):
        serve.PagedCache(None, None)
