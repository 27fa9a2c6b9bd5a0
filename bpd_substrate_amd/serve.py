"""Serving many sequences at once: the operators of include/bpdq_serve.h on torch tensors.

    cache = serve.PagedCache.empty(n_pages, 64, n_kv_heads, head_dim, torch.float16, device="cuda")
    rope  = serve.Rope(head_dim, base=10000.0, device="cuda")
    batch = serve.PagedBatch(table, lens, prefix=system_prompt_pages, prefix_len=8192)
    q     = serve.rope_append(cache, batch, q, k, v, rope=rope)     # every layer of a step
    out   = serve.attention(cache, batch, q)
    token, logprob, kept = serve.sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)

PagedCache, PagedBatch and Rope describe tensors that the program owns: page tables,
lengths and offsets stay on the device and may be changed in place between calls (and between
the replays of a captured graph), their shapes may not.

Calls launch on torch's current stream of the tensors' device and do not wait.  Arguments
that the kernels cannot take raise gpu.BpdqError before anything is launched.  A call's
workspace comes from torch's allocator, so calls on several streams, from several threads and
in several captured graphs do not share one.
"""
import ctypes
import functools
import math

import torch

from . import gpu
from .gpu import BPDQ_ERR_SHAPE, BpdqError

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # BPD_T_*


class _Cache(ctypes.Structure):    # bpd_paged_cache
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("type", ctypes.c_int), ("n_pages", ctypes.c_int),
                ("page_size", ctypes.c_int), ("n_kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("page_stride", ctypes.c_int64), ("row_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class _Batch(ctypes.Structure):    # bpd_paged_batch
    _fields_ = [("table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("table_width", ctypes.c_int),
                ("lens", ctypes.c_void_p), ("q_start", ctypes.c_void_p), ("n_seqs", ctypes.c_int),
                ("n_tokens", ctypes.c_int), ("prefix", ctypes.c_void_p), ("prefix_len", ctypes.c_int)]


class _Rope(ctypes.Structure):     # bpd_rope
    _fields_ = [("turns", ctypes.c_void_p), ("rot_dim", ctypes.c_int), ("neox", ctypes.c_int)]


def _bad(what):
    raise BpdqError(BPDQ_ERR_SHAPE, what)


def _tensor(t, what, dtypes, ndim, device=None, contiguous=False):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} is no tensor")
    if t.dtype not in dtypes:
        _bad(f"{what} is {t.dtype}, not {' or '.join(str(d) for d in dtypes)}")
    if t.dim() != ndim:
        _bad(f"{what} has {t.dim()} dimensions, not {ndim}")
    if device is not None and t.device != device:
        _bad(f"{what} is on {t.device}, not on {device}")
    if contiguous and not t.is_contiguous():
        _bad(f"{what} is not contiguous")
    return t


def _rows(t, what, shape, dtype, device):
    """A tensor [tokens][heads][head_dim] whose tokens may stand apart; its token stride."""
    if t.dtype is not dtype or t.device != device or t.shape != shape:
        _bad(f"{what} is {t.dtype} {list(t.shape)} on {t.device}, not {dtype} {list(shape)} on {device}")
    n, h, d = shape
    s = t.stride()
    if (h > 1 and s[1] != d) or (d > 1 and s[2] != 1) or (n > 1 and s[0] < h * d):
        _bad(f"{what}'s heads are not contiguous within a token, or its tokens overlap")
    return s[0] if n > 1 else h * d


def _launch(device, fn, *args):
    """fn(stream, *args), an entry point of the library, with torch's current stream of `device`.  The stream goes
    with the call: bpd_gpu_set_stream()'s is one for the process, and other threads may choose it in between."""
    if device.type != "cuda":
        _bad(f"{fn.__name__}: the tensors are on {device}, not on a GPU")
    index = device.index
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return _launch(device, fn, *args)
    fn(torch._C._cuda_getCurrentRawStream(index), *args)
    gpu.check()


class PagedCache:
    """K/V pages that sequences share: k, v [n_pages, page_size, n_kv_heads, head_dim], float16 or
    bfloat16, of one layout with contiguous heads of head_dim elements.  Any strides of the
    other dimensions (multiples of 8 elements) will do; pages that hold each head's rows
    together, as empty() lays them out, are read fastest."""

    def __init__(self, k, v):
        for t, what in ((k, "k"), (v, "v")):
            _tensor(t, what, (torch.float16, torch.bfloat16), 4)
        if k.shape != v.shape or k.dtype != v.dtype or k.device != v.device or k.stride() != v.stride():
            _bad("k and v differ in shape, type, device or strides")
        if k.shape[3] > 1 and k.stride(3) != 1:
            _bad("head_dim is not contiguous")
        self.k, self.v, self.dtype, self.device = k, v, k.dtype, k.device
        self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = k.shape
        s = [0 if n == 1 else st for n, st in zip(k.shape, k.stride())]   # of one page, row or head: never used
        self.c = _Cache(k.data_ptr(), v.data_ptr(), TYPES[k.dtype], *k.shape, s[0], s[1], s[2])
        self._p = ctypes.addressof(self.c)

    @classmethod
    def empty(cls, n_pages, page_size, n_kv_heads, head_dim, dtype=torch.float16, device="cuda"):
        def make():
            return torch.zeros(n_pages, n_kv_heads, page_size, head_dim, dtype=dtype, device=device).transpose(1, 2)
        return cls(make(), make())


class PagedBatch:
    """The sequences of a call and their new tokens (bpd_paged_batch).

    table      int32 [n_seqs, width]: pages of each sequence's own part, in order
    lens       int32 [n_seqs]: rows of its own part, the new tokens' included
    q_start    int32 [n_seqs + 1]: first new token of each sequence; None: one each
    n_tokens   rows of q; more than q_start[n_seqs] where a batch is padded
    prefix     int32 [pages]: the pages of the prefix that all sequences share
    prefix_len its rows
    """

    def __init__(self, table, lens, q_start=None, n_tokens=None, prefix=None, prefix_len=0):
        i32 = (torch.int32,)
        _tensor(table, "table", i32, 2)
        self.device, (n, w) = table.device, table.shape
        _tensor(lens, "lens", i32, 1, self.device, contiguous=True)
        if lens.shape[0] != n:
            _bad(f"table has {n} rows and lens {lens.shape[0]}")
        if w > 1 and table.stride(1) != 1 or n > 1 and table.stride(0) < w:
            _bad("table's rows are not contiguous, or overlap")
        if q_start is not None:
            _tensor(q_start, "q_start", i32, 1, self.device, contiguous=True)
            if q_start.shape[0] != n + 1:
                _bad(f"q_start has {q_start.shape[0]} values for {n} sequences")
            if n_tokens is None:
                _bad("q_start needs n_tokens")
        if prefix is not None:
            _tensor(prefix, "prefix", i32, 1, self.device, contiguous=True)
        elif prefix_len:
            _bad("prefix_len without prefix")
        if prefix_len < 0:
            _bad("prefix_len is negative")
        self.table, self.lens, self.q_start, self.prefix = table, lens, q_start, prefix
        self.n_seqs, self.n_tokens, self.prefix_len = n, n if n_tokens is None else n_tokens, prefix_len
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.c = _Batch(p(table), table.stride(0) if n > 1 else w, w, p(lens), p(q_start), n, self.n_tokens, p(prefix),
                        prefix_len)
        self._p = ctypes.addressof(self.c)
        self._bytes = {}

    def _check(self, cache):
        if self.device != cache.device:
            _bad(f"the batch is on {self.device}, the cache on {cache.device}")
        if self.prefix_len > (0 if self.prefix is None else self.prefix.shape[0]) * cache.page_size:
            _bad(f"prefix_len {self.prefix_len} is more than its pages hold")


    def _workspace(self, cache, heads):
        """Bytes that an attention call needs, which go by shapes alone."""
        key = (heads, cache.n_kv_heads, cache.head_dim)
        n = self._bytes.get(key)
        if n is None:
            n = gpu.call("bpd_attn_paged_workspace", cache._p, self._p, heads)
            self._bytes[key] = n
        return n


class Rope:
    """Rotary positions: the first rot_dim elements of a head turn in pairs, pair j by
    position * base^(-2j / rot_dim) / factors[j] radians; pairs are neighbours, or with neox
    an element of each half.  factors as rope_freqs of DecodeModel."""

    def __init__(self, rot_dim, base=10000.0, factors=None, neox=False, device="cuda"):
        if rot_dim < 2 or rot_dim % 2:
            _bad(f"rot_dim {rot_dim} is not an even number above 0")
        f = [float(x) for x in factors] if factors is not None else [1.0] * (rot_dim // 2)
        if len(f) != rot_dim // 2:
            _bad(f"{len(f)} factors for {rot_dim // 2} pairs")
        turns = [base ** (-2.0 * j / rot_dim) / f[j] / (2.0 * math.pi) for j in range(rot_dim // 2)]
        self.rot_dim, self.neox = rot_dim, bool(neox)
        self.turns = torch.tensor(turns, dtype=torch.float64, device=device)
        self.c = _Rope(self.turns.data_ptr(), rot_dim, int(self.neox))
        self._p = ctypes.addressof(self.c)


def rope_append(cache, batch, q, k, v, rope=None, pos=None, q_out=None):
    """Rotates q [n_tokens, heads, head_dim] and k, and writes k and v [n_tokens, n_kv_heads, head_dim]
    into the new tokens' rows of the cache; returns the rotated q (q_out, which may be q itself).  Rows of a padded
    batch that belong to no sequence are left as they are in q_out; in a new tensor they are arbitrary.
    q or both of k and v may be None.  rope None: nothing rotates.  pos int32 [n_tokens]: positions
    other than prefix_len + the token's index.  Token strides of q, k and v are free, so the
    parts of a fused projection's rows will do."""
    batch._check(cache)
    T, D, dev = batch.n_tokens, cache.head_dim, cache.device
    x = q if q is not None else k
    if x is None or (k is None) != (v is None):
        _bad("neither q nor k and v, or only one of k and v")
    if x.dtype not in TYPES:
        _bad(f"q and k are {x.dtype}, not float32, float16 or bfloat16")
    H, qp, qs, op, os_ = 0, None, 0, None, 0
    if q is not None:
        if q.dim() != 3:
            _bad(f"q has {q.dim()} dimensions, not 3")
        H = q.shape[1]
        qs = _rows(q, "q", (T, H, D), x.dtype, dev)
        if q_out is None:
            q_out = torch.empty((T, H, D), dtype=x.dtype, device=dev)
        os_ = _rows(q_out, "q_out", (T, H, D), x.dtype, dev)
        qp, op = q.data_ptr(), q_out.data_ptr()
    kp = vp = None
    ks = vs = 0
    if k is not None:
        shape = (T, cache.n_kv_heads, D)
        ks, vs = _rows(k, "k", shape, x.dtype, dev), _rows(v, "v", shape, x.dtype, dev)
        kp, vp = k.data_ptr(), v.data_ptr()
    if rope is not None and rope.turns.device != dev:
        _bad(f"rope is on {rope.turns.device}, not on {dev}")
    if pos is not None:
        _tensor(pos, "pos", (torch.int32,), 1, dev, contiguous=True)
        if pos.shape[0] != T:
            _bad(f"pos has {pos.shape[0]} values for {T} tokens")
    _launch(dev, gpu._fn("bpd_rope_append_paged_on_gpu"), cache._p, batch._p, None if rope is None else rope._p,
            None if pos is None else pos.data_ptr(), qp, qs, kp, ks, vp, vs, op, os_, TYPES[x.dtype], H)
    return q_out


def attention(cache, batch, q, scale=None, out=None, return_lse=False):
    """softmax(scale q k^T) v of every new token over the prefix's rows and its sequence's own up to
    its own (bpd_attn_paged_gpu).  q [n_tokens, heads, head_dim], of the cache's type or float32, as is out.  With q of
    the cache's type the weights are rounded to it before they meet v; with a float32 q they keep 22 bits or more.
    scale: head_dim ** -0.5 unless given.  return_lse: also the float32 [n_tokens, heads] logarithm of each
    softmax's denominator.  Rows of a padded batch that belong to no sequence are left as they are
    in out; in a new tensor they are arbitrary."""
    batch._check(cache)
    if q.dim() != 3:
        _bad(f"q has {q.dim()} dimensions, not 3")
    T, H, D, dev = batch.n_tokens, q.shape[1], cache.head_dim, cache.device
    if q.dtype not in (cache.dtype, torch.float32):
        _bad(f"q is {q.dtype}, neither float32 nor the cache's {cache.dtype}")
    qs = _rows(q, "q", (T, H, D), q.dtype, dev)
    if out is None:
        out = torch.empty((T, H, D), dtype=q.dtype, device=dev)
    os_ = _rows(out, "out", (T, H, D), q.dtype, dev)
    lse = torch.empty((T, H), dtype=torch.float32, device=dev) if return_lse else None
    n = batch._workspace(cache, H)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    _launch(dev, gpu._fn("bpd_attn_paged_on_gpu"), cache._p, batch._p, q.data_ptr(), qs, out.data_ptr(), os_,
            None if lse is None else lse.data_ptr(), TYPES[q.dtype], H, D ** -0.5 if scale is None else float(scale),
            ws.data_ptr(), n)
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=256)
def _sample_workspace(rows, vocab):
    return gpu.call("bpd_sample_workspace", rows, vocab)


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """One token per row of logits [rows, vocab] from the random numbers u in [0, 1) (bpd_sample_gpu):
    (token int32, logprob float32, kept int32), each [rows].  temperature, top_p, min_p float32 and
    top_k int32, one value per row, or None."""
    if logits.dtype not in TYPES:
        _bad(f"logits are {logits.dtype}, not float32, float16 or bfloat16")
    if logits.dim() != 2:
        _bad(f"logits have {logits.dim()} dimensions, not 2")
    B, V = logits.shape
    dev = logits.device
    if V > 1 and logits.stride(1) != 1 or B > 1 and logits.stride(0) < V:
        _bad("rows of logits are not contiguous, or overlap")
    ptrs = []
    for t, what, dt in ((temperature, "temperature", torch.float32), (top_k, "top_k", torch.int32),
                        (top_p, "top_p", torch.float32), (min_p, "min_p", torch.float32), (u, "u", torch.float32)):
        if t is None and what != "u":
            ptrs.append(None)
            continue
        if t.dtype is not dt or t.shape != (B,) or t.device != dev or not t.is_contiguous():
            _bad(f"{what} is not a contiguous {dt} [{B}] on {dev}")
        ptrs.append(t.data_ptr())
    res = torch.empty((3, B), dtype=torch.int32, device=dev)
    token, logprob, kept = res[0], res[1].view(torch.float32), res[2]
    n = _sample_workspace(B, V)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    _launch(dev, gpu._fn("bpd_sample_on_gpu"), logits.data_ptr(), TYPES[logits.dtype], logits.stride(0) if B > 1 else V,
            B, V, *ptrs, token.data_ptr(), logprob.data_ptr(), kept.data_ptr(), ws.data_ptr(), n)
    return token, logprob, kept
