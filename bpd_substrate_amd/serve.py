"""Serving many sequences at once: the operators of include/bpdq_serve.h on torch tensors.

    cache = serve.PagedCache.empty(n_pages, 64, n_kv_heads, head_dim, torch.float16, device="cuda")
    rope  = serve.Rope(head_dim, base=10000.0, device="cuda")
    batch = serve.PagedBatch(table, lens, prefix=system_prompt_pages, prefix_len=8192)
    q     = serve.rope_append(cache, batch, q, k, v, rope=rope)     # every layer of a step
    out   = serve.attention(cache, batch, q)
    token, logprob, kept = serve.sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)

and around them what a serving loop does on the device from step to step:

    pool  = serve.PagePool.empty(n_pages, 64, n_rows, width, windowed=True, device="cuda")
    step  = pool.extend(new, n_tokens, rows=rows)                   # pages, tables, slots, positions
    q     = serve.rope_append(cache, step.batch(), q, k, v, rope=rope, q_norm=wq, k_norm=wk)
    out   = serve.attention(cache, step.batch(), q, window=1024, sinks=4)
    logits = serve.adjust_logits(logits, tokens=t, lens=n, repetition=r, bias=b, mask=m)
    pool.release(keep, rows=rows, window=1024, sinks=4)

PagedCache, PagedBatch, PagePool and Rope describe tensors that the program owns: page tables,
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


class _Pool(ctypes.Structure):     # bpd_page_pool
    _fields_ = [("table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("table_width", ctypes.c_int),
                ("lens", ctypes.c_void_p), ("gone", ctypes.c_void_p), ("free_pages", ctypes.c_void_p),
                ("n_free", ctypes.c_void_p), ("n_rows", ctypes.c_int), ("n_pages", ctypes.c_int),
                ("page_size", ctypes.c_int)]


class _Rules(ctypes.Structure):    # bpd_logit_rules
    _fields_ = [("tokens", ctypes.c_void_p), ("token_stride", ctypes.c_int64), ("token_width", ctypes.c_int),
                ("lens", ctypes.c_void_p), ("prompt", ctypes.c_void_p), ("repetition", ctypes.c_void_p),
                ("frequency", ctypes.c_void_p), ("presence", ctypes.c_void_p), ("bias_start", ctypes.c_void_p),
                ("bias_token", ctypes.c_void_p), ("bias_value", ctypes.c_void_p), ("n_bias", ctypes.c_int),
                ("mask", ctypes.c_void_p), ("mask_stride", ctypes.c_int64), ("n_masks", ctypes.c_int),
                ("mask_row", ctypes.c_void_p)]


def _bad(what):
    raise BpdqError(BPDQ_ERR_SHAPE, what)


_TOP = 0x7FFFFFFF   # of a C int


def _int(n, what):
    """n, which ctypes would pass on modulo 2^32."""
    if not -_TOP - 1 <= n <= _TOP:
        _bad(f"{what} {n} does not fit 32 bits")
    return n


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
        self.c = _Cache(k.data_ptr(), v.data_ptr(), TYPES[k.dtype], *(_int(n, "a dimension of the pages") for n in k.shape),
                        *s[:3])
        self._geometry = (k.shape[1:], s[1])   # what a workspace goes by
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
        self.c = _Batch(p(table), table.stride(0) if n > 1 else w, _int(w, "table's width"), p(lens), p(q_start),
                        _int(n, "n_seqs"), _int(self.n_tokens, "n_tokens"), p(prefix), _int(prefix_len, "prefix_len"))
        self._p = ctypes.addressof(self.c)
        self._bytes = {}

    def _check(self, cache):
        if self.device != cache.device:
            _bad(f"the batch is on {self.device}, the cache on {cache.device}")
        if self.prefix_len > (0 if self.prefix is None else self.prefix.shape[0]) * cache.page_size:
            _bad(f"prefix_len {self.prefix_len} is more than its pages hold")

    def _workspace(self, cache, dtype, heads, window, sinks):
        """Bytes that an attention call needs, which go by shapes alone."""
        key = (heads, cache._geometry, dtype, window, sinks)
        n = self._bytes.get(key)
        if n is None:
            if window is None:
                n = gpu.call("bpd_attn_paged_workspace", cache._p, self._p, heads)
            else:
                n = gpu.call("bpd_attn_window_paged_workspace", cache._p, self._p, TYPES[dtype], heads, window, sinks)
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


class PageStep:
    """What PagePool.extend gives: for n_seqs sequences and n_tokens new tokens, int32 on the device,

    table    [n_seqs, width]: their pages, -1 behind them (the pool's own table where rows is None)
    lens     [n_seqs]: their rows, the new ones' included
    q_start  [n_seqs + 1]: first new token of each; q_start[n_seqs] of the n_tokens are granted
    slots    [n_tokens]: every new token's row of the cache, page * page_size + row in it; -1 behind the last
    pos      [n_tokens]: its position; -1 behind the last
    refused  [n_seqs]: 0, or why a sequence got nothing: 1 no row, a row named twice or a negative number, 2 the
             table's width, 3 pages, 4 n_tokens
    """

    def __init__(self, table, lens, q_start, slots, pos, refused, n_tokens, prefix_len):
        self.table, self.lens, self.q_start, self.slots, self.pos, self.refused = table, lens, q_start, slots, pos, refused
        self.n_tokens, self.prefix_len = n_tokens, prefix_len
        self._batch = None

    def batch(self, prefix=None):
        """The PagedBatch of these sequences and tokens, behind the pages `prefix` of extend's prefix_len rows."""
        if self._batch is None or self._batch.prefix is not prefix:
            self._batch = PagedBatch(self.table, self.lens, q_start=self.q_start, n_tokens=self.n_tokens, prefix=prefix,
                                     prefix_len=self.prefix_len)
        return self._batch


class PagePool:
    """Pages that sequences take and give back on the device (bpd_page_pool).

    table    int32 [n_rows, width]: the pages of each row's sequence, -1 where there is none
    lens     int32 [n_rows]: its rows
    free     int32 [n_pages]: in its first n_free[0] places the pages that no sequence holds
    n_free   int32 [2]: their number, and a 0
    gone     int32 [n_rows, 2] or None: the pages that slid out of a window; needed to release by window
    """

    def __init__(self, table, lens, free, n_free, page_size, gone=None):
        i32 = (torch.int32,)
        _tensor(table, "table", i32, 2)
        self.device, (R, W) = table.device, table.shape
        if W > 1 and table.stride(1) != 1 or R > 1 and table.stride(0) < W:
            _bad("table's rows are not contiguous, or overlap")
        for t, what, shape in ((lens, "lens", (R,)), (free, "free", None), (n_free, "n_free", (2,)), (gone, "gone", (R, 2))):
            if t is None and what == "gone":
                continue
            _tensor(t, what, i32, 2 if what == "gone" else 1, self.device, contiguous=True)
            if shape is not None and t.shape != shape:
                _bad(f"{what} is {list(t.shape)}, not {list(shape)}")
        self.table, self.lens, self.free, self.n_free, self.gone = table, lens, free, n_free, gone
        self.n_rows, self.width, self.n_pages, self.page_size = R, W, free.shape[0], page_size
        self.c = _Pool(table.data_ptr(), table.stride(0) if R > 1 else W, _int(W, "table's width"), lens.data_ptr(),
                       None if gone is None else gone.data_ptr(), free.data_ptr(), n_free.data_ptr(), _int(R, "n_rows"),
                       _int(self.n_pages, "n_pages"), _int(page_size, "page_size"))
        self._lens = lens.data_ptr(), lens.data_ptr() + 4 * R
        self._p = ctypes.addressof(self.c)

    @classmethod
    def empty(cls, n_pages, page_size, n_rows, width, reserved=0, windowed=False, device="cuda"):
        """A pool of n_pages pages of which the first `reserved` (a prefix's) are never handed out."""
        if not 0 <= reserved <= n_pages:
            _bad(f"reserved {reserved} is not in 0..{n_pages}")
        z = lambda *s: torch.zeros(s, dtype=torch.int32, device=device)  # noqa: E731
        free, n_free = z(n_pages), z(2)
        free[:n_pages - reserved] = torch.arange(n_pages - 1, reserved - 1, -1, dtype=torch.int32, device=device)
        n_free[0] = n_pages - reserved
        return cls(z(n_rows, width) - 1, z(n_rows), free, n_free, page_size, z(n_rows, 2) if windowed else None)

    def _rows(self, rows, t, what):
        """How many sequences a call names, and where."""
        if rows is not None:
            _tensor(rows, "rows", (torch.int32,), 1, self.device, contiguous=True)
        if t is not None:
            _tensor(t, what, (torch.int32,), 1, self.device, contiguous=True)
            if rows is not None and rows.shape != t.shape:
                _bad(f"{what} has {t.shape[0]} values and rows {rows.shape[0]}")
        n = t.shape[0] if t is not None else rows.shape[0] if rows is not None else self.n_rows
        if n > _TOP:
            _int(n, "n_seqs")
        at = None if t is None else t.data_ptr()
        # read for one sequence while another's length is written
        if rows is not None and at is not None and self._lens[0] - 4 * n < at < self._lens[1]:
            _bad(f"{what} lies in the pool's lens: pass a copy, or no rows")
        return n, None if rows is None else rows.data_ptr(), at

    def extend(self, new, n_tokens, rows=None, prefix_len=0):
        """Sequence b, row rows[b] of the pool (None: row b), grows by new[b] rows (int32, on the device): a PageStep.
        n_tokens: room for new tokens, the sum of new or more (bpd_pages_extend_gpu)."""
        if new is None:
            _bad("new is None")
        B, rp, np_ = self._rows(rows, new, "new")
        dev, T, W = self.device, n_tokens, self.width
        if T < 0:
            _bad("n_tokens is negative")
        if T > _TOP or not 0 <= prefix_len <= _TOP:
            _bad(f"n_tokens {T} or prefix_len {prefix_len} does not fit 31 bits")
        sizes = (B, B + 1, T, T, B, 0 if rows is None else B * W)
        out = torch.empty(sum(sizes), dtype=torch.int32, device=dev)
        lens, q_start, slots, pos, refused, table = out.split_with_sizes(sizes)
        if B == 0:
            q_start.zero_()
            slots.fill_(-1)
            pos.fill_(-1)
        table = self.table[:B] if rows is None else table.view(B, W)
        _launch(dev, gpu._fn("bpd_pages_extend_on_gpu"), self._p, rp, np_, B, T, prefix_len,
                None if rows is None else table.data_ptr(), W, lens.data_ptr(), q_start.data_ptr(), slots.data_ptr(),
                pos.data_ptr(), refused.data_ptr())
        return PageStep(table, lens, q_start, slots, pos, refused, T, prefix_len)

    def release(self, keep=None, rows=None, window=None, sinks=0, prefix_len=0):
        """Sequence b keeps its first keep[b] rows (int32, on the device; None: all) and gives its other pages back; with a
        window also those that neither the tokens to come see through it nor hold one of the first `sinks` positions, of
        which the first prefix_len are a shared prefix's (bpd_pages_release_gpu).  rows and keep None: every row."""
        B, rp, kp = self._rows(rows, keep, "keep")
        if window is not None and (window < 1 or self.gone is None):
            _bad(f"window {window} is below 1, or the pool is without gone")
        if sinks < 0 or prefix_len < 0:
            _bad("sinks or prefix_len is negative")
        # rows end below _TOP: beyond it a window, or first rows, are all of them
        w, own = 0 if window is None else window if window < _TOP else _TOP, sinks - prefix_len
        _launch(self.device, gpu._fn("bpd_pages_release_on_gpu"), self._p, rp, kp, B, w,
                0 if own < 0 else own if own < _TOP else _TOP)


def _weights(w, what, x, heads, D):
    """Address and stride of a norm's weights [head_dim] or [heads, head_dim], float32 or of x's type."""
    if w is None:
        return None, 0
    if w.dtype is not torch.float32 and w.dtype is not x.dtype or w.device != x.device:
        _bad(f"{what} is {w.dtype} on {w.device}, not float32 or {x.dtype} on {x.device}")
    if w.shape != (D,) and w.shape != (heads, D) or not w.is_contiguous():
        _bad(f"{what} is not a contiguous [{D}] or [{heads}, {D}]")
    return w.data_ptr(), 0 if w.dim() == 1 else D


def rope_append(cache, batch, q, k, v, rope=None, pos=None, q_out=None, q_norm=None, k_norm=None, eps=1e-6):
    """Rotates q [n_tokens, heads, head_dim] and k, and writes k and v [n_tokens, n_kv_heads, head_dim]
    into the new tokens' rows of the cache; returns the rotated q (q_out, which may be q itself).  Rows of a padded
    batch that belong to no sequence are left as they are in q_out; in a new tensor they are arbitrary.
    q or both of k and v may be None.  rope None: nothing rotates.  pos int32 [n_tokens]: positions
    other than prefix_len + the token's index.  Token strides of q, k and v are free, so the
    parts of a fused projection's rows will do.
    q_norm, k_norm: weights [head_dim] or [heads, head_dim], float32 or of q's type: every head of q or k becomes
    x / sqrt(mean x^2 + eps) * weight before it turns (bpd_norm_rope_append_paged_gpu)."""
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
            q_out, os_ = q.new_empty(T, H, D), H * D   # 0.4 us less than torch.empty
        else:
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
    args = (None if rope is None else rope._p, None if pos is None else pos.data_ptr(), qp, qs, kp, ks, vp, vs, op, os_,
            TYPES[x.dtype], H)
    if q_norm is None and k_norm is None:
        _launch(dev, gpu._fn("bpd_rope_append_paged_on_gpu"), cache._p, batch._p, *args)
    else:
        qw, qws = _weights(q_norm, "q_norm", x, H, D)
        kw, kws = _weights(k_norm, "k_norm", x, cache.n_kv_heads, D)
        wt = (k_norm if q_norm is None else q_norm).dtype
        if q_norm is not None and k_norm is not None and k_norm.dtype is not wt:
            _bad(f"q_norm is {wt} and k_norm {k_norm.dtype}")
        _launch(dev, gpu._fn("bpd_norm_rope_append_paged_on_gpu"), cache._p, batch._p, qw, qws, kw, kws, TYPES[wt], eps, *args)
    return q_out


def attention(cache, batch, q, scale=None, out=None, return_lse=False, window=None, sinks=0):
    """softmax(scale q k^T) v of every new token over the prefix's rows and its sequence's own up to
    its own (bpd_attn_paged_gpu).  q [n_tokens, heads, head_dim], of the cache's type or float32, as is out.  With q of
    the cache's type the weights are rounded to it before they meet v; with a float32 q they keep 22 bits or more.
    scale: head_dim ** -0.5 unless given.  return_lse: also the float32 [n_tokens, heads] logarithm of each
    softmax's denominator.  Rows of a padded batch that belong to no sequence are left as they are
    in out; in a new tensor they are arbitrary.
    window: a token at position p (the prefix's rows are the first) sees positions p - window + 1 .. p alone, and of those
    before them the first `sinks` (bpd_attn_window_paged_gpu); table entries of pages that none sees may be -1."""
    batch._check(cache)
    if q.dim() != 3:
        _bad(f"q has {q.dim()} dimensions, not 3")
    if window is None and sinks != 0:
        _bad("sinks without a window")
    if window is not None:
        if window < 1:
            _bad("window is below 1")
        if sinks < 0:
            _bad("sinks is negative")
        window, sinks = min(window, _TOP), min(sinks, _TOP)   # positions end below _TOP: beyond it every one is seen
    T, H, D, dev = batch.n_tokens, q.shape[1], cache.head_dim, cache.device
    if q.dtype not in (cache.dtype, torch.float32):
        _bad(f"q is {q.dtype}, neither float32 nor the cache's {cache.dtype}")
    qs = _rows(q, "q", (T, H, D), q.dtype, dev)
    if out is None:
        out, os_ = q.new_empty(T, H, D), H * D
    else:
        os_ = _rows(out, "out", (T, H, D), q.dtype, dev)
    lse = torch.empty((T, H), dtype=torch.float32, device=dev) if return_lse else None
    n = batch._workspace(cache, q.dtype, H, window, sinks)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    wp = None if ws is None else ws.data_ptr()
    args = (cache._p, batch._p, q.data_ptr(), qs, out.data_ptr(), os_, None if lse is None else lse.data_ptr(),
            TYPES[q.dtype], H, D ** -0.5 if scale is None else float(scale))
    if window is None:
        _launch(dev, gpu._fn("bpd_attn_paged_on_gpu"), *args, wp, n)
    else:
        _launch(dev, gpu._fn("bpd_attn_window_paged_on_gpu"), *args, window, sinks, wp, n)
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


def _pitch(t, what):
    """Elements from a row of a 2-D tensor to the next."""
    n, w = t.shape
    s = t.stride()
    if w > 1 and s[1] != 1 or n > 1 and s[0] < w:
        _bad(f"rows of {what} are not contiguous, or overlap")
    return s[0] if n > 1 else w


def adjust_logits(logits, tokens=None, lens=None, prompt=None, repetition=None, frequency=None, presence=None, bias=None,
                  mask=None, mask_row=None, out=None, dtype=None):
    """Rows of logits [rows, vocab] under penalties, biases and masks (bpd_adjust_logits_gpu), in that order.

    tokens     int32 [rows, width]: every row's history, of which the first lens[row] (None: all) count, the first
               prompt[row] of them (None: none) as its prompt
    repetition float32 [rows]: l / r above 0, else l * r, of every token in the history
    frequency  float32 [rows]: times how often a token stands behind the prompt, taken off; presence: once
    bias       (start int32 [rows + 1], token int32 [n], value float32 [n]): added; a token's last entry counts
    mask       int32 [masks, ceil(vocab / 32) or more] of bits: a token whose bit is 0 becomes -infinity; mask_row int32
               [rows]: each row's mask, -1 none (None: mask `row`)
    out        may be logits itself; else a new tensor of dtype, the logits' unless float32"""
    if logits.dtype not in TYPES:
        _bad(f"logits are {logits.dtype}, not float32, float16 or bfloat16")
    if logits.dim() != 2:
        _bad(f"logits have {logits.dim()} dimensions, not 2")
    B, V = logits.shape
    if B > _TOP or V > _TOP:
        _bad(f"logits are {B} x {V}: neither may pass 31 bits")
    dev = logits.device
    xs = _pitch(logits, "logits")
    if out is None:
        if dtype is not None and dtype is not torch.float32 and dtype is not logits.dtype:
            _bad(f"dtype is {dtype}, neither float32 nor the logits' {logits.dtype}")
        out, ys = logits.new_empty(B, V) if dtype in (None, logits.dtype) else logits.new_empty((B, V), dtype=dtype), V
    else:
        if out.dtype not in (logits.dtype, torch.float32) or dtype not in (None, out.dtype) or out.shape != (B, V) \
                or out.device != dev:
            _bad(f"out is {out.dtype} {list(out.shape)} on {out.device}, not {logits.dtype} or float32 {[B, V]} on {dev}")
        ys = _pitch(out, "out")
    if tokens is None and (lens is not None or prompt is not None):
        _bad("lens or prompt without tokens")
    if mask is None and mask_row is not None:
        _bad("mask_row without mask")
    if tokens is None and not (repetition is frequency is presence is None):
        _bad("penalties without tokens")
    i32, r = (torch.int32,), _Rules()

    def per_row(t, what, dt):
        if t is None:
            return None
        if t.dtype is not dt or t.shape != (B,) or t.device != dev or not t.is_contiguous():
            _bad(f"{what} is not a contiguous {dt} [{B}] on {dev}")
        return t.data_ptr()

    if tokens is not None:
        _tensor(tokens, "tokens", i32, 2, dev)
        h, w = tokens.shape
        if h != B:
            _bad(f"tokens has {h} rows and logits {B}")
        r.tokens, r.token_stride, r.token_width = tokens.data_ptr(), _pitch(tokens, "tokens"), _int(w, "tokens' width")
        r.lens, r.prompt = per_row(lens, "lens", torch.int32), per_row(prompt, "prompt", torch.int32)
        r.repetition = per_row(repetition, "repetition", torch.float32)
        r.frequency = per_row(frequency, "frequency", torch.float32)
        r.presence = per_row(presence, "presence", torch.float32)
    if mask is not None:
        _tensor(mask, "mask", i32, 2, dev)
        if mask.shape[1] < (V + 31) // 32:
            _bad(f"mask has {mask.shape[1]} words a row for {V} tokens")
        r.mask, r.mask_stride, r.n_masks = mask.data_ptr(), _pitch(mask, "mask"), _int(mask.shape[0], "the number of masks")
        r.mask_row = per_row(mask_row, "mask_row", torch.int32)
    if bias is not None:
        start, token, value = bias
        _tensor(start, "bias's start", i32, 1, dev, contiguous=True)
        _tensor(token, "bias's token", i32, 1, dev, contiguous=True)
        _tensor(value, "bias's value", (torch.float32,), 1, dev, contiguous=True)
        if start.shape[0] != B + 1 or token.shape != value.shape:
            _bad(f"bias has {start.shape[0]} offsets for {B} rows, or {token.shape[0]} tokens and {value.shape[0]} values")
        r.bias_start, r.bias_token, r.bias_value, r.n_bias = (start.data_ptr(), token.data_ptr(), value.data_ptr(),
                                                              _int(token.shape[0], "the number of biases"))
    _launch(dev, gpu._fn("bpd_adjust_logits_on_gpu"), logits.data_ptr(), TYPES[logits.dtype], xs, out.data_ptr(),
            TYPES[out.dtype], ys, B, V, ctypes.addressof(r))
    return out
