"""Performance cases of the operators around a serving step.

Four kinds of case, each a pass through public entry points of bpd_substrate_amd.serve:

  attn     attention over a paged cache in which a token sees the last `window` positions and the
           first `sinks` ones (serve.attention with window and sinks)
  append   queries and keys normed head by head, rotated, keys and values written into the pages
           (serve.rope_append with q_norm and k_norm)
  adjust   logits with penalties for repeated tokens, biases and grammar masks (serve.adjust_logits)
  pages    pages handed to growing sequences, their tables, slots and positions, and taken back
           (serve.PagePool.extend and release)

With `own` false run() computes the same in elementary torch operations.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one user in the middle of a conversation, a layer that sees 512 positions: latency counts
        dict(name="attn_one_user", kind="attn", B=1, n=1, ctx=1500, prefix=0, window=512, sinks=4, H=32, HKV=8, D=64,
             q="f16", kv="f16", page=16, heads_first=True),
        # one token for each of 64 users with long contexts, a window of 1024
        dict(name="attn_window_64", kind="attn", B=64, n=1, ctx=8192, prefix=0, window=1024, sinks=4, H=32, HKV=8, D=128,
             q="bf16", kv="bf16", page=64, heads_first=True),
        # fp32 queries, pages of an odd length whose rows hold all heads, a system prompt of which the first rows
        # stay visible, some windows reaching into it
        dict(name="attn_f32_odd", kind="attn", B=17, n=1, ctx=5000, prefix=777, window=2500, sinks=61, H=20, HKV=5, D=96,
             q="f32", kv="f16", page=21, heads_first=False),
        # chunks of up to 512 prompt tokens of eight users; the largest
        dict(name="attn_chunks", kind="attn", B=8, n=512, ctx=8192, prefix=0, window=4096, sinks=16, H=32, HKV=8, D=128,
             q="bf16", kv="bf16", page=64, heads_first=True),
        # one decode step of 64 users, fp32 activations and binary16 pages: a few hundred kilobytes
        dict(name="append_decode_64", kind="append", B=64, n=1, ctx=1024, prefix=0, H=32, HKV=8, D=128, rot=128,
             neox=True, x="f32", kv="f16", page=16, heads_first=True, fused=True, w="f32"),
        # chunks of several users' prompts, the rows of one fused projection
        dict(name="append_prompt_bf16", kind="append", B=16, n=512, ctx=2048, prefix=1000, H=32, HKV=8, D=128, rot=128,
             neox=True, x="bf16", kv="bf16", page=64, heads_first=True, fused=True, w="bf16"),
        # 80-wide heads of which 40 turn in neighbouring pairs, odd pages
        dict(name="append_odd_f16", kind="append", B=37, n=61, ctx=700, prefix=333, H=20, HKV=5, D=80, rot=40,
             neox=False, x="f16", kv="f16", page=21, heads_first=False, fused=False, w="f32"),
        # one user's logits of a 32,000-word head, penalties over a conversation of up to 2,000 tokens
        dict(name="adjust_one_user", kind="adjust", B=1, V=32000, x="f32", out="f32", hist=2000, bias=0, masks=0,
             allow=1.0),
        # 64 users with settings of their own: long histories, up to 300 biases each, some behind one of 8 grammars
        dict(name="adjust_mixed_64", kind="adjust", B=64, V=128256, x="f32", out="f32", hist=16384, bias=300, masks=8,
             allow=0.02),
        # 256 users, binary16 logits to fp32, a grammar each that lets half of the words through
        dict(name="adjust_masks_256", kind="adjust", B=256, V=128256, x="f16", out="f32", hist=1000, bias=0, masks=256,
             allow=0.5),
        # a decode step of 256 sequences with up to 4 draft tokens each, which are then rejected
        dict(name="pages_drafts_256", kind="pages", B=256, n=4, ctx=8192, page=16, spare=1.0),
        # prompts of up to 2,048 tokens for 64 new sequences from a pool that holds most of them, then all of it back
        dict(name="pages_prompts_64", kind="pages", B=64, n=2048, ctx=0, page=16, spare=0.9),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _heads(rng):
    hkv = rng.choice([1, 2, 4, 5, 8])
    return dict(H=hkv * rng.choice([1, 2, 4, 5, 8]), HKV=hkv)


def draw(rng):
    kind = rng.choice(["attn", "attn", "append", "adjust", "pages"])
    page, heads_first = rng.choice([8, 16, 21, 32, 64, 128]), rng.random() < 0.5
    if kind == "attn":
        kv = rng.choice(["f16", "bf16"])
        B = _log(rng, 1, 128)
        n = rng.choice([1, 1, _log(rng, 2, max(2, 2048 // B))])
        c = dict(kind=kind, B=B, n=n, ctx=_log(rng, max(n, 16), max(n, 131072 // B)),
                 prefix=rng.choice([0, 0, _log(rng, 10, 4096)]), window=_log(rng, 16, 4096),
                 sinks=rng.choice([0, 1, 4, _log(rng, 5, 200)]), **_heads(rng), D=rng.choice([64, 80, 96, 128, 256]),
                 q=rng.choice([kv, kv, "f32"]), kv=kv, page=page, heads_first=heads_first)
        while c["n"] > 1 and work(c)["flops"] > 1.2e11:  # at most the largest listed case's work
            c["n"] = max(1, c["n"] // 2)
        return c
    if kind == "append":
        D = rng.choice([64, 80, 96, 128, 256])
        x = rng.choice(["f32", "f16", "bf16"])
        B = _log(rng, 1, 128)
        return dict(kind=kind, B=B, n=rng.choice([1, _log(rng, 2, 8192 // B)]), ctx=_log(rng, 8192 // B, 32768 // B),
                    prefix=rng.choice([0, _log(rng, 10, 16384)]), **_heads(rng), D=D, rot=rng.choice([D, D // 2]),
                    neox=rng.random() < 0.5, x=x, kv=x if x != "f32" else rng.choice(["f16", "bf16"]), page=page,
                    heads_first=heads_first, fused=rng.random() < 0.5, w=rng.choice(["f32", x]))
    if kind == "adjust":
        x, what = rng.choice(["f32", "f16", "bf16"]), rng.randrange(1, 8)  # any of the three, one at least
        return dict(kind=kind, B=_log(rng, 1, 256), V=_log(rng, 1000, 128256), x=x, out=rng.choice([x, "f32"]),
                    hist=_log(rng, 1, 16384) if what & 1 else 0, bias=_log(rng, 1, 300) if what & 2 else 0,
                    masks=_log(rng, 1, 64) if what & 4 else 0, allow=rng.choice([0.001, 0.02, 0.5, 0.9]))
    B = _log(rng, 1, 512)
    n = rng.choice([1, 4, _log(rng, 5, max(5, 131072 // B))])
    return dict(kind=kind, B=B, n=n, ctx=rng.choice([0, _log(rng, 16, 8192)]), page=rng.choice([1, 8, 16, 21, 64, 128]),
                spare=rng.choice([0.5, 0.9, 1.0, 1.0]))


# ---------------------------------------------------------------- what a user's program has in hand

class _Gen:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.r = random.Random(seed)

    def normal(self, *shape, dtype=torch.float32):
        """Normal values; made in fp32 a part at a time where they are many."""
        t = torch.empty(shape, dtype=dtype, device="cuda")
        flat = t.reshape(-1)
        for at in range(0, flat.numel(), 1 << 27):
            part = flat[at:at + (1 << 27)]
            part.copy_(torch.randn(part.numel(), generator=self.g, device="cuda"))
        return t

    def uniform(self, n):
        return torch.rand(n, generator=self.g, device="cuda")


def _i32(values):
    return torch.tensor(np.asarray(values, np.int64), dtype=torch.int32, device="cuda")


def _lengths(c):
    """New tokens and length (with them) of every sequence's own part: the case's alone, so that every seed
    of a case is the same amount of work and work() can count it."""
    r = random.Random("%d %d %d" % (c["B"], c["n"], c["ctx"]))
    n = [1 if c["n"] == 1 else r.randint(max(1, c["n"] // 2), c["n"]) for _ in range(c["B"])]
    return n, [r.randint(max(k, c["ctx"] // 4), max(k, c["ctx"])) for k in n]


def _paged(c, g, s):
    """The cache's pages in a shuffled order, page tables, lengths: what a serving loop keeps."""
    n, lens = _lengths(c)
    P, page = c["prefix"], c["page"]
    npre, per = -(-P // page), [-(-l // page) for l in lens]
    pages = npre + sum(per) + 3
    order = list(range(pages))
    g.r.shuffle(order)
    table = np.full((c["B"], max(per)), -1, np.int64)
    at = npre
    for b, k in enumerate(per):
        table[b, :k] = order[at:at + k]
        at += k
    shape = ((pages, c["HKV"], page, c["D"]) if c["heads_first"] else (pages, page, c["HKV"], c["D"]))
    k, v = (g.normal(*shape, dtype=TYPES[c["kv"]]) for _ in range(2))
    s["k_pages"], s["v_pages"] = (t.transpose(1, 2) if c["heads_first"] else t for t in (k, v))
    s["table"], s["lens"], s["prefix_pages"] = _i32(table), _i32(lens), _i32(order[:npre]) if npre else None
    s["T"], s["nmax"] = sum(n), max(n)
    s["q_start"] = _i32(np.concatenate([[0], np.cumsum(n)])) if c["n"] > 1 else None
    if own:
        serve = s["serve"]
        s["cache"] = serve.PagedCache(s["k_pages"], s["v_pages"])
        s["batch"] = serve.PagedBatch(s["table"], s["lens"], q_start=s["q_start"], n_tokens=s["T"],
                                      prefix=s["prefix_pages"], prefix_len=P)


def prepare(case, seed):
    c, g = case, _Gen(seed)
    s = dict(c)
    if own:
        from bpd_substrate_amd import serve
        s["serve"] = serve
    if c["kind"] == "adjust":
        return _prepare_adjust(c, g, s)
    if c["kind"] == "pages":
        return _prepare_pages(c, g, s)
    _paged(c, g, s)
    T, H, HKV, D = s["T"], c["H"], c["HKV"], c["D"]
    if c["kind"] == "attn":
        s["qs"] = g.normal(T, H, D, dtype=TYPES[c["q"]])
        return s
    if c["fused"]:  # the rows of one Q/K/V projection
        row = g.normal(T, H + 2 * HKV, D, dtype=TYPES[c["x"]])
        s["qs"], s["ks"], s["vs"] = row[:, :H], row[:, H:H + HKV], row[:, H + HKV:]
    else:
        s["qs"], s["ks"], s["vs"] = (g.normal(T, h, D, dtype=TYPES[c["x"]]) for h in (H, HKV, HKV))
    s["qw"], s["kw"] = ((1.0 + 0.2 * g.normal(D)).to(TYPES[c["w"]]) for _ in range(2))
    s["eps"] = 1e-6
    # the frequency of each rotated pair, in radians per position
    s["freq"] = torch.tensor([10000.0 ** (-2.0 * j / c["rot"]) for j in range(c["rot"] // 2)], dtype=torch.float64,
                             device="cuda")
    if own:
        s["rope"] = s["serve"].Rope(c["rot"], base=10000.0, neox=c["neox"], device="cuda")
    return s


def _prepare_adjust(c, g, s):
    """Logits as a model's head gives them, histories whose words repeat, every user's own settings."""
    B, V = c["B"], c["V"]
    x = 2.0 * g.normal(B, V)
    few = torch.randint(0, V, (B, 40), generator=g.g, device="cuda")
    x.scatter_add_(1, few, 5.0 + 3.0 * g.normal(B, 40))
    s["logits"] = x.to(TYPES[c["x"]])
    r = random.Random("%d %d" % (B, c["hist"]))
    for name in ("tokens", "lens", "prompt", "repetition", "frequency", "presence", "bias", "mask", "mask_row"):
        s[name] = None
    if c["hist"]:
        lens = [r.randint(max(1, c["hist"] // 4), c["hist"]) for _ in range(B)]
        s["tokens"] = (V * torch.rand(B, c["hist"], generator=g.g, device="cuda").pow(4)).int().clamp_(max=V - 1)
        s["lens"], s["prompt"] = _i32(lens), _i32([r.randint(0, k) for k in lens])
        off = lambda x, neutral: torch.where(g.uniform(B) < 0.25, neutral, x)  # noqa: E731
        s["repetition"] = off(1.0 + 0.3 * g.uniform(B), 1.0)
        s["frequency"], s["presence"] = off(0.5 * g.uniform(B), 0.0), off(0.5 * g.uniform(B), 0.0)
    if c["bias"]:
        per = [r.randint(0, c["bias"]) for _ in range(B)]
        words = [g.r.sample(range(V), min(k, V)) for k in per]
        start = np.concatenate([[0], np.cumsum([len(w) for w in words])])
        flat = [w for row in words for w in row]
        s["bias"] = (_i32(start), _i32(flat), 4.0 * g.normal(len(flat)))
    if c["masks"]:
        N = -(-V // 32)
        bits = torch.zeros(c["masks"], N, dtype=torch.int64, device="cuda")
        for i in range(32):
            bits |= (torch.rand(c["masks"], N, generator=g.g, device="cuda") < c["allow"]).long() << i
        bits = torch.where(bits >= 1 << 31, bits - (1 << 32), bits)
        s["mask"] = bits.int()
        s["mask_row"] = _i32([i if c["masks"] == B else r.randint(-1, c["masks"] - 1) for i in range(B)])
    return s


def _page_lengths(c):
    """Rows before and new tokens of every sequence."""
    r = random.Random("%d %d %d" % (c["B"], c["n"], c["ctx"]))
    old = [r.randint(c["ctx"] // 4, c["ctx"]) for _ in range(c["B"])]
    return old, [r.randint(max(1, c["n"] // 4), c["n"]) for _ in range(c["B"])]


def _prepare_pages(c, g, s):
    """A pool in use: every sequence's pages in its row of the table, the others on the free stack."""
    B, page = c["B"], c["page"]
    old, new = _page_lengths(c)
    used = [-(-l // page) for l in old]
    need = sum(-(-(l + k) // page) for l, k in zip(old, new)) - sum(used)
    width = -(-(c["ctx"] + c["n"]) // page)
    R = B + B // 4 + 1  # rows, some of them idle
    n_free = int(math.ceil(need * c["spare"])) + (5 if c["spare"] == 1.0 else 0)
    order = np.random.default_rng(g.r.randrange(1 << 30)).permutation(sum(used) + n_free + 3)
    rows = g.r.sample(range(R), B)
    table, lens, at = np.full((R, width), -1, np.int64), np.zeros(R, np.int64), 0
    for b, row in enumerate(rows):
        table[row, :used[b]] = order[at:at + used[b]]
        lens[row] = old[b]
        at += used[b]
    free = np.full(len(order), -1, np.int64)
    free[:n_free] = order[at:at + n_free]
    s["table"], s["lens"], s["free"], s["n_free"] = _i32(table), _i32(lens), _i32(free), _i32([n_free, 0])
    s["rows"], s["new"], s["old"], s["T"] = _i32(rows), _i32(new), _i32(old), sum(new)
    if own:
        s["pool"] = s["serve"].PagePool(s["table"], s["lens"], s["free"], s["n_free"], page)
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    s = state
    if own:
        serve = s["serve"]
        if s["kind"] == "attn":
            out, lse = serve.attention(s["cache"], s["batch"], s["qs"], window=s["window"], sinks=s["sinks"],
                                       return_lse=True)
            return {"out": out, "lse": lse}
        if s["kind"] == "append":
            q = serve.rope_append(s["cache"], s["batch"], s["qs"], s["ks"], s["vs"], rope=s["rope"], q_norm=s["qw"],
                                  k_norm=s["kw"], eps=s["eps"])
            return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if s["kind"] == "adjust":
            out = serve.adjust_logits(s["logits"], tokens=s["tokens"], lens=s["lens"], prompt=s["prompt"],
                                      repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                                      bias=s["bias"], mask=s["mask"], mask_row=s["mask_row"], dtype=TYPES[s["out"]])
            return {"logits": out}
        step = s["pool"].extend(s["new"], s["T"], rows=s["rows"])
        s["pool"].release(s["old"], rows=s["rows"])
        return _pages_out(s, step.table, step.lens, step.q_start, step.slots, step.pos, step.refused)
    return {"attn": _attn_plain, "append": _append_plain, "adjust": _adjust_plain, "pages": _pages_plain}[s["kind"]](s)


def _pages_out(s, table, lens, q_start, slots, pos, refused):
    return {"table": table, "lens": lens, "q_start": q_start, "slots": slots, "pos": pos, "refused": refused,
            "pool_table": s["table"], "pool_lens": s["lens"], "free": s["free"], "n_free": s["n_free"]}


def _tokens(s):
    """Sequence and index in the sequence's own part of every new token."""
    lens, dev = s["lens"].long(), s["lens"].device
    if s["q_start"] is None:
        return torch.arange(len(lens), device=dev), lens - 1
    start = s["q_start"].long()
    t = torch.arange(s["T"], device=dev)
    seq = torch.searchsorted(start, t, right=True) - 1
    return seq, lens[seq] - (start[seq + 1] - start[seq]) + t - start[seq]


def _attn_plain(s):
    """Every sequence's sinks and the band that its new tokens see, padded to the longest."""
    B, N, H, HKV, D, P, page = s["B"], s["nmax"], s["H"], s["HKV"], s["D"], s["prefix"], s["page"]
    G, dev, lens, W, S = H // HKV, s["lens"].device, s["lens"].long(), s["window"], s["sinks"]
    seq, at = _tokens(s)
    start = torch.arange(B + 1, device=dev) if s["q_start"] is None else s["q_start"].long()
    slot = seq * N + torch.arange(s["T"], device=dev) - start[seq]
    q = torch.zeros(B * N, H, D, device=dev)
    q[slot] = s["qs"].float() * (1.0 / math.sqrt(D))
    q = q.reshape(B, N, HKV, G, D).permute(0, 2, 1, 3, 4).reshape(B, HKV, N * G, D)
    p = torch.full((B * N,), -1, device=dev)  # the tokens' positions
    p[slot] = P + at
    p = p.reshape(B, 1, N, 1).expand(B, 1, N, G).reshape(B, 1, N * G, 1)
    # positions of the keys: the sinks, then the band from the first token's window on
    top = P + lens
    low = (top - (start[1:] - start[:-1]) - W + 1).clamp(min=S)
    n_sinks = min(S, P + s["table"].shape[1] * page)
    band = min(N - 1 + W, P + s["table"].shape[1] * page)
    j = torch.cat([torch.arange(n_sinks, device=dev).expand(B, -1), low[:, None] + torch.arange(band, device=dev)], 1)
    there = j < top[:, None]
    jo = torch.where(there, j - P, 0)
    page_of = s["table"].long().gather(1, (jo.clamp(min=0) // page))
    row_of = jo.clamp(min=0) % page
    if P:
        jp = j.clamp(max=P - 1)
        page_of = torch.where(jo < 0, s["prefix_pages"].long()[jp // page], page_of)
        row_of = torch.where(jo < 0, jp % page, row_of)
    page_of = page_of.clamp(min=0)
    j = j[:, None, None, :]
    seen = there[:, None, None, :] & (j <= p) & ((j > p - W) | (j < S))
    k = s["k_pages"][page_of, row_of].float().permute(0, 2, 3, 1).contiguous()
    x = torch.matmul(q, k).masked_fill_(~seen, -math.inf)
    del k
    m = x.amax(-1, keepdim=True)
    m0 = m.masked_fill(m == -math.inf, 0.0)
    x = torch.exp_(x.sub_(m0))
    norm = x.sum(-1, keepdim=True)
    v = s["v_pages"][page_of, row_of].float().permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(x, v)
    out = torch.where(norm > 0, out / norm, 0.0)
    lse = m0 + torch.log(norm)
    back = lambda x: x.reshape(B, HKV, N, G, -1).transpose(1, 2).reshape(B * N, H, -1)[slot]  # noqa: E731
    return {"out": back(out).to(s["qs"].dtype), "lse": back(lse)[..., 0]}


def _norm(x, w, eps):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.float()


def _rotate(x, cos, sin, rot, neox):
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if neox else (x[..., 0:rot:2], x[..., 1:rot:2])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([ra, rb], -1) if neox else torch.stack([ra, rb], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _append_plain(s):
    seq, at = _tokens(s)
    angle = (s["prefix"] + at).double()[:, None] * s["freq"]
    cos, sin = (f(angle).float()[:, None, :] for f in (torch.cos, torch.sin))
    q, k = (_rotate(_norm(x, w, s["eps"]), cos, sin, s["rot"], s["neox"])
            for x, w in ((s["qs"], s["qw"]), (s["ks"], s["kw"])))
    page, row = s["table"].long()[seq, at // s["page"]], at % s["page"]
    s["k_pages"][page, row] = k.to(s["k_pages"].dtype)
    s["v_pages"][page, row] = s["vs"].to(s["v_pages"].dtype)
    return {"q": q.to(s["qs"].dtype), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _adjust_plain(s):
    x = s["logits"].float()
    B, V, dev = s["B"], s["V"], x.device
    if s["tokens"] is not None:
        i = torch.arange(s["tokens"].shape[1], device=dev)
        there, made = i < s["lens"][:, None], i >= s["prompt"][:, None]
        t = s["tokens"].long()
        count = torch.zeros(B, V, device=dev).scatter_add_(1, t, (there & made).float())
        met = torch.zeros(B, V, device=dev).scatter_add_(1, t, there.float()) > 0
        r = s["repetition"][:, None]
        x = torch.where(met, torch.where(x > 0, x / r, x * r), x)
        x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        start, word, value = s["bias"]
        row = torch.searchsorted(start.long(), torch.arange(len(word), device=dev), right=True) - 1
        x = x.index_put((row, word.long()), value, accumulate=True)
    if s["mask"] is not None:
        v = torch.arange(V, device=dev)
        row = s["mask_row"].long()
        allowed = (s["mask"][row.clamp(min=0)][:, v // 32] >> (v % 32).int()) & 1
        x = x.masked_fill((allowed == 0) & (row >= 0)[:, None], -math.inf)
    return {"logits": x.to(TYPES[s["out"]])}


def _pages_plain(s):
    page, T, rows, new, dev = s["page"], s["T"], s["rows"].long(), s["new"].long(), s["rows"].device
    table, lens, free, n_free = s["table"], s["lens"], s["free"], s["n_free"][0].long()
    B, width = len(rows), table.shape[1]
    before = lens[rows].long()
    used, want = (before + page - 1) // page, (before + new + page - 1) // page
    fits = want <= width
    need = torch.where(fits, want - used, 0)
    paid = fits & ((need == 0) | (torch.cumsum(need, 0) <= n_free))
    granted = paid & (torch.cumsum(torch.where(paid, new, 0), 0) <= T)
    refused = torch.where(~fits, 2, torch.where(~paid, 3, torch.where(~granted, 4, 0)))
    new, need = torch.where(granted, new, 0), torch.where(granted, need, 0)
    # pages from the top of the stack, sequence by sequence
    first = torch.cumsum(need, 0) - need
    i = torch.arange(width, device=dev)
    entry = i[None, :] - used[:, None]
    fresh = (entry >= 0) & (entry < need[:, None])
    at = (n_free - 1 - first[:, None] - entry).clamp(0, free.shape[0] - 1)
    mine = table[rows].masked_fill(i >= used[:, None], -1)
    mine = torch.where(fresh, free[at], mine)
    table[rows] = mine
    after = before + new
    lens[rows] = after.int()
    n_free = n_free - need.sum()
    # the tokens
    start = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), torch.cumsum(new, 0)])
    t = torch.arange(T, device=dev)
    seq = (torch.searchsorted(start, t, right=True) - 1).clamp(max=B - 1)
    row = before[seq] + t - start[seq]
    real = t < start[-1]
    entry = mine[seq, (row // page).clamp(max=width - 1)].long()
    slots = torch.where(real, entry * page + row % page, -1).int()
    pos = torch.where(real, row, -1).int()
    # and back: what stands behind the old lengths goes onto the stack, last first
    keep = torch.minimum(s["old"].long(), after)
    kept = (keep + page - 1) // page
    give = (after + page - 1) // page - kept
    first = torch.cumsum(give, 0) - give
    entry = i[None, :] - kept[:, None]
    gone = (entry >= 0) & (entry < give[:, None])
    total = give.sum()
    at = n_free + total - 1 - first[:, None] - entry
    spill = torch.cat([free, free[:1]])  # entries that stay write behind its end
    spill[torch.where(gone, at, free.shape[0])] = mine
    free.copy_(spill[:-1])
    table[rows] = mine.masked_fill(gone, -1)
    lens[rows] = keep.int()
    s["n_free"][0] = n_free + total
    return _pages_out(s, mine, after.int(), start.int(), slots, pos, refused.int())


# ---------------------------------------------------------------- what a pass cannot do without

def _visible(c, n, length):
    """Pairs of a sequence's new tokens and the keys that they see, and the keys that any of them sees."""
    P, W, S = c["prefix"], c["window"], c["sinks"]
    pairs = 0
    for p in range(P + length - n, P + length):
        low = max(0, p - W + 1)
        pairs += p + 1 - low + min(S, low)
    low = max(0, P + length - n - W + 1)
    return pairs, P + length - low + min(S, low)


def work(case):
    c = case
    if c["kind"] == "adjust":
        r = random.Random("%d %d" % (c["B"], c["hist"]))
        hist = sum(r.randint(max(1, c["hist"] // 4), c["hist"]) for _ in range(c["B"])) if c["hist"] else 0
        return {"bytes": c["B"] * c["V"] * (SIZE[c["x"]] + SIZE[c["out"]]) + 4 * hist + c["masks"] * -(-c["V"] // 32) * 4
                + 4 * c["B"] * c["bias"], "flops": c["B"] * c["V"]}
    if c["kind"] == "pages":
        old, new = _page_lengths(c)
        width = -(-(c["ctx"] + c["n"]) // c["page"])
        entries = sum(-(-(l + k) // c["page"]) for l, k in zip(old, new))
        return {"bytes": 4 * (c["B"] * width + entries) + 8 * sum(new) + 40 * c["B"], "flops": 2 * sum(new)}
    n, lens = _lengths(c)
    T, H, HKV, D = sum(n), c["H"], c["HKV"], c["D"]
    if c["kind"] == "append":
        return {"bytes": T * D * ((2 * H + 2 * HKV) * SIZE[c["x"]] + 2 * HKV * SIZE[c["kv"]]),
                "flops": T * (H + HKV) * (4 * D + 3 * c["rot"])}
    seen = [_visible(c, k, l) for k, l in zip(n, lens)]
    return {"bytes": 2 * T * H * D * SIZE[c["q"]] + 4 * T * H + 2 * sum(x[1] for x in seen) * HKV * D * SIZE[c["kv"]],
            "flops": 4 * sum(x[0] for x in seen) * H * D}


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    if case["kind"] == "pages":  # whole numbers alone
        return None
    s = prepare(case, seed)
    return {"attn": _attn_exact, "append": _append_exact, "adjust": _adjust_exact}[case["kind"]](s)


def _sequences(s):
    """(first token, tokens, length of its own part, its pages) of every sequence."""
    lens, table = s["lens"].tolist(), s["table"].tolist()
    start = s["q_start"].tolist() if s["q_start"] is not None else list(range(len(lens) + 1))
    return [(start[b], start[b + 1] - start[b], lens[b], table[b][:-(-lens[b] // s["page"])]) for b in range(len(lens))]


def _attn_exact(s):
    """One sequence after another over all of its keys."""
    H, HKV, D, P, W, S = s["H"], s["HKV"], s["D"], s["prefix"], s["window"], s["sinks"]
    if 4.0 * s["T"] * (P + s["ctx"]) * H * D > 4e13:
        return None
    G = H // HKV
    flat = lambda pages, x, n: x[torch.tensor(pages, device="cuda")].reshape(-1, HKV, D)[:n].double().transpose(0, 1)  # noqa: E731
    kp = vp = None
    if P:
        kp, vp = (flat(s["prefix_pages"].tolist(), x, P) for x in (s["k_pages"], s["v_pages"]))
    out = torch.zeros(s["T"], H, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["T"], H, dtype=torch.float64, device="cuda")
    for t0, n, length, pages in _sequences(s):
        k, v = (flat(pages, x, length) for x in (s["k_pages"], s["v_pages"]))
        if P:
            k, v = torch.cat([kp, k], 1), torch.cat([vp, v], 1)
        age = (P + length - n + torch.arange(n, device="cuda"))[:, None] - torch.arange(P + length, device="cuda")
        seen = (age >= 0) & (age < W)
        seen[:, :S] |= age[:, :S] >= 0
        kt = k.transpose(1, 2).contiguous()
        for g in range(G):
            q = s["qs"][t0:t0 + n, g::G].double().transpose(0, 1).contiguous()
            x = torch.where(seen, torch.bmm(q, kt) / D ** 0.5, -math.inf)
            z = torch.logsumexp(x, -1)
            out[t0:t0 + n, g::G] = torch.bmm(torch.exp(x - z[..., None]), v.contiguous()).transpose(0, 1)
            lse[t0:t0 + n, g::G] = z.transpose(0, 1)
    return {"out": out, "lse": lse}


def _append_exact(s):
    k_pages, v_pages, q_out = s["k_pages"].double(), s["v_pages"].double(), s["qs"].double()
    half = s["rot"] // 2
    first = [j if s["neox"] else 2 * j for j in range(half)]
    second = [j + half if s["neox"] else 2 * j + 1 for j in range(half)]
    for t0, n, length, pages in _sequences(s):
        at = torch.arange(length - n, length, device="cuda")
        turn = torch.polar(torch.ones(n, half, dtype=torch.float64, device="cuda"),
                           (s["prefix"] + at)[:, None].double() * s["freq"])[:, None, :]
        done = []
        for x, w in ((s["qs"], s["qw"]), (s["ks"], s["kw"])):
            y = x[t0:t0 + n].double()
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / s["D"] + s["eps"]) * w.double()
            z = torch.complex(y[..., first], y[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            done.append(y)
        page = torch.tensor(pages, device="cuda")[at // s["page"]]
        q_out[t0:t0 + n] = done[0]
        k_pages[page, at % s["page"]] = done[1]
        v_pages[page, at % s["page"]] = s["vs"][t0:t0 + n].double()
    return {"q": q_out, "k_pages": k_pages, "v_pages": v_pages}


def _adjust_exact(s):
    """Row by row on the host."""
    host = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    x = s["logits"].double().cpu().numpy()
    B, V = x.shape
    if s["tokens"] is not None:
        tokens, lens, prompt = host(s["tokens"]), host(s["lens"]), host(s["prompt"])
        r, f, p = (host(s[name]).astype(np.float64) for name in ("repetition", "frequency", "presence"))
        for b in range(B):
            met = np.unique(tokens[b, :lens[b]])
            y = x[b, met]
            x[b, met] = np.where(y > 0, y / r[b], y * r[b])
            made, count = np.unique(tokens[b, prompt[b]:lens[b]], return_counts=True)
            x[b, made] -= f[b] * count + p[b]
    if s["bias"] is not None:
        start, word, value = (host(t) for t in s["bias"])
        for b in range(B):
            for i in range(start[b], start[b + 1]):
                x[b, word[i]] += value[i]
    if s["mask"] is not None:
        bits, row = host(s["mask"]).view(np.uint32), host(s["mask_row"])
        for b in range(B):
            if row[b] >= 0:
                one = np.unpackbits(bits[row[b]].view(np.uint8), bitorder="little")[:V]
                x[b, one == 0] = -np.inf
    return {"logits": torch.from_numpy(x)}
