"""Performance cases of the operators that serve many sequences at once.

Three kinds of case, each one call of a public entry point of bpd_substrate_amd.serve:

  append   the new tokens' queries and keys rotated, keys and values written into the pages of a
           paged cache (serve.rope_append)
  attn     attention over a paged cache for a batch whose sequences share a prefix: the prefix is
           read once for all of them, every sequence's own pages for itself (serve.attention)
  sample   one token per row of logits with temperature, top-k, top-p and min-p from given random
           numbers (serve.sample)

With `own` false run() computes the same in elementary torch operations.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one decode step of a 64-user batch, fp32 activations as the decode step has them and binary16
        # pages: a few hundred kilobytes, so latency counts
        dict(name="append_decode_64", kind="append", B=64, n=1, ctx=1024, prefix=0, H=32, HKV=8, D=128, rot=128,
             neox=False, x="f32", kv="f16", page=16, heads_first=True, fused=True),
        # chunks of prompts of several users, 3,500 to 8,000 tokens in all, fused projection rows
        dict(name="append_prompt_bf16", kind="append", B=16, n=512, ctx=2048, prefix=1000, H=32, HKV=8, D=128, rot=128,
             neox=False, x="bf16", kv="bf16", page=64, heads_first=True, fused=True),
        # odd sizes: 96-wide heads of which 48 rotate in halves, odd page length, cache rows across all heads
        dict(name="append_odd_f16", kind="append", B=37, n=61, ctx=700, prefix=333, H=20, HKV=5, D=96, rot=48,
             neox=True, x="f16", kv="f16", page=21, heads_first=False, fused=False),
        # one user early in a conversation: the smallest attention call
        dict(name="attn_one_user", kind="attn", B=1, n=1, ctx=300, prefix=0, H=32, HKV=8, D=64, q="f16", kv="f16",
             page=16, heads_first=True),
        # 64 users behind one 8k system prompt, short turns of their own
        dict(name="attn_prefix8k_64", kind="attn", B=64, n=1, ctx=600, prefix=8192, H=32, HKV=8, D=128, q="f16",
             kv="f16", page=16, heads_first=True),
        # 32 users with long contexts of their own and nothing shared
        dict(name="attn_paged_32", kind="attn", B=32, n=1, ctx=8192, prefix=0, H=32, HKV=8, D=128, q="bf16", kv="bf16",
             page=64, heads_first=True),
        # fp32 queries against binary16 pages whose rows hold all heads, as the decode step's caches are laid out
        dict(name="attn_f32_rows", kind="attn", B=16, n=1, ctx=1500, prefix=2011, H=32, HKV=8, D=128, q="f32",
             kv="f16", page=32, heads_first=False),
        # chunks of up to 512 prompt tokens of eight users behind a 4k prefix
        dict(name="attn_chunks", kind="attn", B=8, n=512, ctx=1024, prefix=4096, H=32, HKV=8, D=128, q="bf16",
             kv="bf16", page=64, heads_first=True),
        # 256 users behind a 32k document; the largest
        dict(name="attn_prefix32k_256", kind="attn", B=256, n=1, ctx=1024, prefix=32768, H=32, HKV=8, D=128, q="bf16",
             kv="bf16", page=64, heads_first=True),
        # one user's next token from a 32,000-word head
        dict(name="sample_one_user", kind="sample", B=1, V=32000, x="f32", how="both"),
        # 64 users, each with settings of their own, a 128k vocabulary
        dict(name="sample_mixed_64", kind="sample", B=64, V=128256, x="f32", how="mixed"),
        # 256 users, binary16 logits, nucleus sampling
        dict(name="sample_topp_256", kind="sample", B=256, V=128256, x="f16", how="top_p"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _heads(rng):
    hkv = rng.choice([1, 2, 4, 5, 8])
    return dict(H=hkv * rng.choice([1, 2, 4, 5, 8]), HKV=hkv)


def draw(rng):
    kind = rng.choice(["append", "attn", "attn", "sample"])
    page, heads_first = rng.choice([8, 16, 21, 32, 64, 128]), rng.random() < 0.5
    if kind == "append":
        D = rng.choice([64, 80, 96, 128, 256])
        x = rng.choice(["f32", "f16", "bf16"])
        B = _log(rng, 1, 128)
        return dict(kind=kind, B=B, n=rng.choice([1, _log(rng, 2, 8192 // B)]), ctx=_log(rng, 8192 // B, 32768 // B),
                    prefix=rng.choice([0, _log(rng, 10, 16384)]), **_heads(rng), D=D,
                    rot=rng.choice([D, D // 2]), neox=rng.random() < 0.5, x=x,
                    kv=x if x != "f32" else rng.choice(["f16", "bf16"]), page=page, heads_first=heads_first,
                    fused=rng.random() < 0.5)
    if kind == "attn":
        kv = rng.choice(["f16", "bf16"])
        B = _log(rng, 1, 128)
        n = rng.choice([1, 1, _log(rng, 2, max(2, 1024 // B))])
        c = dict(kind=kind, B=B, n=n, ctx=_log(rng, max(n, 16), max(n, 65536 // B)),
                 prefix=rng.choice([0, _log(rng, 10, 16384)]), **_heads(rng), D=rng.choice([64, 80, 96, 128, 256]),
                 q=rng.choice([kv, kv, "f32"]), kv=kv, page=page, heads_first=heads_first)
        while c["n"] > 1 and work(c)["flops"] > 1.3e11:  # at most the largest listed case's work
            c["n"] = max(1, c["n"] // 2)
        return c
    return dict(kind=kind, B=_log(rng, 1, 256), V=_log(rng, 1000, 128256), x=rng.choice(["f32", "f16", "bf16"]),
                how=rng.choice(["both", "mixed", "mixed", "top_p", "top_k", "min_p", "plain"]))


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
    if c["kind"] == "sample":
        return _prepare_sample(c, g, s)
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
    # the frequency of each rotated pair, in radians per position
    s["freq"] = torch.tensor([10000.0 ** (-2.0 * j / c["rot"]) for j in range(c["rot"] // 2)], dtype=torch.float64,
                             device="cuda")
    if own:
        s["rope"] = s["serve"].Rope(c["rot"], base=10000.0, neox=c["neox"], device="cuda")
    return s


def _prepare_sample(c, g, s):
    """Logits as a model's head gives them: a wide bulk, and a few dozen words that stand out."""
    B, V = c["B"], c["V"]
    x = 2.0 * g.normal(B, V)
    few = torch.randint(0, V, (B, 40), generator=g.g, device="cuda")
    x.scatter_add_(1, few, 5.0 + 3.0 * g.normal(B, 40))
    s["logits"] = x.to(TYPES[c["x"]])
    s["u"] = g.uniform(B)
    r = lambda lo, hi: lo + (hi - lo) * g.uniform(B)  # noqa: E731
    k = torch.randint(1, 100, (B,), generator=g.g, device="cuda", dtype=torch.int32)
    how = c["how"]
    s["temperature"], s["top_k"], s["top_p"], s["min_p"] = r(0.5, 1.3), None, None, None
    if how in ("both", "top_k"):
        s["top_k"] = k
    if how in ("both", "top_p"):
        s["top_p"] = r(0.5, 0.99)
    if how == "min_p":
        s["min_p"] = r(0.01, 0.2)
    if how == "mixed":  # every user's own settings: each filter on for half of them, some rows greedy
        off = lambda: g.uniform(B) < 0.5  # noqa: E731
        s["temperature"] = torch.where(g.uniform(B) < 0.2, 0.0, s["temperature"])
        s["top_k"] = torch.where(off(), 0, k).int()
        s["top_p"] = torch.where(off(), 1.0, r(0.5, 0.99))
        s["min_p"] = torch.where(off(), 0.0, r(0.01, 0.2))
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    s = state
    if own:
        serve = s["serve"]
        if s["kind"] == "append":
            q = serve.rope_append(s["cache"], s["batch"], s["qs"], s["ks"], s["vs"], rope=s["rope"])
            return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if s["kind"] == "attn":
            out, lse = serve.attention(s["cache"], s["batch"], s["qs"], return_lse=True)
            return {"out": out, "lse": lse}
        token, logprob, kept = serve.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                            top_p=s["top_p"], min_p=s["min_p"])
        return {"token": token, "logprob": logprob, "kept": kept}
    return {"append": _append_plain, "attn": _attn_plain, "sample": _sample_plain}[s["kind"]](s)


def _tokens(s):
    """Sequence and index in the sequence's own part of every new token."""
    lens, dev = s["lens"].long(), s["lens"].device
    if s["q_start"] is None:
        return torch.arange(len(lens), device=dev), lens - 1
    start = s["q_start"].long()
    t = torch.arange(s["T"], device=dev)
    seq = torch.searchsorted(start, t, right=True) - 1
    return seq, lens[seq] - (start[seq + 1] - start[seq]) + t - start[seq]


def _rotate(x, cos, sin, rot, neox):
    x = x.float()
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if neox else (x[..., 0:rot:2], x[..., 1:rot:2])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([ra, rb], -1) if neox else torch.stack([ra, rb], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _append_plain(s):
    seq, at = _tokens(s)
    angle = (s["prefix"] + at).double()[:, None] * s["freq"]
    cos, sin = (f(angle).float()[:, None, :] for f in (torch.cos, torch.sin))
    q, k = (_rotate(x, cos, sin, s["rot"], s["neox"]) for x in (s["qs"], s["ks"]))
    page, row = s["table"].long()[seq, at // s["page"]], at % s["page"]
    s["k_pages"][page, row] = k.to(s["k_pages"].dtype)
    s["v_pages"][page, row] = s["vs"].to(s["v_pages"].dtype)
    return {"q": q.to(s["qs"].dtype), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _attn_plain(s):
    B, N, H, HKV, D, P, page = s["B"], s["nmax"], s["H"], s["HKV"], s["D"], s["prefix"], s["page"]
    G, dev, lens = H // HKV, s["lens"].device, s["lens"].long()
    seq, at = _tokens(s)
    slot = seq * N + (torch.arange(s["T"], device=dev) - (seq if s["q_start"] is None else s["q_start"].long()[seq]))
    q = torch.zeros(B * N, H, D, device=dev)
    q[slot] = s["qs"].float() * (1.0 / math.sqrt(D))
    q = q.reshape(B, N, HKV, G, D).permute(0, 2, 1, 3, 4).reshape(B, HKV, N * G, D)
    # the sequences' own keys, padded to the longest; the new tokens see what stands before them
    L = s["table"].shape[1] * page
    t = torch.arange(L, device=dev)
    rows = s["table"].long().clamp(min=0)[:, t // page]
    seen = torch.full((B * N,), -1, device=dev)
    seen[slot] = at
    seen = seen.reshape(B, 1, N, 1).expand(B, 1, N, G).reshape(B, 1, N * G, 1)
    ks = s["k_pages"][rows, t % page].float().permute(0, 2, 3, 1).contiguous()
    own_s = torch.matmul(q, ks).masked_fill_(t > seen, -math.inf)
    del ks
    m = own_s.amax(-1, keepdim=True)
    if P:
        tp = torch.arange(P, device=dev)
        pre = s["prefix_pages"].long()[tp // page]
        kp = s["k_pages"][pre, tp % page].float().permute(1, 2, 0).contiguous()
        qp = q.transpose(0, 1).reshape(HKV, B * N * G, D)
        pre_s = torch.matmul(qp, kp).reshape(HKV, B, N * G, P).transpose(0, 1)
        m = torch.maximum(m, pre_s.amax(-1, keepdim=True))
    m0 = m.masked_fill(m == -math.inf, 0.0)
    own_s = torch.exp_(own_s.sub_(m0))
    norm = own_s.sum(-1, keepdim=True)
    vs = s["v_pages"][rows, t % page].float().permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(own_s, vs)
    del vs, own_s
    if P:
        pre_s = torch.exp(pre_s - m0)
        norm = norm + pre_s.sum(-1, keepdim=True)
        vp = s["v_pages"][pre, tp % page].float().transpose(0, 1).contiguous()
        pre_s = pre_s.transpose(0, 1).reshape(HKV, B * N * G, P)
        out = out + torch.matmul(pre_s, vp).reshape(HKV, B, N * G, D).transpose(0, 1)
    out = torch.where(norm > 0, out / norm, 0.0)
    lse = m0 + torch.log(norm)
    back = lambda x: x.reshape(B, HKV, N, G, -1).transpose(1, 2).reshape(B * N, H, -1)[slot]  # noqa: E731
    return {"out": back(out).to(s["qs"].dtype), "lse": back(lse)[..., 0]}


def _sample_plain(s):
    """In 64 bits throughout: a token is chosen next to borders between cumulated sums."""
    x = s["logits"].double()
    B, V = x.shape
    ones = torch.ones(B, 1, device=x.device, dtype=torch.float64)
    col = lambda p, off: ones * off if p is None else p.double()[:, None]  # noqa: E731
    t, k, p, mp = col(s["temperature"], 1.0), col(s["top_k"], 0.0), col(s["top_p"], 1.0), col(s["min_p"], 0.0)
    greedy = t <= 0
    x, order = torch.sort(x, dim=1, descending=True, stable=True)  # equal logits by index
    w = torch.exp((x - x[:, :1]) / torch.where(greedy, 1.0, t))
    rank = torch.arange(V, device=x.device)
    keep = (rank < torch.where(greedy, 1.0, torch.where((k <= 0) | (k > V), float(V), k))) & (x > -math.inf)
    w = w * keep
    cum = torch.cumsum(w, 1)
    keep &= (p >= 1) | (cum - w < p * cum[:, -1:]) | (rank == 0)
    keep &= (w >= mp) | (rank == 0)
    w = torch.zeros_like(w).scatter_(1, order, w * keep)  # back in the order of the vocabulary
    cum = torch.cumsum(w, 1)
    total = cum[:, -1:]
    token = (cum <= s["u"].double()[:, None] * total).sum(1).clamp_(max=V - 1)
    logprob = torch.log(w.gather(1, token[:, None]) / total)[:, 0]
    return {"token": token.int(), "logprob": logprob.float(), "kept": keep.sum(1).int()}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if c["kind"] == "sample":
        return {"bytes": c["B"] * c["V"] * size[c["x"]] + c["B"] * 32, "flops": 4 * c["B"] * c["V"]}
    n, lens = _lengths(c)
    T, H, HKV, D = sum(n), c["H"], c["HKV"], c["D"]
    if c["kind"] == "append":
        return {"bytes": T * D * ((2 * H + 2 * HKV) * size[c["x"]] + 2 * HKV * size[c["kv"]]),
                "flops": 3 * T * (H + HKV) * c["rot"]}
    pairs = T * c["prefix"] + sum(k * l - k * (k - 1) // 2 for k, l in zip(n, lens))
    return {"bytes": 2 * T * H * D * size[c["q"]] + 4 * T * H + 2 * (c["prefix"] + sum(lens)) * HKV * D * size[c["kv"]],
            "flops": 4 * pairs * H * D}


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _append_exact, "attn": _attn_exact, "sample": _sample_exact}[case["kind"]](s)


def _sequences(s):
    """(first token, tokens, length of its own part, its pages) of every sequence."""
    lens, table = s["lens"].tolist(), s["table"].tolist()
    start = s["q_start"].tolist() if s["q_start"] is not None else list(range(len(lens) + 1))
    return [(start[b], start[b + 1] - start[b], lens[b], table[b][:-(-lens[b] // s["page"])]) for b in range(len(lens))]


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
        for x in (s["qs"], s["ks"]):
            y = x[t0:t0 + n].double().clone()
            z = torch.complex(y[..., first], y[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            done.append(y)
        page = torch.tensor(pages, device="cuda")[at // s["page"]]
        q_out[t0:t0 + n] = done[0]
        k_pages[page, at % s["page"]] = done[1]
        v_pages[page, at % s["page"]] = s["vs"][t0:t0 + n].double()
    return {"q": q_out, "k_pages": k_pages, "v_pages": v_pages}


def _attn_exact(s):
    """One sequence and one block of keys after another, with running sums."""
    H, HKV, D, P, page = s["H"], s["HKV"], s["D"], s["prefix"], s["page"]
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
        limit = P + length - n + torch.arange(n, device="cuda")  # the last key that each new token sees
        place = torch.arange(k.shape[1], device="cuda")
        kt = k.transpose(1, 2).contiguous()
        for g in range(G):
            q = s["qs"][t0:t0 + n, g::G].double().transpose(0, 1).contiguous()
            x = torch.bmm(q, kt) / D ** 0.5
            x = torch.where(place[None, None, :] <= limit[None, :, None], x, -math.inf)
            z = torch.logsumexp(x, -1)
            out[t0:t0 + n, g::G] = torch.bmm(torch.exp(x - z[..., None]), v.contiguous()).transpose(0, 1)
            lse[t0:t0 + n, g::G] = z.transpose(0, 1)
    return {"out": out, "lse": lse}


def _sample_exact(s):
    """Row by row on the host, with a sort by (logit, index)."""
    x = s["logits"].double().cpu().numpy()
    B, V = x.shape
    get = lambda name, off: np.full(B, off) if s[name] is None else s[name].double().cpu().numpy()  # noqa: E731
    t, k, p, mp, u = get("temperature", 1.0), get("top_k", 0), get("top_p", 1.0), get("min_p", 0.0), get("u", 0.0)
    logprob = np.zeros(B)
    for b in range(B):
        if t[b] <= 0:
            continue
        order = np.argsort(-x[b], kind="stable")
        if 0 < k[b] < V:
            order = order[:int(k[b])]
        w = np.exp((x[b][order] - x[b][order[0]]) / t[b])
        n = len(order)
        if p[b] < 1:
            n = max(1, int(np.searchsorted(np.cumsum(w), p[b] * w.sum())) + 1)
        chosen = np.arange(len(order)) < n
        chosen &= w >= mp[b]
        chosen[0] = True
        at = np.sort(order[chosen])
        w = np.exp((x[b][at] - x[b].max()) / t[b])
        c = np.cumsum(w)
        j = int(np.searchsorted(c, u[b] * c[-1], side="right"))
        logprob[b] = np.log(w[j] / c[-1])
    return {"token": None, "logprob": torch.from_numpy(logprob), "kept": None}
