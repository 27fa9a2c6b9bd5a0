"""The operators of a serving step together, as a loop calls them: pages, normed append, attention over a window,
adjusted logits, sampling, pages back.  Every output against a plain float64 form of what the caches and histories hold."""
import threading

import numpy as np
import pytest
import torch

import paged_oracle as O
from bpd_substrate_amd import gpu, serve
from test_gpu_adjust import plain as adjusted

pytestmark = pytest.mark.gpu

H, HKV, D, PAGE, V = 8, 2, 64, 16, 1000


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Loop:
    """Users that come and go, behind a prefix of `P` rows, with a window and first rows that stay."""

    def __init__(self, dev, seed, P=20, window=40, sinks=25, users=6):
        self.dev, self.P, self.W, self.S = dev, P, window, sinks
        self.g = torch.Generator(device=dev).manual_seed(seed)
        self.r = np.random.default_rng(seed)
        npre = -(-P // PAGE)
        self.pool = serve.PagePool.empty(60, PAGE, users, 40, reserved=npre, windowed=True, device=dev)
        self.cache = serve.PagedCache.empty(60, PAGE, HKV, D, torch.bfloat16, device=dev)
        self.prefix = i32(list(range(npre)), dev) if P else None
        if P:
            c = self.cache
            for x in (c.k, c.v):
                x[:npre] = torch.randn(npre, PAGE, HKV, D, generator=self.g, device=dev).bfloat16()
        self.rope = serve.Rope(D, neox=True, device=dev)
        self.qw, self.kw = (1 + 0.2 * torch.randn(D, generator=self.g, device=dev) for _ in range(2))
        self.slots = [[] for _ in range(users)]    # of every row of a user, as extend gave them
        self.tokens = torch.full((users, 400), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(users, dtype=torch.int32, device=dev)

    def step(self, rows, new):
        dev, T = self.dev, sum(new) + 3
        rows_d, new_d = i32(rows, dev), i32(new, dev)
        step = self.pool.extend(new_d, T, rows=rows_d, prefix_len=self.P)
        batch = step.batch(self.prefix)
        x = torch.randn(T, H + 2 * HKV, D, generator=self.g, device=dev).bfloat16()
        q = serve.rope_append(self.cache, batch, x[:, :H], x[:, H:H + HKV], x[:, H + HKV:], rope=self.rope, q_norm=self.qw,
                              k_norm=self.kw)
        out = serve.attention(self.cache, batch, q, window=self.W, sinks=self.S)
        logits = 3 * torch.randn(len(rows), V, generator=self.g, device=dev)
        rule = dict(tokens=self.tokens[rows_d.long()], lens=self.lens[rows_d.long()],
                    repetition=torch.full((len(rows),), 1.3, device=dev), presence=torch.full((len(rows),), 0.5, device=dev),
                    mask=torch.randint(-2 ** 31, 2 ** 31, (2, 32), generator=self.g, device=dev).int(),
                    mask_row=i32([b % 3 - 1 for b in range(len(rows))], dev))
        y = serve.adjust_logits(logits, **rule)
        u = torch.rand(len(rows), generator=self.g, device=dev)
        token, logprob, kept = serve.sample(y, u, top_k=i32([20] * len(rows), dev))
        self.check(step, rows, new, q, out, logits, rule, y, u, token, logprob, kept)
        for b, row in enumerate(rows):
            self.tokens[row, self.lens[row]] = token[b]
            self.lens[row] += 1

    def check(self, step, rows, new, q, out, logits, rule, y, u, token, logprob, kept):
        assert step.refused.tolist() == [0] * len(rows)
        slots, start = step.slots.tolist(), step.q_start.tolist()
        k, v = (O.f64(c).reshape(-1, HKV, D) for c in (self.cache.k, self.cache.v))
        q, out = O.f64(q), O.f64(out)
        pre = list(range(self.P))
        for b, row in enumerate(rows):
            mine = self.slots[row]
            for t in range(start[b], start[b + 1]):
                mine.append(slots[t])
                p = self.P + len(mine) - 1
                assert int(step.pos[t]) == p
                at = [s for j, s in enumerate(pre + mine) if j > p - self.W or j < self.S]
                for h in range(H):
                    kh, vh = k[at, h // (H // HKV)], v[at, h // (H // HKV)]
                    s = kh @ q[t, h] / D ** 0.5
                    w = np.exp(s - s.max())
                    ref = w @ vh / w.sum()
                    # paged_oracle's bound: scores, weights rounded to bf16, sums, and the result rounded once
                    a = (np.abs(kh) @ np.abs(q[t, h])).max() / D ** 0.5
                    ds = (D + 6) * 2.0 ** -24 * (a + 2 * np.abs(s).max()) + 2.0 ** -22
                    spread = w @ np.abs(vh) / w.sum()
                    bound = 2.0 ** -8 * np.abs(ref) + spread * (2 * ds + 2 * 2.0 ** -8 + 2 * (len(at) + 8) * 2.0 ** -24) + 2.0 ** -25
                    assert (np.abs(out[t, h] - ref) <= bound).all()
        host = {n: x.cpu().numpy() for n, x in rule.items()}
        ref, err = adjusted(O.f64(logits), host["tokens"], host["lens"], None, host["repetition"], None, host["presence"], None,
                            host["mask"], host["mask_row"])
        got = O.f64(y)
        inf = np.isinf(ref)
        assert np.array_equal(np.isinf(got), inf) and (np.abs(got - ref)[~inf] <= err[~inf]).all()
        for b in range(len(rows)):
            O.check_sample(got[b], int(token[b]), float(logprob[b]), int(kept[b]), float(u[b]), top_k=20)

    def keep(self, rows, drop):
        """The last `drop` rows of each are rejected, and what no token to come sees goes back."""
        for row, n in zip(rows, drop):
            del self.slots[row][len(self.slots[row]) - n:]
        self.pool.release(i32([len(self.slots[r]) for r in rows], self.dev), rows=i32(rows, self.dev), window=self.W,
                          sinks=self.S, prefix_len=self.P)

    def leave(self, row):
        self.slots[row] = []
        self.pool.release(i32([0], self.dev), rows=i32([row], self.dev), window=self.W, sinks=self.S, prefix_len=self.P)
        self.lens[row] = 0


@pytest.mark.parametrize("P,sinks", [(20, 25), (0, 4), (70, 0)])
def test_a_serving_loop(dev, P, sinks):
    loop = Loop(dev, P + sinks, P=P, sinks=sinks)
    loop.step([0, 3, 5], [30, 1, 60])
    loop.keep([0, 3, 5], [0, 0, 0])
    for i in range(12):
        rows = [int(x) for x in loop.r.permutation(6)[:4]]
        new = [int(x) for x in loop.r.choice([1, 1, 4, 33], 4)]
        loop.step(rows, new)
        loop.keep(rows, [2 if n == 4 else 0 for n in new])
        if i % 4 == 3:
            loop.leave(rows[0])
    held = loop.pool.table[loop.pool.table >= 0].tolist() + loop.pool.free[:int(loop.pool.n_free[0])].tolist()
    assert sorted(held) == list(range(-(-P // PAGE), 60)), "pages were lost or held twice"


def state_of(loop):
    p, c = loop.pool, loop.cache
    return [p.table, p.lens, p.gone, p.free, p.n_free, c.k, c.v]


def captured_step(dev, loop, new, rows, x, logits, u, keep):
    step = loop.pool.extend(new, 8, rows=rows, prefix_len=loop.P)
    batch = step.batch(loop.prefix)
    q = serve.rope_append(loop.cache, batch, x[:, :H], x[:, H:H + HKV], x[:, H + HKV:], rope=loop.rope, q_norm=loop.qw,
                          k_norm=loop.kw)
    out = serve.attention(loop.cache, batch, q, window=loop.W, sinks=loop.S)
    y = serve.adjust_logits(logits, tokens=loop.tokens[:2], lens=loop.lens[:2], repetition=u + 1)
    token, _, _ = serve.sample(y, u)
    loop.pool.release(keep, rows=rows, window=loop.W, sinks=loop.S, prefix_len=loop.P)
    return out, token, step.slots


def test_a_captured_step_follows_its_inputs(dev):
    """Replayed several times, with eager work between: each replay gives what the same step gives eagerly."""
    loop = Loop(dev, 3)
    loop.step([0, 1], [40, 7])
    new, rows, keep = i32([1, 2], dev), i32([1, 0], dev), i32([300, 300], dev)
    x = torch.randn(8, H + 2 * HKV, D, device=dev).bfloat16()
    logits, u = torch.randn(2, V, device=dev), torch.rand(2, device=dev)
    args = (dev, loop, new, rows, x, logits, u, keep)
    captured_step(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        got = captured_step(*args)
    from test_gpu_serve_graphs import KERNEL, nodes
    kinds, edges = nodes(graph)
    assert kinds == [KERNEL] * len(kinds) and edges == [(i, i + 1) for i in range(len(kinds) - 1)]
    for n in ([1, 2], [3, 0], [0, 5], [1, 1], [2, 2]):
        new.copy_(torch.tensor(n, dtype=torch.int32))
        x.normal_()
        logits.normal_()
        u.uniform_()
        before = [t.clone() for t in state_of(loop)]
        want = [t.clone() for t in captured_step(*args)]
        after = [t.clone() for t in state_of(loop)]
        for t, s in zip(state_of(loop), before):
            t.copy_(s)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        tokens = sum(n)
        assert torch.equal(got[0][:tokens], want[0][:tokens]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
        assert all(torch.equal(a, b) for a, b in zip(state_of(loop), after))


def calls(dev, seed):
    """One call of each operator on tensors of its own, each giving a tensor."""
    b = O.Batch(seed, [1] * 6, [90, 20, 333, 1, 64, 50], 30, 8, 2, 64, "f16", "f16", 16, decode=True)
    c = O.Batch(seed + 1, [70, 3], [90, 200], 30, 8, 2, 64, "f16", "f16", 16)
    w = torch.rand(64, device=dev)
    rope = serve.Rope(64, device=dev)
    parts = [x.device(dev) for x in (b, c, O.Batch(seed + 2, [1] * 6, [9] * 6, 30, 8, 2, 64, "f16", "f16", 16))]
    k = torch.randn(6, 2, 64, device=dev).half()
    logits, tok = torch.randn(6, 5000, device=dev), torch.randint(0, 5000, (6, 700), device=dev).int()
    r = torch.rand(6, device=dev) + 1
    pool = serve.PagePool.empty(200, 16, 6, 20, device=dev)
    new, none = i32([30, 5, 17, 0, 100, 1], dev), i32([0] * 6, dev)

    def pages():
        step = pool.extend(new, 160)
        out = torch.cat([step.slots, step.pos, step.q_start, step.lens])
        pool.release(none)
        return out

    return [lambda: serve.attention(*parts[0], window=60, sinks=5), lambda: serve.attention(*parts[1], window=60, sinks=5),
            lambda: serve.rope_append(*parts[2], k, k, rope=rope, q_norm=w, k_norm=w),
            lambda: serve.adjust_logits(logits, tokens=tok, repetition=r, frequency=r), pages]


def test_on_streams_of_their_own_side_by_side(dev):
    """Threads with a stream each: every call gives what it gives alone."""
    work = calls(dev, 40)
    want = [f() for f in work]
    torch.cuda.synchronize()
    wrong, ready = [], threading.Barrier(len(work))

    def go(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            ready.wait()
            for _ in range(60):
                got = work[i]()
                st.synchronize()
                if not torch.equal(got, want[i]):
                    wrong.append(i)

    ts = [threading.Thread(target=go, args=(i,)) for i in range(len(work))]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not wrong


def test_calls_leave_the_launch_stream_alone(dev):
    x, y = torch.zeros(64, device=dev), torch.zeros(64, device=dev)
    mine, other = torch.cuda.Stream(), torch.cuda.Stream()
    for call in calls(dev, 50):
        call()
        y.zero_()
        torch.cuda.synchronize()
        gpu.call("bpd_gpu_set_stream", mine.cuda_stream)
        try:
            with torch.cuda.stream(mine):
                torch.cuda._sleep(500_000_000)
            call()
            gpu.call("bpd_expf_gpu", x, y, 64)     # on `mine`, behind the sleep
            with torch.cuda.stream(other):
                seen = y.clone()
            other.synchronize()
            assert not mine.query(), "the sleep was over too early to tell"
            assert (seen == 0).all()
            mine.synchronize()
            assert (y == 1).all()
        finally:
            gpu.call("bpd_gpu_set_stream", 0)


def test_two_graphs_that_replay_side_by_side(dev):
    """Chunks need a workspace: each graph has one of its own."""
    f, g = calls(dev, 60)[1], calls(dev, 70)[1]
    want = f(), g()
    torch.cuda.synchronize()
    made = []
    for h in (f, g):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            out = h()
        made.append((graph, out, torch.cuda.Stream()))
    for _ in range(20):
        for graph, out, st in made:
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, w) for (_, out, _), w in zip(made, want))
