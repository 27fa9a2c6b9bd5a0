"""The forms of the windowed attention that need a workspace (tiles that are planned, units dealt to all waves), where
few tokens stand before many rows, against window_oracle."""
import threading

import pytest
import torch

from bpd_substrate_amd import serve
from test_gpu_serve_graphs import KERNEL, nodes
from test_gpu_window import DEALT, TILES, check
from window_oracle import Batch

pytestmark = pytest.mark.gpu


def needs_workspace(b, dev, window, sinks):
    cache, batch, q = b.device(dev)
    return batch._workspace(cache, q.dtype, q.shape[1], window, sinks) > 0


# new tokens, own rows, prefix, H, HKV, D, q, kv, page, heads_first, padding rows; window, sinks
FEW = [
    (([1], [9000], 0, 8, 2, 128, "bf16", "bf16", 64, True, 0), (8500, 4)),
    (([4], [8301], 61, 10, 2, 64, "f16", "f16", 16, False, 1), (7000, 70)),
    (([4, 0, 1], [6300, 20, 700], 0, 12, 4, 96, "f32", "f16", 21, False, 0), (5000, 3)),
    (([2, 3], [40, 4600], 100, 6, 2, 256, "bf16", "bf16", 32, True, 0), (4100, 0)),
    (([1, 1], [7000, 6999], 0, 4, 2, 80, "f32", "bf16", 16, True, 2), (2 ** 31 - 1, 0)),
]


@pytest.mark.parametrize("slide", [False, True])
@pytest.mark.parametrize("case", range(len(FEW)))
def test_few_tokens_before_many_rows(dev, case, slide):
    args, win = FEW[case]
    b = Batch(900 + case, *args)
    if slide:
        b.slide(*win)
    assert needs_workspace(b, dev, *win)
    check(b, dev, *win)


# one token each, of sequences of which one is long: its units go to all waves
LONG = [
    (([1] * 17, [30] * 9 + [4800] + [1, 2, 64, 0, 700, 33, 32], 0, 16, 8, 128, "bf16", "bf16", 64, True, 0), (4500, 4)),
    (([1] * 65, [40] * 64 + [4300], 50, 4, 2, 64, "f32", "f16", 16, False, 0), (4200, 60)),
    (([1] * 65, [4700] + [3] * 64, 0, 4, 2, 256, "f16", "f16", 32, True, 0), (2 ** 31 - 1, 0)),
]


@pytest.mark.parametrize("slide", [False, True])
@pytest.mark.parametrize("case", range(len(LONG)))
def test_one_long_sequence_among_many(dev, case, slide):
    args, win = LONG[case]
    b = Batch(920 + case, *args, decode=True)
    if slide:
        b.slide(*win)
    assert needs_workspace(b, dev, *win)
    check(b, dev, *win)


# ---------------------------------------------------------------- workspaces of calls side by side

SIDE = [(TILES[1], False), (TILES[4], False), (DEALT[0], True), (DEALT[2], True), (FEW[2], False), (LONG[1], True)]


def calls(dev, seed):
    """Calls on tensors of their own, all with a workspace; (out, lse) of each."""
    made = []
    for i, ((args, win), decode) in enumerate(SIDE):
        b = Batch(seed + i, *args, decode=decode)
        assert needs_workspace(b, dev, *win)
        cache, batch, q = b.device(dev)
        out = torch.zeros_like(q)   # rows of no sequence stay

        def call(cache=cache, batch=batch, q=q, out=out, win=win):
            return serve.attention(cache, batch, q, out=out, return_lse=True, window=win[0], sinks=win[1])

        named = slice(int(b.start[0]), int(b.start[-1]))
        made.append((call, lambda r, named=named: torch.cat([r[0][named].float().flatten(), r[1][named].flatten()])))
    return made


def test_on_streams_of_their_own_side_by_side(dev):
    work = calls(dev, 940)
    want = [get(f()).clone() for f, get in work]
    torch.cuda.synchronize()
    wrong, ready = [], threading.Barrier(len(work))

    def go(i):
        f, get = work[i]
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            ready.wait()
            for _ in range(40):
                got = get(f())
                st.synchronize()
                if not torch.equal(got, want[i]):
                    wrong.append(i)

    ts = [threading.Thread(target=go, args=(i,)) for i in range(len(work))]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not wrong


def test_graphs_that_replay_side_by_side(dev):
    """Each has a workspace of its own, is kernels alone, and gives what the call gives eagerly, also with eager calls
    between the replays."""
    work = calls(dev, 960)
    want = [get(f()).clone() for f, get in work]
    torch.cuda.synchronize()
    made = []
    for f, get in work:
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            got = f()
        kinds, edges = nodes(graph)
        assert len(kinds) >= 2 and kinds == [KERNEL] * len(kinds) and edges == [(i, i + 1) for i in range(len(kinds) - 1)]
        made.append((graph, got, torch.cuda.Stream()))
    for turn in range(12):
        for (out, _) in (m[1] for m in made):
            out.zero_()
        torch.cuda.synchronize()
        for graph, _, st in made:
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(get(got), w) for (_, got, _), (_, get), w in zip(made, work, want))
        if turn % 3 == 2:
            assert all(torch.equal(get(f()), w) for (f, get), w in zip(work, want))
            torch.cuda.synchronize()
