"""bpd_pages_extend_gpu and bpd_pages_release_gpu against a pool that goes page by page (pages_oracle)."""
import numpy as np
import pytest
import torch

import pages_oracle as P
from bpd_substrate_amd import serve

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=dev)


class Both:
    """A pool on the device and its model, which every call compares."""

    def __init__(self, dev, n_pages, page, n_rows, width, reserved=0, windowed=False):
        self.dev, self.windowed = dev, windowed
        self.pool = serve.PagePool.empty(n_pages, page, n_rows, width, reserved, windowed, device=dev)
        self.model = P.Pool(n_pages, page, n_rows, width, reserved)
        self.same()

    def same(self):
        p, m = self.pool, self.model
        n = len(m.free)
        assert p.n_free.tolist() == [n, 0]
        assert p.free[:n].tolist() == m.free
        assert p.table.tolist() == m.table and p.lens.tolist() == m.lens
        if self.windowed:
            assert p.gone.tolist() == m.gone
        held = [x for row in m.table for x in row if x >= 0]
        assert len(set(held + m.free)) == len(held) + n, "a page is held twice"

    def extend(self, new, n_tokens, rows=None, prefix_len=0):
        step = self.pool.extend(i32(new, self.dev), n_tokens, rows=i32(rows, self.dev), prefix_len=prefix_len)
        want = self.model.extend(new, n_tokens, rows, prefix_len)
        for name in ("lens", "q_start", "slots", "pos", "refused"):
            assert getattr(step, name).tolist() == want[name], name
        assert rows is None or step.table.tolist() == want["table"]
        self.same()
        return want["refused"]

    def release(self, keep=None, rows=None, window=None, sinks=0):
        self.pool.release(i32(keep, self.dev), rows=i32(rows, self.dev), window=window, sinks=sinks)
        self.model.release(keep, rows, window, sinks)
        self.same()


@pytest.mark.parametrize("page,rows", [(1, True), (16, True), (21, True), (16, False), (64, False)])
def test_a_serving_loop(dev, page, rows):
    """Prompts, steps of a few tokens, drafts that are rejected and sequences that end, in any order."""
    r = np.random.default_rng(page)
    R, width = 37, 300 // page + 2
    b = Both(dev, 37 * width // 2, page, R, width, reserved=2)
    for step in range(25):
        B = int(r.integers(1, R + 1))
        pick = [int(x) for x in r.permutation(R)[:B]] if rows else None
        new = [int(x) for x in r.choice([0, 1, 1, 4, 40, 150], B)]
        b.extend(new, int(r.choice([sum(new), sum(new) + 5, max(0, sum(new) - 30)])), pick, prefix_len=7)
        lens = b.model.lens if pick is None else [b.model.lens[x] for x in pick]
        keep = [int(r.choice([n, max(0, n - 3), n // 2, 0, n + 9])) for n in lens[:B]]
        b.release(keep, pick)
        if step % 7 == 6:
            b.release([0] * R)


def test_release_undoes_extend(dev):
    b = Both(dev, 100, 4, 8, 12)
    b.extend([5, 9, 0, 31], 45, [3, 1, 0, 6])
    before = b.pool.free.tolist(), b.pool.table.tolist()
    b.extend([4, 4, 4], 12, [6, 0, 3])
    b.release([31, 0, 5], [6, 0, 3])
    assert (b.pool.free.tolist(), b.pool.table.tolist()) == before


def test_what_is_refused(dev):
    b = Both(dev, 10, 4, 9, 5)
    rows = [0, 9, 1, 1, 2, -1, 3, 4, 5, 6]
    assert b.extend([8, 1, 12, 3, -1, 2, 21, 25, 7], 100, rows[:9]) == [0, 1, 0, 1, 1, 1, 2, 2, 0]
    # 7 pages are held, 3 left.  Four are too many, none is not, and who asks for one behind those four has to wait
    assert b.extend([16, 4, 0, 1, 1], 100, [6, 7, 8, 5, 1]) == [3, 3, 0, 0, 3]
    assert b.extend([1, 1, 1], 2, [2, 3, 4]) == [0, 0, 4]


def test_more_tokens_than_there_is_room_for(dev):
    b = Both(dev, 50, 4, 6, 5)
    assert b.extend([5, 5, 5, 0, 1], 12, [0, 1, 2, 3, 4]) == [0, 0, 4, 4, 4]
    b.release([0, 0], [0, 1])


@pytest.mark.parametrize("sinks", [0, 4, 33])
def test_pages_slide_out_of_a_window(dev, sinks):
    """The pages that the tokens to come still see are those that the attention reads."""
    r = np.random.default_rng(sinks)
    page, window, R = 8, 50, 5
    b = Both(dev, 300, page, R, 60, windowed=True)
    for step in range(30):
        pick = [int(x) for x in r.permutation(R)[:int(r.integers(1, R + 1))]]
        new = [int(x) for x in r.choice([1, 1, 5, 60], len(pick))]
        b.extend(new, 10000, pick)
        keep = [b.model.lens[x] - (int(r.choice([0, 2])) if k > 1 else 0) for x, k in zip(pick, new)]
        b.release(keep, pick, window, sinks)
        for x in pick:
            n = b.model.lens[x]
            for i in range(P.used(n, page)):
                rows = range(i * page, min(n, (i + 1) * page))
                seen = any(j > n - window or j < sinks for j in rows)
                assert (b.model.table[x][i] >= 0) == (seen or i < P.used(sinks, page))
        if step % 10 == 9:
            b.release([0] * len(pick), pick, window, sinks)
    b.release([0] * R, None)
    assert len(b.model.free) == 300


def test_more_sequences_than_a_workgroup_has_threads(dev):
    r = np.random.default_rng(5)
    b = Both(dev, 20000, 4, 2500, 9)
    rows = [int(x) for x in r.integers(-1, 2501, 2500)]            # some twice, some none
    b.extend([int(x) for x in r.integers(0, 30, 2500)], 40000, rows)
    b.release([int(x) for x in r.integers(0, 30, 2500)], rows)
    b.extend([int(x) for x in r.integers(0, 9, 2500)], 3000)
    b.release()


def test_the_largest_pool(dev):
    b = Both(dev, 20000, 4, 16384, 3)
    r = np.random.default_rng(6)
    rows = [int(x) for x in r.permutation(16384)[:700]]
    b.extend([int(x) for x in r.integers(0, 9, 700)], 5000, rows)
    b.release([int(x) for x in r.integers(0, 5, 700)], rows)
    b.extend([1] * 16384, 16384)
    b.release([0] * 16384)


def test_one_long_sequence_and_empty_calls(dev):
    b = Both(dev, 5000, 16, 3, 4400)
    b.extend([0, 70000, 1], 70001, [2, 1, 0])
    b.release([69990], [1])
    step = b.pool.extend(i32([], dev), 3, rows=i32([], dev))
    assert step.q_start.tolist() == [0] and step.slots.tolist() == step.pos.tolist() == [-1] * 3
    b.release([], [])
    b.same()


def test_the_widest_table(dev):
    """A step of the threads past its end is beyond 2^31."""
    n_tokens = 4
    W = 2 ** 31 - 1025 - n_tokens
    pool = serve.PagePool.empty(100, 1, 1, W, device=dev)
    step = pool.extend(i32([n_tokens], dev), n_tokens, rows=i32([0], dev))
    assert step.refused.tolist() == [0] and step.pos.tolist() == list(range(n_tokens))
    for table in (step.table, pool.table):
        assert table[0, :n_tokens].tolist() == step.slots.tolist() and sorted(set(step.slots.tolist())) == sorted(step.slots.tolist())
        assert int(table[0, n_tokens:].max()) == -1 and int(table[0, n_tokens:].min()) == -1
    pool.release(i32([0], dev))
    assert pool.n_free.tolist() == [100, 0] and sorted(pool.free.tolist()) == list(range(100))
    assert int(pool.table.max()) == -1
    pool.lens.fill_(W)   # more than the pool has: the whole table is gone through
    pool.release(i32([0], dev))
    assert pool.n_free.tolist() == [100, 0] and pool.lens.tolist() == [0] and int(pool.table.max()) == -1


def test_pools_of_any_content_stay_inside(dev):
    """Lengths, counts and pages that no pool has: every access stays in the tensors."""
    big = 2 ** 31 - 1
    z = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
    guard = torch.full((64,), 77, dtype=torch.int32, device=dev)
    for lens, n_free, gone in (([big, -5, 7], 99, [[3, 2], [-4, big], [1, 2]]), ([-big, 3, big], -3, [[big, -1], [0, 0], [2, 1]]),
                               ([12, 12, 12], big, [[0, 3], [5, 9], [0, 1]])):
        free = torch.tensor([5, -1, big, 2], dtype=torch.int32, device=dev)
        pool = serve.PagePool(z(3, 4) + big, i32(lens, dev), free, i32([n_free, 0], dev), 4, gone=i32(gone, dev))
        step = pool.extend(i32([3, 2, 1], dev), 6, rows=i32([2, 0, 1], dev))
        pool.release(i32([1, big, -2], dev), rows=i32([1, 0, 2], dev), window=3, sinks=1)
        pool.release(window=1)
        torch.cuda.synchronize()
        assert 0 <= int(pool.n_free[0]) <= 4 and (step.slots < 16).all() and (guard == 77).all()


def test_a_replayed_graph_hands_out_other_pages_each_time(dev):
    b = Both(dev, 400, 4, 6, 40)
    new, rows, keep = i32([3, 1, 2], dev), i32([4, 0, 2], dev), i32([200, 200, 200], dev)
    b.extend([3, 1, 2], 6, [4, 0, 2])
    b.release([200] * 3, [4, 0, 2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        step = b.pool.extend(new, 8, rows=rows)
        b.pool.release(keep, rows=rows)
    for n in ([3, 1, 2], [0, 5, 3], [9, 0, 1], [1, 1, 1]):
        new.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = b.model.extend(n, 8, [4, 0, 2])
        b.model.release([200] * 3, [4, 0, 2])
        for name in ("table", "lens", "q_start", "slots", "pos", "refused"):
            assert getattr(step, name).tolist() == want[name], name
        b.same()


def test_the_step_is_a_batch(dev):
    """Appending by the pool's batch writes the rows that the slots name."""
    pool = serve.PagePool.empty(40, 8, 5, 9, reserved=3, device=dev)
    cache = serve.PagedCache.empty(40, 8, 2, 64, torch.float16, device=dev)
    prefix = i32([2, 0], dev)
    step = pool.extend(i32([5, 0, 20], dev), 27, rows=i32([4, 1, 3], dev), prefix_len=11)
    k = torch.randn(27, 2, 64, device=dev).half()
    serve.rope_append(cache, step.batch(prefix), None, k, k)
    rows = cache.k.reshape(40 * 8, 2, 64) if cache.k.is_contiguous() else cache.k.contiguous().view(320, 2, 64)
    slots = step.slots.long()
    assert torch.equal(rows[slots[:25]], k[:25]) and slots[25:].tolist() == [-1, -1]
    assert (rows.abs().sum((1, 2)) > 0).sum() == 25 and step.pos[:25].tolist() == [*range(11, 16), *range(11, 31)]
