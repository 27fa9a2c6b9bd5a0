"""Host replay of the index arithmetic of the paged kernels (csrc/paged_attn.hip, bpdq_paged.h): shares of units,
places of partial results, the search for a token's sequence, divisions by the page size.  It mirrors the
formulas there; a change there must be mirrored here.  No GPU."""
import numpy as np
import pytest


def unit_of(w, U, n):
    return w * U // n


def group_of(u, U, n):
    return ((u + 1) * n - 1) // U


@pytest.mark.parametrize("U,groups", [(1, 256), (5, 256), (255, 256), (256, 256), (257, 256), (1000, 256), (99991, 256),
                                      (41000, 2048), (2047, 2048), (3, 8)])
def test_shares_hold_every_unit_once_and_are_found_again(U, groups):
    n = min(U, groups)
    start = [unit_of(w, U, n) for w in range(n + 1)]
    assert start[0] == 0 and start[n] == U and all(a < b for a, b in zip(start, start[1:]))
    for u in list(range(min(U, 2000))) + list(range(max(0, U - 2000), U)):
        w = group_of(u, U, n)
        assert 0 <= w < n and start[w] <= u < start[w + 1]


@pytest.mark.parametrize("seed", range(8))
def test_places_of_results_differ_and_fit(seed):
    """share + head * items + item over all (share, head, item) that meet; the results of one pair are in a row, from
    the place that its first share gives, as many as k_attn_join is told."""
    r = np.random.default_rng(seed)
    items, hkv, groups = int(r.integers(1, 40)), int(r.integers(1, 9)), int(r.choice([8, 64, 256]))
    nk = r.integers(0, 30, items)          # units of each item, some none
    first = np.concatenate([[0], np.cumsum(nk)])
    UH = int(first[-1])
    if UH == 0:
        return
    U = UH * hkv
    n = min(U, groups)
    seen, of = set(), {}
    for w in range(n):
        u, u1 = unit_of(w, U, n), unit_of(w + 1, U, n)
        while u < u1:
            head, at = divmod(u, UH)
            item = int(np.searchsorted(first[:items], at, side="right")) - 1     # count_le - 1: the last that starts there
            assert first[item] <= at < first[item + 1]
            kt = at - first[item]
            k1 = min(nk[item], kt + u1 - u)
            place = w + head * items + item
            assert place not in seen and place < groups + items * hkv
            seen.add(place)
            of.setdefault((head, item), []).append(place)
            if kt == 0:
                count = group_of(head * UH + int(first[item]) + int(nk[item]) - 1, U, n) - w + 1
                of[(head, item, "told")] = (place, count)
            u += k1 - kt
    for (head, item) in [k for k in of if len(k) == 2]:
        place, count = of[(head, item, "told")]
        assert of[(head, item)] == list(range(place, place + count))
    assert len([k for k in of if len(k) == 2]) == hkv * int((nk > 0).sum())


def count_le(p, n, t):
    lo, hi, reads = 0, n, []
    while lo < hi:
        step = (hi - lo + 63) >> 6
        c = 0
        for lane in range(64):
            i = lo + lane * step
            reads.append(i if i < hi else lo)
            c += i < hi and p[i if i < hi else lo] <= t
        if c == 0:
            return lo, reads
        if step == 1:
            return lo + c, reads
        hi, lo = min(hi, lo + c * step), lo + (c - 1) * step + 1
    return lo, reads


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 129, 4095, 4097, 70000])
def test_search_for_a_sequence(n):
    r = np.random.default_rng(n)
    p = np.sort(r.integers(0, max(2, n // 2), n))
    for t in [-1, 0, int(p[-1]), int(p[-1]) + 1] + [int(x) for x in r.integers(0, n, 20)]:
        got, reads = count_le(p, n, t)
        assert got == np.searchsorted(p, t, side="right") and 0 <= min(reads, default=0) and max(reads, default=0) < n
    q = r.integers(-2 ** 31, 2 ** 31 - 1, n)     # offsets that decrease: some count in range, nothing read beyond
    for t in [0, 5, 2 ** 30]:
        got, reads = count_le(q, n, t)
        assert 0 <= got <= n and 0 <= min(reads) and max(reads) < n


@pytest.mark.parametrize("d", [1, 2, 3, 5, 7, 16, 21, 63, 64, 100, 4096, 65537, 2 ** 30, 2 ** 31 - 1])
def test_division_by_the_page_size(d):
    s = 0
    while (1 << s) < d:
        s += 1
    m = ((1 << 32) * ((1 << s) - d)) // d + 1
    assert m < 1 << 32
    r = np.random.default_rng(d)
    for n in [0, 1, d - 1, d, min(d + 1, 2 ** 31 - 1), 2 ** 31 - 1] + [int(x) for x in r.integers(0, 2 ** 31 - 1, 300)]:
        hi = (m * n) >> 32
        assert hi + n < 1 << 32 and (hi + n) >> s == n // d


@pytest.mark.parametrize("DT", [64, 128, 256])
def test_lds_slots_meet_every_bank_once(DT):
    """K's operand read: 16 lanes, a row each, one chunk: 16 different 16-byte places of the 64 banks.  V's transposing
    read: 16 rows, two chunks each: every 32-byte place twice, as the read takes two rounds."""
    cpr = DT // 8
    k_slot = lambda row, c: c ^ ((row >> 1) & 7) if DT == 64 else c ^ (row & 15)  # noqa: E731
    v_slot = lambda row, c: c ^ (((row >> 1) & 3) << 1) if DT == 64 else c ^ ((row & 7) << 1)  # noqa: E731
    for c in range(cpr):
        places = [(row * cpr + k_slot(row, c)) % 16 for row in range(16)]
        assert sorted(places) == list(range(16))
    for e in range(DT // 16):
        pairs = [((row * cpr + v_slot(row, 2 * e)) % 16) // 2 for row in range(16)]
        assert sorted(pairs) == sorted(list(range(8)) * 2)
        assert all(v_slot(row, 2 * e + 1) == v_slot(row, 2 * e) ^ 1 for row in range(16))
    for row in range(64):
        for f in (k_slot, v_slot):
            assert sorted(f(row, c) for c in range(cpr)) == list(range(cpr))


def seq_tokens(q_start, b, T):
    t0 = min(max(q_start[b], 0), T)
    return t0, max(min(max(q_start[b + 1], 0), T) - t0, 0)


@pytest.mark.parametrize("seed", range(60))
def test_plan_of_any_offsets_stays_inside(seed):
    """k_attn_plan's arrays and what k_attn_tile and k_attn_join read of them, for offsets of any kind."""
    r = np.random.default_rng(seed)
    B, T, G, R, P = int(r.integers(1, 12)), int(r.integers(1, 300)), int(r.choice([1, 2, 5, 8, 40])), int(r.choice([64, 128])), 70
    kind = seed % 3
    if kind == 0:
        q_start = np.sort(r.integers(0, T + 1, B + 1))
    elif kind == 1:
        q_start = r.integers(-T, 2 * T, B + 1)
    else:
        q_start = r.choice([-2 ** 31, -1, 0, T // 2, T, 2 ** 31 - 1], B + 1)
    q_start = [int(x) for x in q_start]
    own = [int(x) for x in r.integers(0, 200, B)]
    ntp, size = (P + 63) // 64, 2 * (T * G // R + 1) + B     # the workspace's items
    joint = lambda n: n * G * 2 >= R  # noqa: E731
    packed, place, n_packed = {}, {}, 0
    for b in range(B):
        t0, n = seq_tokens(q_start, b, T)
        if n > 0 and not joint(n):
            for i in range(n):
                k = n_packed + i
                if k < T:
                    packed[k] = t0 + i
                assert 0 <= t0 + i < T
                place[t0 + i] = k if k < T else -1
            n_packed = min(n_packed + n, T)
    np_ = -(-n_packed * G // R)
    most = np_ + B + T * G // R
    seq, rt, item0, items = [-1] * np_, list(range(np_)), [], np_
    for b in range(B):
        t0, n = seq_tokens(q_start, b, T)
        item0.append(items)
        for k in range(-(-n * G // R)):
            if items < most:
                seq.append(b)
                rt.append(k)
                items += 1
    assert items <= size and len(seq) == items
    if kind == 0:
        assert items - np_ == sum(-(-seq_tokens(q_start, b, T)[1] * G // R) for b in range(B))   # none is cut off
    first = [i * ntp for i in range(np_)]
    units = np_ * ntp
    for k in range(np_, items):
        t0, n = seq_tokens(q_start, seq[k], T)
        assert n > 0 and rt[k] * R < n * G
        first.append(units)
        units += (ntp if joint(n) else 0) + (own[seq[k]] + 63) // 64
    first.append(units)
    for k in range(items):                    # the tile's rows
        t0, n = (0, n_packed) if seq[k] < 0 else seq_tokens(q_start, seq[k], T)
        for row in range(rt[k] * R, (rt[k] + 1) * R):
            i = row // G
            if i < n:
                assert 0 <= (packed[i] if seq[k] < 0 else t0 + i) < T
    for t in range(T):                        # the join's
        b = count_le(np.array(q_start), B + 1, t)[0] - 1
        if b < 0 or b >= B:
            continue
        t0, n = seq_tokens(q_start, b, T)
        i = t - t0
        if i < 0 or i >= n:
            continue
        for gq in range(G):
            if not joint(n):
                at = place[t]                 # set by this sequence, if by no other
                assert at < T
                if at >= 0:
                    assert (at * G + gq) // R < np_
            item = item0[b] + (i * G + gq) // R
            assert item >= 0
            if item < items:
                assert seq[item] == b and first[item + 1] >= first[item]
