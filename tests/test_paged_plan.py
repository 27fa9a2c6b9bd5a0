"""The index arithmetic of the paged kernels as they include it (csrc/bpdq_paged_plan.h), compiled for the CPU: values
against exact integers up to the limits that the entry points allow, and every place that a batch's results and
plan take against the workspace that the library asks for.  No GPU."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from bpd_substrate_amd import _native, build
from test_serve_host import batch, cache

SRC = r"""
#include "bpdq_paged_plan.h"
using namespace bpdq;
extern "C" {
int t_div(int d, int n) { return fdiv(fast_div(d), n); }
int t_units(int v) { return units_of(v); }
long long t_slot(int w, int item, int n, int h) { return slot_of(w, item, n, h); }
long long t_unit(int w, long long U, int n) { return unit_of(w, U, n); }
int t_group(long long u, long long U, int n) { return group_of(u, U, n); }
int t_joint(int n, int G, int R) { return is_joint(n, G, R); }
int t_clamp(int s, int e, int T, int* n) { int t0; clamp_tokens(s, e, T, t0, *n); return t0; }
int t_rows(int D, int parts) { return rows_of(D, parts); }
int t_padded(int D) { return padded(D); }
void t_sizes(int planned, int B, int T, int G, int HKV, int R, int DT, int P, long long* out) {
    const Sizes s = sizes(planned != 0, B, T, G, HKV, R, DT, P);
    const long long v[] = {s.items, s.ints, s.part, s.ml, s.where, s.part1, s.ml1, s.where1, s.total};
    for (int i = 0; i < 9; i++) out[i] = v[i];
}
int t_groups() { return kGroups; }
int t_waves() { return kStreamWaves; }
}
"""
TOP = (1 << 31) - 1025     # rows and tokens of a call add up to this at most


@pytest.fixture(scope="module")
def C(tmp_path_factory):
    d = str(tmp_path_factory.mktemp("plan"))
    src, so = os.path.join(d, "plan.cpp"), os.path.join(d, "plan.so")
    with open(src, "w") as f:
        f.write(SRC)
    subprocess.run([build.CXX, "-std=c++17", "-O2", "-Wall", "-fPIC", "-shared", "-I", build.CSRC, "-o", so, src],
                   check=True)
    lib = ctypes.CDLL(so)
    for name in ("t_slot", "t_unit"):
        getattr(lib, name).restype = ctypes.c_longlong
    lib.t_unit.argtypes = [ctypes.c_int, ctypes.c_longlong, ctypes.c_int]
    lib.t_group.argtypes = [ctypes.c_longlong, ctypes.c_longlong, ctypes.c_int]
    return lib


def clamp(C, s, e, T):
    n = ctypes.c_int()
    return C.t_clamp(s, e, T, ctypes.byref(n)), n.value


def sizes(C, planned, B, T, G, HKV, R, DT, P):
    out = (ctypes.c_longlong * 9)()
    C.t_sizes(planned, B, T, G, HKV, R, DT, P, out)
    return dict(zip(("items", "ints", "part", "ml", "where", "part1", "ml1", "where1", "total"), out))


@pytest.mark.parametrize("d", [1, 2, 3, 5, 7, 16, 21, 63, 64, 100, 4096, 65537, 2 ** 30, 2 ** 31 - 1])
def test_division(C, d):
    r = np.random.default_rng(d)
    for n in [0, 1, d - 1, d, min(d + 1, 2 ** 31 - 1), 2 ** 31 - 1] + [int(x) for x in r.integers(0, 2 ** 31 - 1, 500)]:
        assert C.t_div(d, n) == n // d


def test_units_up_to_the_limit(C):
    for v in (0, 1, 63, 64, 65, 1 << 20, TOP - 64, TOP - 1, TOP):
        assert C.t_units(v) == -(-v // 64)


@pytest.mark.parametrize("U,groups", [(1, 256), (255, 256), (256, 256), (257, 256), (99991, 256), (41000, 2048), (3, 8),
                                      ((1 << 31) * (1 << 16) - 1, 256), ((1 << 31) * (1 << 16) - 7, 2048)])
def test_shares(C, U, groups):
    """Exact up to the most units that a call may have: 2^31 of one kv head, 2^16 heads."""
    n = min(U, groups)
    start = [C.t_unit(w, U, n) for w in range(n + 1)]
    assert start == [w * U // n for w in range(n + 1)] and start[0] == 0 and start[n] == U
    assert all(a < b for a, b in zip(start, start[1:]))
    some = {u for s in start for u in (s - 1, s, s + 1) if 0 <= u < U} | set(range(min(U, 300)))
    for u in some:
        w = C.t_group(u, U, n)
        assert 0 <= w < n and start[w] <= u < start[w + 1]


@pytest.mark.parametrize("s,e,T", [(0, 5, 5), (-7, 2, 5), (2, 50, 5), (2, 2 ** 31 - 1, 5), (-2 ** 31, 2 ** 31 - 1, 9),
                                   (4, 2, 5), (9, 12, 5), (2 ** 31 - 1, -2 ** 31, 3), (3, 3, 5), (0, 0, 0)])
def test_tokens_are_clamped(C, s, e, T):
    lo, hi = (min(max(x, 0), T) for x in (s, e))
    t0, n = clamp(C, s, e, T)
    assert n == max(hi - lo, 0) and t0 == lo and 0 <= t0 <= T and t0 + n <= T


def replay(C, nk, hkv, groups, slots):
    """Results that the shares of `groups` leave of items of nk units for each of hkv heads: all in different places
    below `slots`, those of a pair one after the other from where its first share says, as many as it says."""
    first = np.concatenate([[0], np.cumsum(nk)])
    UH, items = int(first[-1]), len(nk)
    if UH == 0:
        return
    U = UH * hkv
    n = min(U, groups)
    seen, of, told = set(), {}, {}
    for w in range(n):
        u, u1 = C.t_unit(w, U, n), C.t_unit(w + 1, U, n)
        while u < u1:
            head, at = divmod(u, UH)
            item = int(np.searchsorted(first[:items], at, side="right")) - 1
            kt = at - int(first[item])
            k1 = min(int(nk[item]), kt + u1 - u)
            place = C.t_slot(w, item, items, head)
            assert place not in seen and 0 <= place < slots
            seen.add(place)
            of.setdefault((head, item), []).append(place)
            if kt == 0:
                told[head, item] = place, C.t_group(head * UH + int(first[item + 1]) - 1, U, n) - w + 1
            u += k1 - kt
    for pair, places in of.items():
        place, count = told[pair]
        assert places == list(range(place, place + count))
    assert len(of) == hkv * int((np.asarray(nk) > 0).sum())


@pytest.mark.parametrize("seed", range(40))
def test_a_planned_batch_fits_its_workspace(C, seed):
    """k_attn_plan's items, their order and the places of their results, for offsets of any kind."""
    r = np.random.default_rng(seed)
    D, parts, HKV = int(r.choice([8, 64, 80, 128, 200, 256])), int(r.choice([1, 2])), int(r.integers(1, 5))
    B, T, G = int(r.integers(1, 12)), int(r.integers(1, 300)), int(r.choice([1, 2, 5, 8, 40]))
    P, R, DT = int(r.choice([0, 70, 500])), C.t_rows(D, parts), C.t_padded(D)
    q_start = [np.sort(r.integers(0, T + 1, B + 1)), r.integers(-T, 2 * T, B + 1),
               r.choice([-2 ** 31, -1, 0, T // 2, T, 2 ** 31 - 1], B + 1)][seed % 3]
    tok = [clamp(C, int(q_start[b]), int(q_start[b + 1]), T) for b in range(B)]
    z = sizes(C, 1, B, T, G, HKV, R, DT, P)
    packed = min(sum(n for _, n in tok if n > 0 and not C.t_joint(n, G, R)), T) if P else 0
    n_packed = -(-packed * G // R)
    most = n_packed + B + T * G // R
    own = [int(x) for x in r.integers(0, 400, B)]
    nk = [C.t_units(P)] * n_packed
    for b, (t0, n) in enumerate(tok):
        for _ in range(-(-n * G // R)):
            if len(nk) < most:
                nk.append((C.t_units(P) if C.t_joint(n, G, R) else 0) + C.t_units(own[b]))
    assert len(nk) <= z["items"]
    assert 4 * (4 + (z["items"] + 1) + 2 * z["items"] + B + 2 * T) <= z["ints"]
    slots = z["part"] // (R * DT * 4)
    assert slots * R * 8 <= z["ml"] and len(nk) * HKV * 8 <= z["where"]
    replay(C, nk, HKV, C.t_groups(), slots)
    asked = library_asks(B, T, G, HKV, D, P, planned=True)
    assert asked == max(sizes(C, 1, B, T, G, HKV, C.t_rows(D, x), DT, P)["total"] for x in (1, 2))
    assert asked >= z["total"]


def library_asks(B, T, G, HKV, D, P, planned):
    lib = _native.load_hip()
    lib.bpd_gpu_last_error()
    c = cache(n_kv_heads=HKV, head_dim=D)
    b = batch(n_seqs=B, n_tokens=T, q_start=0x9000 if planned else None, prefix=0x8000 if P else None, prefix_len=P)
    n = lib.bpd_attn_paged_workspace(ctypes.addressof(c), ctypes.addressof(b), G * HKV)
    assert lib.bpd_gpu_last_error() == 0
    return n


@pytest.mark.parametrize("seed", range(20))
def test_a_batch_of_single_tokens_fits_its_workspace(C, seed):
    """The prefix's tiles by 8 x of the workgroups (all without own keys), the sequences' own keys by the waves of the
    others, 2,048 at most."""
    r = np.random.default_rng(seed)
    D, parts, HKV = int(r.choice([8, 64, 80, 128, 200, 256])), int(r.choice([1, 2])), int(r.integers(1, 5))
    B, G, P = int(r.integers(1, 90)), int(r.choice([1, 2, 5, 8, 16])), int(r.choice([0, 70, 500, 2000]))
    R, DT = C.t_rows(D, parts), C.t_padded(D)
    z = sizes(C, 0, B, B, G, HKV, R, DT, P)
    own = [int(x) for x in r.integers(0, 400, B)]
    for x8 in (1, 13, 31, 32) if P else (0,):
        if P:
            replay(C, [C.t_units(P)] * (-(-B * G // R)), HKV, 8 * x8, z["part"] // (R * DT * 4))
        waves = 8 * (32 - x8) * (4 if DT == 256 else 8) if P else C.t_waves()
        if waves:
            assert waves <= C.t_waves()
            replay(C, [-(-n // 32) for n in own], HKV, waves, z["part1"] // (G * DT * 4))
    assert -(-B * G // R) <= z["items"] or not P
    assert z["part1"] // (G * DT * 4) * G * 8 <= z["ml1"] and B * HKV * 8 <= z["where1"]
    assert library_asks(B, B, G, HKV, D, P, planned=False) == \
        max(sizes(C, 0, B, B, G, HKV, C.t_rows(D, x), DT, P)["total"] for x in (1, 2))
