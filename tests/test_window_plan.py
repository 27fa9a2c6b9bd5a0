"""Which units a windowed item reads (csrc/bpdq_paged_plan.h, compiled for the CPU) against the rows that its tokens see
one by one.  No GPU."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from bpd_substrate_amd import build

SRC = r"""
#include "bpdq_paged_plan.h"
using namespace bpdq;
extern "C" {
void t_span(long long first, int W, int S, int P, int seen, int U, int* out) {
    const Span s = span_of(first, W, S, P, seen, U);
    const int v[] = {s.a1, s.b0, s.b1, s.c1, s.d0, s.d1, prefix_units(s), own_units(s)};
    for (int i = 0; i < 8; i++) out[i] = v[i];
}
int t_first_tile(int t0, int b, int G) { return first_tile(t0, b, G); }
int t_unit_at(long long first, int W, int S, int P, int seen, int U, int t, int* pre) {
    bool p;
    const int r = unit_at(span_of(first, W, S, P, seen, U), t, p);
    *pre = p;
    return r;
}
}
"""


@pytest.fixture(scope="module")
def C(tmp_path_factory):
    d = str(tmp_path_factory.mktemp("span"))
    src, so = os.path.join(d, "span.cpp"), os.path.join(d, "span.so")
    with open(src, "w") as f:
        f.write(SRC)
    subprocess.run([build.CXX, "-std=c++17", "-O2", "-Wall", "-fPIC", "-shared", "-I", build.CSRC, "-o", so, src],
                   check=True)
    lib = ctypes.CDLL(so)
    lib.t_span.argtypes = [ctypes.c_longlong] + [ctypes.c_int] * 5 + [ctypes.c_void_p]
    lib.t_unit_at.argtypes = [ctypes.c_longlong] + [ctypes.c_int] * 6 + [ctypes.c_void_p]
    return lib


def units(C, first, W, S, P, seen, U):
    out, pre = (ctypes.c_int * 8)(), ctypes.c_int()
    C.t_span(first, W, S, P, seen, U, out)
    a1, b0, b1, c1, d0, d1, np_, no = out
    assert 0 <= a1 <= b0 <= b1 == -(-P // U) and 0 <= c1 <= d0 <= d1 == -(-seen // U)
    got = []
    for t in range(np_ + no):
        u = C.t_unit_at(first, W, S, P, seen, U, t, ctypes.byref(pre))
        got.append((not pre.value, u))
    return got


@pytest.mark.parametrize("seed", range(40))
def test_units_are_those_with_a_row_that_is_seen(C, seed):
    r = np.random.default_rng(seed)
    for _ in range(50):
        U = int(r.choice([32, 64]))
        P, own = int(r.choice([0, r.integers(1, 400)])), int(r.integers(0, 500))
        n = int(r.integers(1, max(2, own + 1)))
        W, S = int(r.choice([1, r.integers(1, 600), 2 ** 31 - 1])), int(r.choice([0, r.integers(1, 600), 2 ** 31 - 1]))
        first = P + own - n                      # position of the first new token
        low = max(0, first - W + 1)
        got = units(C, first, W, S, P, own, U)
        assert got == sorted(set(got)), "units in order, each once"
        want = {(j >= P, (j if j < P else j - P) // U) for j in range(P + own) if j >= low or j < S}
        assert set(got) == want


@pytest.mark.parametrize("seed", range(30))
def test_tiles_of_sequences_lie_behind_each_other(C, seed):
    """Every sequence's ceil(n G / 16) tiles have places of their own, within the launch's T G / 16 + B."""
    r = np.random.default_rng(seed)
    B, G = int(r.integers(1, 300)), int(r.choice([1, 2, 3, 5, 8, 16, 40, 64]))
    n = [int(x) for x in r.choice([0, 0, 1, 1, 2, 7, 64, 333], B)]
    start = np.concatenate([[int(r.integers(0, 5))], n]).cumsum()
    T, end = int(start[-1] + r.integers(0, 5)), 0
    for b in range(B):
        at = C.t_first_tile(int(start[b]), b, G)
        assert at >= end
        end = at + -(-n[b] * G // 16)
        assert b + 1 == B or end <= C.t_first_tile(int(start[b + 1]), b + 1, G)
    assert end <= T * G // 16 + B
    assert C.t_first_tile(1 << 23, (1 << 23) - 1, 8) == (1 << 22) + (1 << 23) - 1


def test_extreme_positions_and_lengths(C):
    top = 2 ** 31 - 1025
    assert units(C, 2 ** 31, 1, 0, 0, 5, 64) == []                      # a length beyond the table: nothing of it is seen
    assert units(C, -(2 ** 31), 7, 0, 70, 0, 64) == [(False, 0), (False, 1)]
    assert units(C, top - 1, 64, 0, 0, top, 64)[-1] == (True, (top - 1) // 64)
    assert len(units(C, top - 1, 64, 0, 0, top, 64)) in (1, 2)
    assert units(C, top - 1, 1, 3, top - 10, 10, 64) == [(False, 0), (True, 0)]
