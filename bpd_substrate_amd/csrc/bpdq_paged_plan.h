// bpdq_paged_plan.h — the index arithmetic of the paged kernels that needs neither a GPU nor its intrinsics: divisions
// by the page size, which share takes which units, places of results, tiles and the workspace.  The kernels and their
// launchers include it as the CPU's tests do.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define BPDQ_BOTH __host__ __device__ __forceinline__
#else
#define BPDQ_BOTH inline
#endif

namespace bpdq {

// n / d for 0 <= n < 2^31, d >= 1: with s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1,
// n / d = (mulhi(m, n) + n) >> s (division by an invariant integer, Granlund and Montgomery 1994).
struct FastDiv {
    uint32_t m, s, d;
};
inline FastDiv fast_div(int d) {
    FastDiv f;
    f.d = (uint32_t)d;
    f.s = 0;
    while ((1ull << f.s) < (uint64_t)d) f.s++;
    f.m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << f.s) - (uint64_t)d)) / (uint64_t)d + 1);
    return f;
}
BPDQ_BOTH int fdiv(FastDiv f, int n) {
    const uint32_t hi = (uint32_t)(((uint64_t)f.m * (uint32_t)n) >> 32);
    return (int)((hi + (uint32_t)n) >> f.s);
}

// The first and one past the last new token of a sequence, q_start's two values given, within [0, T].
BPDQ_BOTH void clamp_tokens(int start, int end, int T, int& t0, int& n) {
    const int lo = start < 0 ? 0 : start, hi = end < 0 ? 0 : end;
    t0 = lo < T ? lo : T;
    n = (hi < T ? hi : T) - t0;
    if (n < 0) n = 0;
}

constexpr int kKeys = 64;     // keys of a unit
constexpr int kGroups = 256;  // workgroups that share the units: one per CU
constexpr int kStreamWaves = 2048;  // k_attn_wave's: two per SIMD

// Units of v rows.
BPDQ_BOTH constexpr int units_of(int v) { return (v + 63) / 64; }
// Units are numbered head by head, as a head's items may share keys (a prefix), which its neighbours in
// the order then find in the L2 of their XCD.  [w U / n, (w + 1) U / n) go to share w of n = min(groups, U).
// A share leaves at most one result per (head, item): share and pair never repeat together
// in share + pair, as each step along the units raises one or both.
BPDQ_BOTH int64_t slot_of(int share, int item, int nitems, int h) {
    return (int64_t)share + (int64_t)h * nitems + item;
}
BPDQ_BOTH int64_t unit_of(int w, int64_t U, int n) { return w * U / n; }
BPDQ_BOTH int group_of(int64_t u, int64_t U, int n) { return (int)(((u + 1) * n - 1) / U); }
// Whether a sequence's n tokens of G heads fill half a tile by themselves: then it takes the prefix's keys too.
BPDQ_BOTH bool is_joint(int n, int G, int R) { return n * G * 2 >= R; }

inline int padded(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
// Waves of a workgroup and 16-row tiles of a wave: 8 waves of 32 rows where the accumulators and the
// parts of the queries fit the 256 registers of two waves per SIMD.
struct Tile {
    int mt, nw;
};
inline Tile tile_of(int D, int parts) {
    if (D <= 64) return {2, 8};
    if (D <= 128) return {parts == 1 ? 2 : 1, 8};
    return {1, 4};
}
inline int rows_of(int D, int parts) {
    const Tile t = tile_of(D, parts);
    return 16 * t.mt * t.nw;
}

inline int64_t up16(int64_t v) { return (v + 15) / 16 * 16; }

// The workspace of either way: planned, or one token per sequence by k_attn_wave with the prefix packed.
// ints: info 4, first items + 1, seq and rt items each, item0 B, packed and place T each.
struct Sizes {
    int64_t items, ints, part, ml, where, part1, ml1, where1, total;
};
inline Sizes sizes(bool planned, int B, int T, int G, int HKV, int R, int DT, int P) {
    Sizes s = {};
    const int64_t per_rows = (int64_t)T * G / R + 1;
    s.items = planned ? 2 * per_rows + B : P > 0 ? per_rows : 0;
    const int64_t slots = s.items > 0 ? kGroups + s.items * HKV : 0;
    s.ints = planned ? up16(4 * (4 + (s.items + 1) + 2 * s.items + B + 2 * (int64_t)T)) : 0;
    s.part = slots * R * DT * 4;
    s.ml = up16(slots * R * 8);
    s.where = up16(s.items * HKV * 8);
    if (!planned) {
        const int64_t n = (kStreamWaves + (int64_t)B * HKV) * G;
        s.part1 = n * DT * 4;
        s.ml1 = up16(n * 8);
        s.where1 = up16((int64_t)B * HKV * 8);
    }
    s.total = s.ints + s.part + s.ml + s.where + s.part1 + s.ml1 + s.where1;
    return s;
}

}  // namespace bpdq
