// paged_attn.hip — bpd_attn_paged_gpu: attention over a paged cache.
//
//   s_i = scale q.k_i,  out = sum_i exp(s_i - m) v_i / sum_i exp(s_i - m),  m = max s_i,
//   lse = m + log sum_i exp(s_i - m)
//
// in one pass over the keys: a row of a query head keeps a reference exponent r (base 2), its
// sum l = sum 2^(s - r) and O = sum 2^(s - r) v in fp32.  Where a later part of the
// keys has another reference, sums join as O 2^(r - r') + O' (k_attn_join).  Weights are rounded
// to the cache's type for their product with v, as the matrix instructions take them (half a step each, relative to
// the weight; with an fp32 q two or three parts keep 22 or 24 bits); l sums them unrounded.
//
// Work.  The query heads of one kv head share its keys, so a row is a (token, query head)
// pair.  Two kernels take the keys:
//   - k_attn_tile: R rows against 64 keys at a time, through LDS.  The matrix units bound it.
//   - k_attn_wave, for sequences with one new token and up to 16 heads on a kv head: a wave by itself
//     streams a sequence's keys past one 16-row tile.  Memory bounds it.
// With one token each (q_start NULL) the tokens' rows are packed against the prefix, which is so
// read once for R / (heads per kv head) sequences, and the own keys are k_attn_wave's; k_attn_both runs the two
// side by side.  Otherwise k_attn_plan lays out items, tile rows with all their keys, on the device, as the lengths are
// there:
//   - own items: the rows of one sequence against its own keys, causal, and where a
//     sequence fills half a tile by itself, the prefix before them;
//   - packed items: the rows of all other sequences together against the prefix.
// Units of 64 keys (32 of k_attn_wave's), item by item, are dealt evenly to the workgroups, whose number
// does not depend on the batch: a workgroup runs through its units, and where an item ends in
// the middle leaves its O, r and l for k_attn_join, in a place of its own.
//
// Measured, bf16 unless said (H 32, 8 kv heads, D 128; calls back to back):
//   8 chunks of up to 512 tokens, 3,070 in all, over 4096
//   shared and up to 1024 own keys                        332 us   705 TFLOP/s (an 8192^3 product: 1256)
//   the same with fp32 queries, f16 / bf16 pages          586 / 682 us
//   32 sequences of up to 8192 own keys, 670 MB           113 us   5.9 TB/s (reads alone: 6.8)
//   256 sequences behind 32,768 shared keys, 1024 own     243 us   140 GFLOP and 781 MB: 112 + 115 us
//   64 sequences (f16) behind 8192 shared keys, 600 own    46 us   9 GFLOP and 130 MB: 14 + 19 us
//   1 sequence of 300 keys, D 64                           14 us   two launches
#include <type_traits>

#include "bpdq_paged.h"

namespace bpdq {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_inff();

// The plan in the workspace.  Items are those of all kv heads of a tile: (item, head).
struct Plan {
    int32_t* info;    // [0] items, [1] units of one kv head, [2] packed tokens
    int32_t* first;   // [items + 1] units of one kv head before the item's
    int32_t* seq;     // [items] sequence, -1 packed
    int32_t* rt;      // [items] which tile of its rows
    int32_t* item0;   // [B] first own item of a sequence
    int32_t* packed;  // [T] token of a packed index
    int32_t* place;   // [T] packed index of a token, -1
};

struct AttnArgs {
    Paged a;
    const uint8_t* q;
    uint8_t* out;
    int64_t qs, os;
    float* lse;
    int H, G;
    float scale;
    FastDiv g;  // by G
    int R, DT;   // rows of a tile, padded head size
    int groups;  // workgroups
    bool planned;  // the items are the plan's; otherwise every token is packed, and sequences are k_attn_wave's
    Plan p;
    float* part;   // [slot][R][DT]
    float2* ml;    // [slot][R] reference exponent, sum
    int2* where;   // [head][item] first slot of its results and their number, 0 where the output is written
    int waves;     // k_attn_wave: shares
    float tile_cost, wave_cost;
    float* part1;  // k_attn_wave's results, [slot][G][DT], and the same of them
    float2* ml1;
    int2* where1;  // [head][sequence]
};

// Rows of a sequence's own part that the table holds.
__device__ __forceinline__ int own_rows(const Paged& a, int b) {
    return max(0, min(a.lens[b], a.W * (int)a.page.d));
}
__device__ __forceinline__ bool is_joint(const AttnArgs& g, int n) { return bpdq::is_joint(n, g.G, g.R); }

// Whole own rows that row `last` (token index within the sequence) of a tile can see.
__device__ __forceinline__ int seen_rows(const Paged& a, int b, int n, int i, int own) {
    const int64_t s = (int64_t)a.lens[b] - n + i + 1;
    return (int)(s < 0 ? 0 : s > own ? own : s);
}

// One workgroup lays out the items: sequences are taken 1024 at a time, a thread each, then their tiles and
// tokens, a thread each.  Latency bounds it: 6 us for 3,070 tokens of 8 sequences, beside the 350 of what follows.
__global__ __launch_bounds__(1024) void k_attn_plan(AttnArgs g) {
    constexpr int N = 1024;
    __shared__ int s_wave[N / 64];
    __shared__ int s_at[N];   // exclusive sums of a round
    const Paged& a = g.a;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int ntp = units_of(a.P);
    auto scan = [&](int v) {  // (exclusive sum, total) over the workgroup
        int x = v;
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(x, d);
            if (lane >= d) x += o;
        }
        __syncthreads();
        if (lane == 63) s_wave[wave] = x;
        __syncthreads();
        int before = 0, total = 0;
        for (int i = 0; i < N / 64; i++) {
            if (i < wave) before += s_wave[i];
            total += s_wave[i];
        }
        return make_int2(before + x - v, total);
    };
    // the packed tokens
    int packed = 0;
    if (a.P > 0) {
        for (int b0 = 0; b0 < a.B; b0 += N) {
            const int b = b0 + tid;
            int t0 = 0, n = 0;
            if (b < a.B) seq_tokens(a, b, t0, n);
            const bool in = n > 0 && !is_joint(g, n);
            const int2 at = scan(in ? n : 0);
            if (in)  // fewer than R / 2G tokens
                for (int i = 0; i < n; i++) {
                    const int k = packed + at.x + i;
                    if (k < a.T) g.p.packed[k] = t0 + i;
                    g.p.place[t0 + i] = k < a.T ? k : -1;
                }
            packed = min(packed + at.y, a.T);
        }
    }
    const int np = packed > 0 ? (packed * g.G + g.R - 1) / g.R : 0;
    for (int i = tid; i < np; i += N) {
        g.p.first[i] = i * ntp;
        g.p.seq[i] = -1;
        g.p.rt[i] = i;
    }
    // the sequences' own tiles
    int items = np;
    // more than this many only offsets that decrease can ask for: the plan ends there
    const int most = np + a.B + (int)(((int64_t)a.T * g.G) / g.R);
    for (int b0 = 0; b0 < a.B; b0 += N) {
        const int b = b0 + tid;
        int t0 = 0, n = 0;
        if (b < a.B) seq_tokens(a, b, t0, n);
        const int nrt = n > 0 ? (n * g.G + g.R - 1) / g.R : 0;
        const int2 at = scan(nrt);
        if (b < a.B) g.p.item0[b] = items + at.x;
        __syncthreads();
        s_at[tid] = at.x;
        __syncthreads();
        for (int k = tid; k < at.y && items + k < most; k += N) {
            int lo = 0, hi = N;  // the last sequence of the round that starts at or before k
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (s_at[mid] <= k) lo = mid;
                else hi = mid;
            }
            g.p.seq[items + k] = b0 + lo;
            g.p.rt[items + k] = k - s_at[lo];
        }
        items = min(items + at.y, most);
    }
    __threadfence_block();
    __syncthreads();
    // units before each
    int units = np * ntp;
    for (int k0 = np; k0 < items; k0 += N) {
        const int k = k0 + tid;
        int mine = 0;
        if (k < items) {
            const int b = g.p.seq[k], r = g.p.rt[k];
            int t0, n;
            seq_tokens(a, b, t0, n);
            const int last = min(n, ((r + 1) * g.R - 1) / g.G + 1) - 1;
            mine = (is_joint(g, n) ? ntp : 0) + units_of(seen_rows(a, b, n, last, own_rows(a, b)));
        }
        const int2 at = scan(mine);
        if (k < items) g.p.first[k] = units + at.x;
        units += at.y;
    }
    if (tid == 0) {
        g.p.first[items] = units;
        g.p.info[0] = items;
        g.p.info[1] = units;
        g.p.info[2] = packed;
    }
}

// Element offset of row i % page_size of a page.
__device__ __forceinline__ int64_t row_at(const Paged& a, int page, int in_page) {
    return (int64_t)page * a.page_stride + (int64_t)in_page * a.row_stride;
}

// A value at an address that is the same in every lane, through the scalar cache.
__device__ __forceinline__ int load_uniform(const int32_t* p) {
    return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)p;
}

template <int CT>
struct Mfma;
template <>
struct Mfma<BPD_T_F16> {
    using T = _Float16;
    using V = f16x8;
    static __device__ __forceinline__ f32x4 go(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
};
template <>
struct Mfma<BPD_T_BF16> {
    using T = __bf16;
    using V = bf16x8;
    static __device__ __forceinline__ f32x4 go(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
};

// x as NS values of the cache's type whose sum keeps 11 NS (f16) or 8 NS (bf16) bits of it, 8 elements.
template <int CT, int NS>
__device__ __forceinline__ void split8(const float (&x)[8], u32x4 (&out)[NS]) {
    using V = typename Mfma<CT>::V;
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = x[i];
#pragma unroll
    for (int s = 0; s < NS; s++) {
        typedef float F8 __attribute__((ext_vector_type(8)));
        const V v = __builtin_convertvector((F8){r[0], r[1], r[2], r[3], r[4], r[5], r[6], r[7]}, V);
        if (s + 1 < NS) {
#pragma unroll
            for (int i = 0; i < 8; i++) r[i] -= (float)v[i];
        }
        out[s] = __builtin_bit_cast(u32x4, v);
    }
}

// The largest of lanes l, l ^ 16, l ^ 32 and l ^ 48.
__device__ __forceinline__ float xor_max(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t v = __float_as_uint(fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1])));
    const auto q = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}

// Elements 8 (4 k + lg) .. + 7 of a query, in binary32; zeros behind its end and for a row that is none.
template <int KS, typename Q>
__device__ __forceinline__ void load_query(const Q* __restrict__ q, bool row, int per, int lg, float sign,
                                           float (&x)[KS][8]) {
#pragma unroll
    for (int k = 0; k < KS; k++) {
        const int c = 4 * k + lg;
        Vec<Q, 8> v;
#pragma unroll
        for (int e = 0; e < 8; e++) v.v[e] = (Q)0.f;
        if (row && c < per) v = *reinterpret_cast<const Vec<Q, 8>*>(q + 8 * c);
#pragma unroll
        for (int e = 0; e < 8; e++) x[k][e] = sign == 1.f ? (float)v.v[e] : (float)v.v[e] * sign;
    }
}

// Scales an fp32 query by a power of two to a largest element in [1, 2), so that two binary16 parts keep
// 22 bits of that; returns the exponent taken out.
template <int KS>
__device__ __forceinline__ int row_exponent(float (&x)[KS][8]) {
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, __builtin_fabsf(x[k][e]));
    top = xor_max(top);
    int e2 = (int)((__float_as_uint(top) >> 23) & 255) - 127;
    if (top == 0.f || e2 == 128) e2 = 0;
    e2 = max(e2, -100);
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
        for (int e = 0; e < 8; e++) x[k][e] = ldexpf(x[k][e], -e2);
    return e2;
}

// What a score is multiplied by, the exponent put back.  Not 0: a row that is not there has a score of -infinity.
__device__ __forceinline__ float score_scale(float scale2, int e2) {
    const float s = ldexpf(scale2, e2);
    return s < 0x1p-126f ? 0x1p-126f : s;  // scores of less than 2^-90 weigh 1
}

// The lane's elements of a row of O, of the first D, where row c of product 8 vb + e holds element
// 128 vb + 2 VD c + e.
template <typename Q, int VD, int VB>
__device__ __forceinline__ void store_row(Q* out, int D, int lg, const f32x4* o, float f) {
#pragma unroll
    for (int vb = 0; vb < VB; vb++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = vb * 128 + 2 * VD * (4 * lg + r);
            if (d >= D) continue;
            Vec<Q, 2 * VD> v;
#pragma unroll
            for (int e = 0; e < 2 * VD; e++) v.v[e] = (Q)(o[vb * 8 + e][r] * f);
            *reinterpret_cast<Vec<Q, 2 * VD>*>(out + d) = v;
        }
}

// The same where product e holds elements 16 e .. 16 e + 15.
template <typename Q, int NE>
__device__ __forceinline__ void store_row4(Q* out, int D, int lg, const f32x4* o, float f) {
#pragma unroll
    for (int e = 0; e < NE; e++) {
        const int d = 16 * e + 4 * lg;
        if (d >= D) continue;
        Vec<Q, 4> v;
#pragma unroll
        for (int r = 0; r < 4; r++) v.v[r] = (Q)(o[e][r] * f);
        *reinterpret_cast<Vec<Q, 4>*>(out + d) = v;
    }
}

// Which 16-byte chunk slot of a row in LDS holds chunk c.  K: the 16 rows of an operand read differ in it, so
// that the read meets every bank once.  V: a transposing read takes 32 bytes of each of 16 rows, so pairs
// of chunks differ.
template <int DT>
__device__ __forceinline__ int k_slot(int row, int c) {
    return DT == 64 ? c ^ ((row >> 1) & 7) : c ^ (row & 15);
}
template <int DT>
__device__ __forceinline__ int v_slot(int row, int c) {
    return DT == 64 ? c ^ (((row >> 1) & 3) << 1) : c ^ ((row & 7) << 1);
}

template <int DT>
struct Lds {
    uint4 k[2][kKeys][DT / 8];
    uint4 v[2][kKeys][DT / 8];
    float bias[2][kKeys];  // 0, or -inf for a row that is not there
};

// Bit 15 of each half: that 16-bit value is an infinity or NaN (the exponent's carry).
template <int CT>
__device__ __forceinline__ uint32_t not_finite(uint32_t d) {
    constexpr uint32_t e = CT == BPD_T_F16 ? 0x7C007C00u : 0x7F807F80u;
    constexpr uint32_t one = CT == BPD_T_F16 ? 0x04000400u : 0x00800080u;
    return ((d & e) + one) & 0x80008000u;
}
template <int CT>
__device__ __forceinline__ uint32_t finite_or_0(uint32_t d) {
    return d & ~((not_finite<CT>(d) >> 15) * 0xFFFFu);
}

// The 4 x 16 transposing LDS read: of each 16 lanes, lane 4 i + c gives the place of elements 4 c .. 4 c + 3 of
// row i, and lane l gets element l of rows 0..3.
typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x2 read_tr(const uint8_t* p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (__attribute__((address_space(3))) s16x4*)(const_cast<uint8_t*>(p))));
}

// NW waves of 16 MT rows each, the units [u0, u1) of this workgroup.  Scores are taken as
// S^T = K Q^T (lane: query l % 16, keys 4 (l / 16) + r), which is the layout in which
// O^T = V^T P^T takes P: the 32 keys of two score tiles in the order 4g..4g+3, 16+4g..16+4g+3 of
// lane group g.  V's operand comes in that order from two transposing reads; row c of it is
// element 16 e + c of the head in product e.
// UNI: pages hold multiples of 16 rows, so the rows that a wave's lanes move at a time share a page.
//
// 8 waves of 32 rows: a half's K operands serve both row tiles of a wave, and 256 rows share what a unit brings to
// LDS.  What bounds it at 705 TFLOP/s: a SIMD's two waves are both in their softmax for part of the time (matrix units
// busy 32 % of the clocks, vector units 42 %, no LDS conflicts), and registers: all 256, with 9-11 vector and 87-143
// scalar ones of the 16-bit form kept aside.  Measured and left: K of the next half read behind P V (338 us against
// 334), wave priorities around the products (no change).
template <int QT, int CT, int NS, int DT, int MT, int NW, bool UNI>
__device__ __forceinline__ void tile_share(const AttnArgs& g, Lds<DT>& s, int w, int groups) {
    using M = Mfma<CT>;
    using T = typename M::T;
    using Q = typename Elem<QT>::type;
    constexpr int CPR = DT / 8;           // 16-byte chunks of a row
    constexpr int NI = kKeys * CPR / (64 * NW);  // chunks of K and of V that a thread moves per unit
    constexpr int KS = DT / 32;           // products of a score tile
    constexpr int NE = DT / 16;           // products of O
    constexpr int LR = 64 / CPR;          // rows that a wave moves at a time
    static_assert(NI >= 1 && 16 % LR == 0, "a chunk per thread, rows of one page");
    const Paged& a = g.a;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, lg = lane >> 4;
    const int ntiles = units_of(a.P);
    const int nitems = g.planned ? g.p.info[0] : (a.T * g.G + g.R - 1) / g.R;
    const int UH = g.planned ? g.p.info[1] : nitems * ntiles;
    const int64_t U = (int64_t)UH * a.hkv;
    const int n_groups = (int)(U < groups ? U : groups);
    if (w >= n_groups) return;
    int64_t u = unit_of(w, U, n_groups);
    const int64_t u1 = unit_of(w + 1, U, n_groups);
    const int per = a.D / 8;  // chunks that exist
    const float sign = g.scale > 0.f ? 1.f : g.scale < 0.f ? -1.f : 0.f;
    const float scale2 = (g.scale == 0.f ? 1.f : __builtin_fabsf(g.scale)) * kLog2e;

    while (u < u1) {
        // ---- the item of unit u
        const int head = (int)(u / UH), in = (int)(u - (int64_t)head * UH);
        int item, f0, nk, b = -1, rt, t0 = 0, n = a.T, own = 0, ntp = ntiles;
        if (g.planned) {
            item = __builtin_amdgcn_readfirstlane(count_le(g.p.first, nitems, in) - 1);
            f0 = g.p.first[item];
            nk = g.p.first[item + 1] - f0;
            b = g.p.seq[item];
            rt = g.p.rt[item];
            if (b >= 0) {
                seq_tokens(a, b, t0, n);
                own = own_rows(a, b);
                if (!is_joint(g, n)) ntp = 0;
            } else {
                n = g.p.info[2];
            }
        } else {
            rt = item = in / ntiles;
            f0 = item * ntiles;
            nk = ntiles;
        }
        int kt = in - f0;
        const int k0 = kt;
        const int k1 = (int)(u1 - u < nk - kt ? kt + (u1 - u) : nk);
        const bool last_word = kt == 0 && k1 == nk && b >= 0 && (ntp > 0 || a.P == 0);
        if (kt == 0 && tid == 0) {
            const int64_t ue = (int64_t)head * UH + f0 + nk - 1;
            g.where[(int64_t)head * nitems + item] =
                make_int2((int)slot_of(w, item, nitems, head), last_word ? 0 : group_of(ue, U, n_groups) - w + 1);
        }
        const int64_t hoff = (int64_t)head * a.head_stride;
        const int32_t* table = b >= 0 ? a.table + (int64_t)b * a.table_stride : nullptr;

        // ---- this wave's queries
        u32x4 qf[MT][KS][NS];
        int e2[MT];   // the exponents taken out of them
        int lim[MT];  // own keys that the lane's query sees, -1: no query
        auto query_of = [&](int m, int& tok, int& hq) {
            const int row = rt * g.R + (wave * MT + m) * 16 + col, i = fdiv(g.g, row);
            hq = head * g.G + (row - i * g.G);
            tok = i >= n ? -1 : b >= 0 ? t0 + i : g.planned ? g.p.packed[i] : i;
            return i;
        };
#pragma unroll
        for (int m = 0; m < MT; m++) {
            int tok, hq;
            const int i = query_of(m, tok, hq);
            lim[m] = tok < 0 ? -1 : b >= 0 ? seen_rows(a, b, n, i, own) : 0;
            float x[KS][8];
            load_query<KS>(reinterpret_cast<const Q*>(g.q) + max(tok, 0) * g.qs + (int64_t)hq * a.D, tok >= 0, per, lg,
                           sign, x);
            e2[m] = 0;
            if constexpr (NS > 1 && CT == BPD_T_F16) e2[m] = row_exponent<KS>(x);
#pragma unroll
            for (int k = 0; k < KS; k++) split8<CT, NS>(x[k], qf[m][k]);
        }
        float qscale[MT];
#pragma unroll
        for (int m = 0; m < MT; m++) qscale[m] = NS > 1 && CT == BPD_T_F16 ? score_scale(scale2, e2[m]) : scale2;
        const bool busy = __ballot(lim[0] >= 0) != 0;  // rows of a wave fill from its first
        f32x4 o[MT][NE];
        float ref[MT], l[MT];
        int mend0 = 1 << 30, mend1 = 0;
#pragma unroll
        for (int m = 0; m < MT; m++) {
            ref[m] = kNegInf;
            l[m] = 0.f;
#pragma unroll
            for (int e = 0; e < NE; e++) o[m][e] = f32x4{0.f, 0.f, 0.f, 0.f};
        }

        // ---- staging of one unit's rows: a thread moves chunk tid % CPR of rows tid / CPR + 64 NW / CPR j
        const int srow = tid / CPR, sc = tid % CPR;
        const uint8_t *kthread = a.k + 2 * (hoff + 8 * sc), *vthread = a.v + 2 * (hoff + 8 * sc);
        if constexpr (UNI) {
            const int64_t at = 2 * (int64_t)(lane / CPR) * a.row_stride;
            kthread += at;
            vthread += at;
        }
        int pg[NI];
        uint4 rk[NI], rv[NI];
        bool rin[NI];
        // own or prefix index of this thread's (UNI: its wave's first) row j of unit t, rows there are
        auto key_of = [&](int t, int j, int& i, int& top) {
            const bool pre = t < ntp;
            i = (pre ? t : t - ntp) * kKeys + (UNI ? wave * LR : srow) + NW * LR * j;
            top = pre ? a.P : own;
            return pre ? a.prefix : table;
        };
        auto look = [&](int t) {  // the pages of unit t's rows
#pragma unroll
            for (int j = 0; j < NI; j++) {
                int i, top;
                const int32_t* tab = key_of(t, j, i, top);
                pg[j] = i < top ? UNI ? load_uniform(tab + fdiv(a.page, i)) : tab[fdiv(a.page, i)] : -1;
            }
        };
        auto load = [&](int t) {
#pragma unroll
            for (int j = 0; j < NI; j++) {
                int i, top;
                key_of(t, j, i, top);
                const bool there = pg[j] >= 0 && pg[j] < a.n_pages;
                const int64_t at = 2 * row_at(a, pg[j], i - fdiv(a.page, i) * (int)a.page.d);
                const auto* kp = reinterpret_cast<const uint4*>(kthread + at);
                const auto* vp = reinterpret_cast<const uint4*>(vthread + at);
                if (UNI && there && i + LR <= top && per == CPR) {  // all lanes
                    rin[j] = true;
                    rk[j] = *kp;
                    rv[j] = *vp;
                    continue;
                }
                rin[j] = there && i + (UNI ? lane / CPR : 0) < top;
                rk[j] = rv[j] = make_uint4(0, 0, 0, 0);
                if (rin[j] && sc < per) {
                    rk[j] = *kp;
                    rv[j] = *vp;
                }
            }
        };
        auto store = [&](int buf) {
#pragma unroll
            for (int j = 0; j < NI; j++) {
                const int row = srow + NW * LR * j;
                s.k[buf][row][k_slot<DT>(row, sc)] = rk[j];
                s.v[buf][row][v_slot<DT>(row, sc)] = rv[j];
                if (sc == 0) s.bias[buf][row] = rin[j] ? 0.f : kNegInf;
            }
        };
        bool fresh = true;  // a query of the wave has not met a key yet
        look(kt);
        load(kt);
        if (kt + 1 < k1) look(kt + 1);
        __syncthreads();  // the last item's units are done with the buffers
        store(kt & 1);
        for (; kt < k1; kt++) {
            const int buf = kt & 1;
            __syncthreads();
            if (kt + 1 < k1) load(kt + 1);
            if (kt + 2 < k1) look(kt + 2);
            if (busy) {
                const int key0 = (kt - ntp) * kKeys;  // own index of the unit's first key; below 0 in the prefix
#pragma unroll 1
                for (int half = 0; half < 2; half++) {
                    f32x4 sc4[2][MT], bias[2];
                    u32x4 kf[2][KS];
#pragma unroll
                    for (int kk = 0; kk < 2; kk++) {
                        const int r0 = half * 32 + kk * 16;
                        bias[kk] = *reinterpret_cast<const f32x4*>(&s.bias[buf][r0 + 4 * lg]);
#pragma unroll
                        for (int k = 0; k < KS; k++)
                            kf[kk][k] = __builtin_bit_cast(u32x4, s.k[buf][r0 + col][k_slot<DT>(col, 4 * k + lg)]);
                    }
                    __builtin_amdgcn_sched_barrier(0);  // every operand read is under way before the first product
#pragma unroll
                    for (int k = 0; k < KS; k++)
#pragma unroll
                        for (int kk = 0; kk < 2; kk++)
#pragma unroll
                            for (int m = 0; m < MT; m++)
#pragma unroll
                                for (int x = 0; x < NS; x++)
                                    sc4[kk][m] = M::go(kf[kk][k], qf[m][k][x],
                                                       k == 0 && x == 0 ? bias[kk] : sc4[kk][m]);
                    u32x4 vf[NE];
#pragma unroll
                    for (int e = 0; e < NE; e++)
#pragma unroll
                        for (int kk = 0; kk < 2; kk++) {
                            const int row = half * 32 + kk * 16 + 4 * lg + (col >> 2);
                            const u32x2 t = read_tr(reinterpret_cast<const uint8_t*>(
                                                        &s.v[buf][row][v_slot<DT>(row, 2 * e + ((col >> 1) & 1))]) +
                                                    8 * (col & 1));
                            vf[e][2 * kk] = t[0];
                            vf[e][2 * kk + 1] = t[1];
                        }
                    __builtin_amdgcn_sched_barrier(0);  // V's reads run behind the softmax
                    bool diag = false;
                    if (kt >= ntp && b >= 0) {
                        bool d = false;
#pragma unroll
                        for (int m = 0; m < MT; m++) d |= lim[m] >= 0 && lim[m] < min(own, key0 + half * 32 + 32);
                        diag = __ballot(d) != 0;
                    }
                    if (diag) {
#pragma unroll
                        for (int m = 0; m < MT; m++)
#pragma unroll
                            for (int e = 0; e < 8; e++)
                                if (key0 + half * 32 + (e >> 2) * 16 + 4 * lg + (e & 3) >= lim[m])
                                    sc4[e >> 2][m][e & 3] = kNegInf;
                    }
                    // weights 2^(x - ref), x = score log2(e).  Only where the 8 of a lane add up to more than
                    // 2^15.5 is the largest score looked for, and ref set to 10 below it: binary16 weights
                    // stay below their largest value, and normal 24 places below the largest weight
                    float p[MT][8], s8[MT];
                    auto weigh = [&](int m) {
                        const float base = ref[m] == kNegInf ? 0.f : ref[m];
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            p[m][e] = __builtin_amdgcn_exp2f(fmaf(sc4[e >> 2][m][e & 3], qscale[m], -base));
                        s8[m] = ((p[m][0] + p[m][1]) + (p[m][2] + p[m][3])) +
                                ((p[m][4] + p[m][5]) + (p[m][6] + p[m][7]));
                    };
                    bool over = fresh;
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        weigh(m);
                        over |= !(s8[m] <= 46340.f);
                    }
                    if (__ballot(over) != 0) {
                        bool none = false;
#pragma unroll
                        for (int m = 0; m < MT; m++) {
                            const f32x4 x = sc4[0][m], y = sc4[1][m];
                            const float top = xor_max(fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                                                            fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])))) * qscale[m];
                            const float nr = top - 12.f > ref[m] ? top - 10.f : ref[m];
                            const float f = nr == ref[m] ? 1.f : __builtin_amdgcn_exp2f(ref[m] - nr);
                            l[m] *= f;
#pragma unroll
                            for (int e = 0; e < NE; e++) o[m][e] *= f;
                            ref[m] = nr;
                            none |= lim[m] >= 0 && nr == kNegInf;
                            weigh(m);
                        }
                        fresh = __ballot(none) != 0;
                    }
                    u32x4 pf[MT][NS];
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        l[m] += s8[m];
                        split8<CT, NS>(p[m], pf[m]);
                    }
                    if (diag) {
                        // an infinity or NaN in a row that some queries do not see: 0 times it is no 0.  It
                        // counts as 0 here, and is added to the rows that see it after the last unit
                        uint32_t x = 0;
#pragma unroll
                        for (int e = 0; e < NE; e++)
#pragma unroll
                            for (int d = 0; d < 4; d++) x |= not_finite<CT>(vf[e][d]);
                        if (__ballot(x != 0) != 0) {
#pragma unroll
                            for (int e = 0; e < NE; e++)
#pragma unroll
                                for (int d = 0; d < 4; d++) vf[e][d] = finite_or_0<CT>(vf[e][d]);
                            mend0 = min(mend0, key0 + half * 32);
                            mend1 = key0 + half * 32 + 32;
                        }
                    }
                    // ---- O^T += V^T P^T
#pragma unroll
                    for (int e = 0; e < NE; e++)
#pragma unroll
                        for (int m = 0; m < MT; m++)
#pragma unroll
                            for (int x = 0; x < NS; x++) o[m][e] = M::go(vf[e], pf[m][x], o[m][e]);
                }
            }
            if (kt + 1 < k1) store((kt + 1) & 1);
        }

        // the infinities and NaN of the units at the causal border
        for (int key = mend0; key < min(mend1, own); key++) {
            const int pgi = fdiv(a.page, key), page = table[pgi];
            if (page < 0 || page >= a.n_pages) continue;
            const T* v = reinterpret_cast<const T*>(a.v) + row_at(a, page, key - pgi * (int)a.page.d) + hoff;
#pragma unroll
            for (int e = 0; e < NE; e++) {
                const int d = 16 * e + 4 * lg;
                if (d >= a.D) continue;
                const Vec<T, 4> x = *reinterpret_cast<const Vec<T, 4>*>(v + d);
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    if (key >= lim[m]) continue;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float y = (float)x.v[r];
                        if (!(__builtin_fabsf(y) < -kNegInf)) o[m][e][r] += y;
                    }
                }
            }
        }

        // ---- the item's rows, or this workgroup's part of them
        if (busy) {
            const int64_t slot = slot_of(w, item, nitems, head);
#pragma unroll
            for (int m = 0; m < MT; m++) {
                l[m] += __shfl_xor(l[m], 16);
                l[m] += __shfl_xor(l[m], 32);
                int tok, hq;
                query_of(m, tok, hq);
                if (tok < 0) continue;
                if (last_word) {
                    store_row4<Q, NE>(reinterpret_cast<Q*>(g.out) + tok * g.os + (int64_t)hq * a.D, a.D, lg, o[m],
                                         l[m] != 0.f ? 1.f / l[m] : 0.f);
                    if (g.lse != nullptr && lg == 0)
                        g.lse[(int64_t)tok * g.H + hq] =
                            l[m] != 0.f ? (ref[m] + __builtin_log2f(l[m])) * kLn2 : kNegInf;
                } else {
                    const int64_t row = slot * g.R + (wave * MT + m) * 16 + col;
                    store_row4<float, NE>(g.part + row * DT, DT, lg, o[m], 1.f);
                    if (lg == 0) g.ml[row] = make_float2(ref[m], l[m]);
                }
            }
        }
        u += k1 - k0;
    }
}

// One new token per sequence: its G <= 16 query heads of a kv head are the columns of one 16-row tile, and
// a wave reads the keys by itself, 32 at a time, V straight into the operand's registers, K through LDS of
// its own: no barrier.  The shares of all waves are dealt as k_attn_tile's, in units of 32 keys.
// UNI: pages hold multiples of 16 rows, which span less than 2^32 bytes, so the 16 rows of a score tile share
// a page, its lookup and the high half of their addresses.
// One read of every key and value: 5.9 TB/s for 670 MB, two units of loads in flight in each of 2048 waves.
template <int QT, int CT, int NS, int DT, bool UNI>
__device__ __forceinline__ void wave_share(const AttnArgs& g, uint4 (&ks)[32][DT / 8], int w, int waves, int UH) {
    using M = Mfma<CT>;
    using T = typename M::T;
    using Q = typename Elem<QT>::type;
    constexpr int KS = DT / 32, NE = DT / 16, VD = DT < 128 ? 2 : 4, VB = DT < 128 ? 1 : DT / 128;
    // units in flight: what 256 registers hold
    constexpr int BUF = UNI && (DT == 64 || (DT == 128 && NS == 1)) ? 2 : 1;
    const Paged& a = g.a;
    const int lane = (int)threadIdx.x & 63, col = lane & 15, lg = lane >> 4;
    const int per = a.D / 8;
    const int64_t U = (int64_t)UH * a.hkv;
    const int n_waves = (int)(U < waves ? U : waves);
    if (w >= n_waves) return;
    int64_t u = unit_of(w, U, n_waves);
    const int64_t u1 = unit_of(w + 1, U, n_waves);
    int head = (int)(u / UH), b = 0, before = 0;  // units of the head before sequence b
    {
        const int in = (int)(u - (int64_t)head * UH);
        for (int b0 = 0;; b0 += 64) {
            int x = b0 + lane < a.B ? (own_rows(a, b0 + lane) + 31) >> 5 : 0;
            const int mine = x;
            for (int d = 1; d < 64; d <<= 1) {
                const int o = __shfl_up(x, d);
                if (lane >= d) x += o;
            }
            const uint64_t over = __ballot(before + x > in);
            if (over != 0 || b0 + 64 >= a.B) {
                const int at = over != 0 ? __builtin_ctzll(over) : 63;
                b = b0 + at;
                before += __shfl(x - mine, at);
                break;
            }
            before += __shfl(x, 63);
        }
        b = __builtin_amdgcn_readfirstlane(b);
        before = __builtin_amdgcn_readfirstlane(before);
    }
    const float sign = g.scale > 0.f ? 1.f : g.scale < 0.f ? -1.f : 0.f;
    const float scale2 = (g.scale == 0.f ? 1.f : __builtin_fabsf(g.scale)) * kLog2e;
    // keys and values beyond the 256 MB of the MALL are read past it (128 -> 114 us for 670 MB); fewer may be there
    // from the call before (27.4 us for 74 MB, 30 read past it)
    const bool stream = U * 32 * a.D * 4 > (int64_t)256 << 20;

    while (u < u1) {
        const int own = own_rows(a, b), nk = (own + 31) >> 5;
        const int in = (int)(u - (int64_t)head * UH);
        if (in >= before + nk) {  // the next sequence, or the next head's first
            before += nk;
            b++;
            if (b == a.B) {
                b = 0;
                before = 0;
                head++;
            }
            continue;
        }
        int kt = in - before;
        const int k0 = kt, k1 = (int)(u1 - u < nk - kt ? kt + (u1 - u) : nk);
        const bool last_word = kt == 0 && k1 == nk && a.P == 0;
        const int64_t slot = slot_of(w, b, a.B, head);
        if (kt == 0 && lane == 0) {
            const int64_t ue = (int64_t)head * UH + before + nk - 1;
            g.where1[(int64_t)head * a.B + b] = make_int2((int)slot, last_word ? 0 : group_of(ue, U, n_waves) - w + 1);
        }
        const int32_t* table = a.table + (int64_t)b * a.table_stride;
        const int64_t hoff = (int64_t)head * a.head_stride;
        const T* kbase = reinterpret_cast<const T*>(a.k) + hoff;
        const T* vbase = reinterpret_cast<const T*>(a.v) + hoff;

        // the rows of units in flight: row 16 (j / 4) + 4 lg + j % 4, 16 lanes across it
        struct Unit {
            u32x4 k[8][VB], v[8][VB];
            uint32_t ok;  // bit j: row j is there
        };
        Unit un[BUF];
        int pg[BUF][2];
        const uint32_t row_bytes = 2u * (uint32_t)a.row_stride, lane_at = 4u * lg * row_bytes + 4u * VD * col;
        const bool all_lanes = a.D == DT;
        auto look = [&](int (&p)[2], int t) {
            if constexpr (UNI) {
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const int i = t * 32 + 16 * x;
                    p[x] = t < k1 && i < own ? load_uniform(table + fdiv(a.page, i)) : -1;
                }
            }
        };
        auto load = [&](u32x4 (&to)[8][VB], uint32_t& oks, const T* base, const int (&p)[2], int t) {
            // a whole unit: two scalar bases, the lane's part the same for each
            if (UNI && all_lanes && t * 32 + 32 <= own && (uint32_t)p[0] < (uint32_t)a.n_pages &&
                (uint32_t)p[1] < (uint32_t)a.n_pages) {
                oks = 255u;
                auto get = [&](auto nt) {
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const int i0 = t * 32 + 16 * x, in_page = i0 - fdiv(a.page, i0) * (int)a.page.d;
                        const auto* at = reinterpret_cast<const uint8_t*>(base + row_at(a, p[x], in_page));
#pragma unroll
                        for (int j = 0; j < 4; j++)
#pragma unroll
                            for (int vb = 0; vb < VB; vb++) {
                                const auto* q = at + (uint32_t)(lane_at + (uint32_t)j * row_bytes + 256 * vb);
                                using R = std::conditional_t<VD == 4, u32x4, u32x2>;
                                const auto* r = reinterpret_cast<const R*>(q);
                                R y;
                                if constexpr (decltype(nt)::value) y = __builtin_nontemporal_load(r);
                                else y = *r;
#pragma unroll
                                for (int d = 0; d < VD; d++) to[4 * x + j][vb][d] = y[d];
                            }
                    }
                };
                if (stream) {
                    asm volatile("");  // keeps the two kinds of load from being merged into one
                    get(std::true_type());
                } else {
                    get(std::false_type());
                }
                return;
            }
            oks = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int x = j >> 2, i0 = t * 32 + 16 * x, i = i0 + 4 * lg + (j & 3);
                int page, in_page;
                if constexpr (UNI) {
                    page = p[x];
                    in_page = i - fdiv(a.page, i0) * (int)a.page.d;
                } else {
                    const int at = fdiv(a.page, i);
                    page = i < own ? table[at] : -1;
                    in_page = i - at * (int)a.page.d;
                }
                const bool ok = page >= 0 && page < a.n_pages && i < own;
                oks |= ok ? 1u << j : 0u;
                const int64_t at = row_at(a, page, in_page);
#pragma unroll
                for (int vb = 0; vb < VB; vb++) {
                    const int d = vb * 128 + 2 * VD * col;
                    to[j][vb] = u32x4{0u, 0u, 0u, 0u};
                    if (ok && d < a.D) {
                        if constexpr (VD == 4) {
                            to[j][vb] = *reinterpret_cast<const u32x4*>(base + at + d);
                        } else {
                            const u32x2 y = *reinterpret_cast<const u32x2*>(base + at + d);
                            to[j][vb][0] = y[0];
                            to[j][vb][1] = y[1];
                        }
                    }
                }
            }
        };
#pragma unroll
        for (int i = 0; i < BUF; i++) look(pg[i], kt + i);
#pragma unroll
        for (int i = 0; i < BUF; i++) {
            if (kt + i >= k1) break;
            load(un[i].k, un[i].ok, kbase, pg[i], kt + i);
            load(un[i].v, un[i].ok, vbase, pg[i], kt + i);
        }

        // the queries
        u32x4 qf[KS][NS];
        float qscale = scale2;
        {
            const bool row = col < g.G;
            const Q* q = reinterpret_cast<const Q*>(g.q) + b * g.qs + (int64_t)(head * g.G + (row ? col : 0)) * a.D;
            float x[KS][8];
            load_query<KS>(q, row, per, lg, sign, x);
            if constexpr (NS > 1 && CT == BPD_T_F16) qscale = score_scale(scale2, row_exponent<KS>(x));
#pragma unroll
            for (int k = 0; k < KS; k++) split8<CT, NS>(x[k], qf[k]);
        }
        f32x4 o[NE];
#pragma unroll
        for (int e = 0; e < NE; e++) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
        float ref = kNegInf, l = 0.f;
        // unit t, held in n; then the unit BUF further on is asked for
        auto step = [&](Unit& n, int (&p)[2], int t) {
            // K's rows through the wave's own LDS into the order of the product's operand: read from memory as
            // the operand takes them, 16 lanes would meet 16 rows at a time
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int vb = 0; vb < VB; vb++) {
                    const int row = 16 * (j >> 2) + 4 * lg + (j & 3);
                    if constexpr (VD == 4)
                        *reinterpret_cast<u32x4*>(&ks[row][k_slot<DT>(row, vb * 16 + col)]) = n.k[j][vb];
                    else
                        reinterpret_cast<u32x2*>(&ks[row][k_slot<DT>(row, col >> 1)])[col & 1] =
                            u32x2{n.k[j][vb][0], n.k[j][vb][1]};
                }
            const uint32_t ok = n.ok;
            const bool more = t + BUF < k1;
            int pn[2] = {p[0], p[1]};
            if (more) {
                load(n.k, n.ok, kbase, pn, t + BUF);
                look(p, t + 2 * BUF);
            }
            u32x4 kf[2][KS];
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int k = 0; k < KS; k++)
                    kf[x][k] = __builtin_bit_cast(u32x4, ks[16 * x + col][k_slot<DT>(col, 4 * k + lg)]);
            f32x4 sc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int y = 0; y < NS; y++) sc[x] = M::go(kf[x][k], qf[k][y], sc[x]);
            // keys that are not there: the lane's scores are those of the rows that it read
            if (__ballot(ok != 255u) != 0) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (!((ok >> e) & 1u)) sc[e >> 2][e & 3] = kNegInf;
            }
            const float top = xor_max(fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                                            fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])))) * qscale;
            if (__ballot(top - 15.f > ref) != 0) {
                const float nr = top - 15.f > ref ? top - 12.f : ref;
                const float f = nr == ref ? 1.f : __builtin_amdgcn_exp2f(ref - nr);
                l *= f;
#pragma unroll
                for (int e = 0; e < NE; e++) o[e] *= f;
                ref = nr;
            }
            const float base = ref == kNegInf ? 0.f : ref;
            float w8[8];
#pragma unroll
            for (int e = 0; e < 8; e++) w8[e] = __builtin_amdgcn_exp2f(fmaf(sc[e >> 2][e & 3], qscale, -base));
            l += ((w8[0] + w8[1]) + (w8[2] + w8[3])) + ((w8[4] + w8[5]) + (w8[6] + w8[7]));
            u32x4 pf[NS];
            split8<CT, NS>(w8, pf);
#pragma unroll
            for (int vb = 0; vb < VB; vb++)
#pragma unroll
                for (int e = 0; e < 2 * VD; e++) {
                    const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
                    u32x4 vf;
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        vf[j] = __builtin_amdgcn_perm(n.v[2 * j + 1][vb][e >> 1], n.v[2 * j][vb][e >> 1], sel);
#pragma unroll
                    for (int x = 0; x < NS; x++) o[vb * 8 + e] = M::go(vf, pf[x], o[vb * 8 + e]);
                }
            if (more) load(n.v, n.ok, vbase, pn, t + BUF);
        };
        // the pages of the units behind those in flight
#pragma unroll
        for (int i = 0; i < BUF; i++) look(pg[i], kt + BUF + i);
        while (true) {
#pragma unroll
            for (int i = 0; i < BUF; i++) {
                if (kt + i >= k1) break;
                step(un[i], pg[i], kt + i);
            }
            kt += BUF;
            if (kt >= k1) break;
        }
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (col < g.G) {
            const int h = head * g.G + col;
            if (last_word) {
                const float inv = l != 0.f ? 1.f / l : 0.f;
                Q* out = reinterpret_cast<Q*>(g.out) + b * g.os + (int64_t)h * a.D;
                store_row<Q, VD, VB>(out, a.D, lg, o, inv);
                if (g.lse != nullptr && lg == 0)
                    g.lse[(int64_t)b * g.H + h] = l != 0.f ? (ref + __builtin_log2f(l)) * kLn2 : kNegInf;
            } else {
                store_row<float, VD, VB>(g.part1 + (slot * g.G + col) * DT, DT, lg, o, 1.f);
                if (lg == 0) g.ml1[slot * g.G + col] = make_float2(ref, l);
            }
        }
        u += k1 - k0;
    }
}

// Units of 32 keys of one kv head's sequences.
__device__ __forceinline__ int wave_units(const Paged& a) {
    int n = 0;
    for (int b = (int)threadIdx.x & 63; b < a.B; b += 64) n += (own_rows(a, b) + 31) >> 5;
    for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d);
    return __builtin_amdgcn_readfirstlane(n);
}

// Workgroups go to the 8 XCDs in turn: each XCD takes an eighth of the tiles' shares in a row.
__device__ __forceinline__ int xcd_share(int block, int groups) {
    return groups % 8 == 0 ? (block & 7) * (groups >> 3) + (block >> 3) : block;
}

template <int QT, int CT, int NS, int DT, int MT, int NW, bool UNI>
__global__ __launch_bounds__(64 * NW, DT == 256 ? 1 : 2) void k_attn_tile(AttnArgs g) {
    __shared__ Lds<DT> s;
    tile_share<QT, CT, NS, DT, MT, NW, UNI>(g, s, xcd_share((int)blockIdx.x, g.groups), g.groups);
}

template <int QT, int CT, int NS, int DT, bool UNI>
__global__ __launch_bounds__(256, DT == 256 ? 1 : 2) void k_attn_wave(AttnArgs g) {
    __shared__ uint4 ks[4][32][DT / 8];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    wave_share<QT, CT, NS, DT, UNI>(g, ks[wave], (int)blockIdx.x * 4 + wave, g.waves, wave_units(g.a));
}

// One token per sequence behind a prefix: x of the workgroups take the prefix's tiles, which the matrix
// units bound, the others the sequences' own keys, which memory bounds, at the same time.  x by
// the time that a unit of each takes a CU: tile_cost (64 keys x R rows) against wave_cost (32 keys x 16).
template <int QT, int CT, int NS, int DT, int MT, int NW, bool UNI>
__global__ __launch_bounds__(64 * NW, DT == 256 ? 1 : 2) void k_attn_both(AttnArgs g) {
    __shared__ union {
        Lds<DT> tile;
        uint4 k[NW][32][DT / 8];
    } s;
    const Paged& a = g.a;
    const int uw = wave_units(a), eighths = g.groups >> 3;
    const float ct = (float)(((a.T * g.G + g.R - 1) / g.R) * units_of(a.P)) * g.tile_cost, cw = (float)uw * g.wave_cost;
    const int x8 = cw == 0.f ? eighths : max(1, min(eighths - 1, (int)((float)eighths * ct / (ct + cw) + 0.5f)));
    const int row = (int)blockIdx.x >> 3;
    if (row < x8) {
        tile_share<QT, CT, NS, DT, MT, NW, UNI>(g, s.tile, ((int)blockIdx.x & 7) * x8 + row, 8 * x8);
    } else {
        const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
        const int w = (((int)blockIdx.x & 7) * (eighths - x8) + row - x8) * NW + wave;
        wave_share<QT, CT, NS, DT, UNI>(g, s.k[wave], w, 8 * (eighths - x8) * NW, uw);
    }
}

// Whether a row that token i of n new ones of sequence b sees is there.  The whole wave.
__device__ __forceinline__ bool sees_a_row(const Paged& a, int b, int n, int i) {
    const int lane = (int)threadIdx.x & 63, own = seen_rows(a, b, n, i, own_rows(a, b));
    auto any = [&](const int32_t* pages, int rows) {
        const int used = rows > 0 ? fdiv(a.page, rows - 1) + 1 : 0;
        for (int p0 = 0; p0 < used; p0 += 64) {
            const int page = p0 + lane < used ? pages[p0 + lane] : -1;
            if (__ballot(page >= 0 && page < a.n_pages) != 0) return true;
        }
        return false;
    };
    return any(a.prefix, a.P) || any(a.table + (int64_t)b * a.table_stride, own);
}

// Joins what was left of each (token, query head): its packed results, then its sequence's.  A
// workgroup takes a token and HW heads for each of its 4 waves; a lane looks up one of the wave's heads.
// Three dependent lookups and the results bound it: 8 us at 64 tokens of 32 heads, 12 at 256, 21 at 3,070.
// A query with infinities or NaN has NaN for k_attn_tile's rows that are not there too (0 times infinity).  Where all
// are absent the result is that of no row; that is looked for here, as a mask within the tiles' loop or at their items'
// ends took 2 % of the prompt chunks' time.
template <int QT, int HW>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs g) {
    using Q = typename Elem<QT>::type;
    const Paged& a = g.a;
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int t = (int)blockIdx.x, h0 = ((int)blockIdx.y * 4 + wave) * HW;
    if (h0 >= g.H) return;
    int b = t;
    if (a.q_start != nullptr) {
        b = __builtin_amdgcn_readfirstlane(count_le(a.q_start, a.B + 1, t) - 1);
        if (b < 0 || b >= a.B) return;
    }
    int t0, n;
    seq_tokens(a, b, t0, n);
    const int i = t - t0;
    if (i < 0 || i >= n) return;  // offsets that decrease: the token is not really the sequence's
    int2 wp = make_int2(0, 0), wo = make_int2(0, 0);  // this lane's head: packed results, the sequence's
    int rp = 0, ro = 0;
    bool done = lane >= HW || h0 + lane >= g.H;
    if (!done) {
        const int h = h0 + lane, head = fdiv(g.g, h), gq = h - head * g.G;
        if (g.planned) {
            const int nitems = g.p.info[0];
            const bool packed = a.P > 0 && !is_joint(g, n);
            const int at = packed ? g.p.place[t] : -1;
            if (at >= 0) {
                const int r = at * g.G + gq, item = r / g.R;
                if (item < nitems) wp = g.where[(int64_t)head * nitems + item];
                rp = r - item * g.R;
            }
            const int r = i * g.G + gq, rt = r / g.R, item = g.p.item0[b] + rt;
            if (item < nitems && g.p.first[item + 1] > g.p.first[item]) {
                wo = g.where[(int64_t)head * nitems + item];
                done = wo.y == 0;
            }
            ro = r - rt * g.R;
        } else {
            if (a.P > 0) {
                const int r = t * g.G + gq, item = r / g.R, nitems = (a.T * g.G + g.R - 1) / g.R;
                wp = g.where[(int64_t)head * nitems + item];
                rp = r - item * g.R;
            }
            if (own_rows(a, b) > 0) {
                wo = g.where1[(int64_t)head * a.B + b];
                done = wo.y == 0;
            }
            ro = gq;
        }
    }
    const float* part1 = g.planned ? g.part : g.part1;
    const float2* ml1 = g.planned ? g.ml : g.ml1;
    const int R1 = g.planned ? g.R : g.G;
    if (g.planned) {  // results that were written, but are NaN
        Q* out = reinterpret_cast<Q*>(g.out) + t * g.os + (int64_t)(h0 + lane) * a.D;
        const bool odd = done && lane < HW && h0 + lane < g.H && (float)out[0] != (float)out[0];
        if (__ballot(odd) != 0 && !sees_a_row(a, b, n, i) && odd) {
            for (int d = 0; d < a.D; d++) out[d] = (Q)0.f;
            if (g.lse != nullptr) g.lse[(int64_t)t * g.H + h0 + lane] = kNegInf;
        }
    }
    uint64_t todo = __ballot(!done);
    // a row of the head in 16-byte pieces by DT / 4 lanes: 64 / (DT / 4) results at a time
    const int lanes = g.DT >> 2, sub = lane / lanes, piece = lane - sub * lanes, step = 64 / lanes;
    constexpr int FEW = 4;
    if (HW > 1 && __ballot(!done && wp.y + wo.y > FEW) == 0) {
        // few results each: a lane weighs its head's, then each group of lanes adds up a head
        const int64_t sp = (int64_t)wp.x * g.R + rp, so = (int64_t)wo.x * R1 + ro;
        float2 x[FEW];
        float m = kNegInf, l = 0.f, f[FEW];
#pragma unroll
        for (int k = 0; k < FEW; k++) {
            x[k] = make_float2(kNegInf, 0.f);
            if (!done && k < wp.y + wo.y)
                x[k] = k < wp.y ? g.ml[sp + (int64_t)k * g.R] : ml1[so + (int64_t)(k - wp.y) * R1];
            m = fmaxf(m, x[k].x);
        }
#pragma unroll
        for (int k = 0; k < FEW; k++) {
            f[k] = x[k].x == kNegInf ? (x[k].y != 0.f ? x[k].y : 0.f) : __builtin_amdgcn_exp2f(x[k].x - m);
            l += x[k].y * f[k];
        }
        if (__ballot(!done && l != l) != 0 && !sees_a_row(a, b, n, i)) l = 0.f;
        const bool any = l != 0.f;
        if (!done && g.lse != nullptr)
            g.lse[(int64_t)t * g.H + h0 + lane] = any ? (m + __builtin_log2f(l)) * kLn2 : kNegInf;
#pragma unroll
        for (int k = 0; k < FEW; k++) f[k] = any ? f[k] / l : 0.f;
#pragma unroll 4
        for (int j0 = 0; j0 < HW; j0 += step) {
            const int j = j0 + sub;  // below 64: HW is 8 at most, sub 4
            const int np = __shfl(wp.y, j), n = np + __shfl(wo.y, j);
            const int64_t p0 = __shfl(sp, j), p1 = __shfl(so, j);
            const bool skip = __shfl((int)done, j) != 0 || j >= HW;
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < FEW; k++) {
                const float fk = __shfl(f[k], j);
                if (skip || k >= n || fk == 0.f) continue;  // nothing, or what is not there
                const float* p = k < np ? g.part + (p0 + (int64_t)k * g.R) * g.DT
                                        : part1 + (p1 + (int64_t)(k - np) * R1) * g.DT;
                acc += *reinterpret_cast<const f32x4*>(p + 4 * piece) * fk;
            }
            if (!skip && 4 * piece < a.D) {
                Vec<Q, 4> v;
#pragma unroll
                for (int c = 0; c < 4; c++) v.v[c] = (Q)acc[c];
                Q* to = reinterpret_cast<Q*>(g.out) + t * g.os + (int64_t)(h0 + j) * a.D + 4 * piece;
                *reinterpret_cast<Vec<Q, 4>*>(to) = v;
            }
        }
        return;
    }
    while (todo != 0) {
        const int j = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int np = __shfl(wp.y, j), no = __shfl(wo.y, j);
        const int64_t sp = (int64_t)__shfl(wp.x, j) * g.R + __shfl(rp, j);
        const int64_t so = (int64_t)__shfl(wo.x, j) * R1 + __shfl(ro, j);
        auto ml_at = [&](int k) {
            return k < np ? g.ml[sp + (int64_t)k * g.R] : ml1[so + (int64_t)(k - np) * R1];
        };
        float m = kNegInf;
        for (int k = lane; k < np + no; k += 64) m = fmaxf(m, ml_at(k).x);
        for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
        float l = 0.f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int k0 = 0; k0 < np + no; k0 += 64) {
            float f = 0.f;  // the weight of result k0 + lane
            if (k0 + lane < np + no) {
                const float2 x = ml_at(k0 + lane);
                // an untouched result (-inf, 0) weighs nothing; one of NaN scores alone keeps its NaN
                f = x.x == kNegInf ? (x.y != 0.f ? x.y : 0.f) : __builtin_amdgcn_exp2f(x.x - m);
                l += x.y * f;
            }
            const int top = min(64, np + no - k0);
            for (int k = 0; k < top; k += 4 * step) {
                f32x4 v[4];
                float fk[4];
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int kx = k + x * step + sub, kk = k0 + kx;
                    fk[x] = __shfl(f, kx & 63);
                    v[x] = f32x4{0.f, 0.f, 0.f, 0.f};
                    if (kx >= top) fk[x] = 0.f;
                    if (fk[x] != 0.f)  // nothing, or what is not there
                        v[x] = *reinterpret_cast<const f32x4*>(
                            (kk < np ? g.part + (sp + (int64_t)kk * g.R) * g.DT
                                     : part1 + (so + (int64_t)(kk - np) * R1) * g.DT) + 4 * piece);
                }
#pragma unroll
                for (int x = 0; x < 4; x++) acc += v[x] * fk[x];
            }
        }
        for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
        for (int d = lanes; d < 64; d <<= 1)
#pragma unroll
            for (int c = 0; c < 4; c++) acc[c] += __shfl_xor(acc[c], d);
        if (l != l && !sees_a_row(a, b, n, i)) {
            l = 0.f;
            acc = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        const bool any = l != 0.f;
        const float inv = any ? 1.f / l : 0.f;
        const int h = h0 + j;
        if (sub == 0 && 4 * piece < a.D) {
            Vec<Q, 4> v;
#pragma unroll
            for (int c = 0; c < 4; c++) v.v[c] = (Q)(acc[c] * inv);
            *reinterpret_cast<Vec<Q, 4>*>(reinterpret_cast<Q*>(g.out) + t * g.os + (int64_t)h * a.D + 4 * piece) = v;
        }
        if (g.lse != nullptr && lane == 0)
            g.lse[(int64_t)t * g.H + h] = any ? (m + __builtin_log2f(l)) * kLn2 : kNegInf;
    }
}

// ---------------------------------------------------------------- host

bool planned_way(const int32_t* q_start, int G) { return q_start != nullptr || G > 16; }

template <int QT, int CT, int NS, int DT, int MT, int NW, bool UNI>
void launch_dim(const AttnArgs& g, hipStream_t s) {
    const dim3 grid((unsigned)g.groups), block(64 * NW);
    if (g.planned)
        hipLaunchKernelGGL((k_attn_tile<QT, CT, NS, DT, MT, NW, UNI>), grid, block, 0, s, g);
    else if (g.a.P > 0 && g.a.W > 0)
        hipLaunchKernelGGL((k_attn_both<QT, CT, NS, DT, MT, NW, UNI>), grid, block, 0, s, g);
    else if (g.a.P > 0)
        hipLaunchKernelGGL((k_attn_tile<QT, CT, NS, DT, MT, NW, UNI>), grid, block, 0, s, g);
    else if (g.a.W > 0)
        hipLaunchKernelGGL((k_attn_wave<QT, CT, NS, DT, UNI>), dim3((unsigned)(g.waves / 4)), dim3(256), 0, s, g);
}

template <int QT, int CT, int NS, bool UNI>
void launch_uni(const AttnArgs& g, hipStream_t s) {
    if (g.DT == 64) launch_dim<QT, CT, NS, 64, 2, 8, UNI>(g, s);
    else if (g.DT == 128) launch_dim<QT, CT, NS, 128, NS == 1 ? 2 : 1, 8, UNI>(g, s);
    else launch_dim<QT, CT, NS, 256, 1, 4, UNI>(g, s);
}

template <int QT, int CT, int NS>
void launch_types(const AttnArgs& g, hipStream_t s) {
    if (g.planned) hipLaunchKernelGGL(k_attn_plan, dim3(1), dim3(1024), 0, s, g);
    if (g.a.page.d % 16 == 0 && g.a.row_stride < 1 << 26) launch_uni<QT, CT, NS, true>(g, s);
    else launch_uni<QT, CT, NS, false>(g, s);
    // one head per wave while that fills the chip twice at most, more where most rows are done
    if ((int64_t)g.a.T * g.H <= 32768)
        hipLaunchKernelGGL((k_attn_join<QT, 1>), dim3((unsigned)g.a.T, (unsigned)((g.H + 3) / 4)), dim3(256), 0, s, g);
    else
        hipLaunchKernelGGL((k_attn_join<QT, 8>), dim3((unsigned)g.a.T, (unsigned)((g.H + 31) / 32)), dim3(256), 0, s,
                           g);
}

}  // namespace

int64_t attn_paged_ws(const int32_t* q_start, int B, int T, int H, int HKV, int D, int P) {
    const int G = H / HKV, DT = padded(D);  // for either type of q
    const bool pl = planned_way(q_start, G);
    const int64_t x = sizes(pl, B, T, G, HKV, rows_of(D, 1), DT, P).total;
    const int64_t y = sizes(pl, B, T, G, HKV, rows_of(D, 2), DT, P).total;
    return x > y ? x : y;
}

void launch_attn_paged(const Paged& a0, int cache_type, const void* q, int64_t qs, void* out, int64_t os, float* lse,
                       int q_type, int H, float scale, void* ws, hipStream_t s) {
    Paged a = a0;
    if (a.n_pages == 0) a.W = a.P = 0;  // no row is there
    AttnArgs g = {};
    g.a = a;
    g.q = static_cast<const uint8_t*>(q);
    g.out = static_cast<uint8_t*>(out);
    g.qs = qs;
    g.os = os;
    g.lse = lse;
    g.H = H;
    g.G = H / a.hkv;
    g.g = fast_div(g.G);
    g.scale = scale;
    g.R = rows_of(a.D, q_type == BPD_T_F32 ? 2 : 1);
    g.DT = padded(a.D);
    g.groups = kGroups;
    g.waves = kStreamWaves;
    // us of a CU: 64 keys x 256 rows of 128 by 8 waves (630 TFLOP/s), 32 keys of 128 (a CU draws 34 GB/s beside the
    // others)
    const int parts = q_type != BPD_T_F32 ? 1 : cache_type == BPD_T_BF16 ? 3 : 2;
    g.tile_cost = 3.4f * (float)(g.R * g.DT * parts) / (256.f * 128.f) * (g.DT == 256 ? 2.f : 1.f);
    g.wave_cost = 0.48f * (float)g.DT / 128.f;
    g.planned = planned_way(a.q_start, g.G);
    const Sizes z = sizes(g.planned, a.B, a.T, g.G, a.hkv, g.R, g.DT, a.P);
    uint8_t* at = static_cast<uint8_t*>(ws);
    auto take = [&](int64_t n) {
        uint8_t* p = at;
        at += n;
        return p;
    };
    int32_t* p = reinterpret_cast<int32_t*>(take(z.ints));
    g.p.info = p;
    g.p.first = p + 4;
    g.p.seq = g.p.first + z.items + 1;
    g.p.rt = g.p.seq + z.items;
    g.p.item0 = g.p.rt + z.items;
    g.p.packed = g.p.item0 + a.B;
    g.p.place = g.p.packed + a.T;
    g.part = reinterpret_cast<float*>(take(z.part));
    g.ml = reinterpret_cast<float2*>(take(z.ml));
    g.where = reinterpret_cast<int2*>(take(z.where));
    g.part1 = reinterpret_cast<float*>(take(z.part1));
    g.ml1 = reinterpret_cast<float2*>(take(z.ml1));
    g.where1 = reinterpret_cast<int2*>(take(z.where1));
    const bool bf = cache_type == BPD_T_BF16;
    if (q_type == BPD_T_F32 && bf) launch_types<BPD_T_F32, BPD_T_BF16, 3>(g, s);
    else if (q_type == BPD_T_F32) launch_types<BPD_T_F32, BPD_T_F16, 2>(g, s);
    else if (bf) launch_types<BPD_T_BF16, BPD_T_BF16, 1>(g, s);
    else launch_types<BPD_T_F16, BPD_T_F16, 1>(g, s);
}

}  // namespace bpdq
