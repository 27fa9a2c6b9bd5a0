// paged_attn.hip — bpd_attn_paged_gpu: attention over a paged cache.
//
//   s_i = scale q.k_i,  out = sum_i exp(s_i - m) v_i / sum_i exp(s_i - m),  m = max s_i,
//   lse = m + log sum_i exp(s_i - m)
//
// in one pass over the keys: a row of a query head keeps a reference exponent r (base 2), its
// sum l = sum 2^(s - r) and O = sum 2^(s - r) v in fp32.  Where a later part of the
// keys has another reference, sums join as O 2^(r - r') + O' (k_attn_join).
//
// Work.  The query heads of one kv head share its keys, so a row is a (token, query head)
// pair and a tile is R rows of one kv head against 64 keys at a time.  An item is a tile's
// rows with all their keys:
//   - own items: the rows of one sequence against its own keys, causal, and where a
//     sequence fills half a tile by itself, the prefix before them;
//   - packed items: the rows of all other sequences together against the prefix, which is so
//     read once for R / (heads per kv head) sequences.
// Units of 64 keys, item by item, are dealt evenly to the workgroups, whose number does
// not depend on the batch: a workgroup runs through its units, and where an item ends in the
// middle leaves its O, r and l for k_attn_join, in a place of its own.  The plan (k_attn_plan) is
// made on the device, as the lengths are there.
#include "bpdq_paged.h"

namespace bpdq {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kKeys = 64;   // keys of a unit
constexpr int kGroups = 512;  // workgroups that share the units: 2 per CU
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
    int R, DT;  // rows of a tile, padded head size
    Plan p;
    float* part;  // [slot][R][DT]
    float2* ml;   // [slot][R] reference exponent, sum
};

__host__ __device__ constexpr int round64(int v) { return (v + 63) / 64; }
__device__ __forceinline__ int64_t slot_of(int group, int item, int hkv, int h) {
    return (int64_t)group + (int64_t)item * hkv + h;
}
// Units are dealt as [w U / n, (w + 1) U / n) to workgroup w of n = min(kGroups, U).
__device__ __forceinline__ int64_t unit_of(int w, int64_t U, int n) { return w * U / n; }
__device__ __forceinline__ int group_of(int64_t u, int64_t U, int n) { return (int)(((u + 1) * n - 1) / U); }

// Rows of a sequence's own part that the table holds.
__device__ __forceinline__ int own_rows(const Paged& a, int b) {
    return max(0, min(a.lens[b], a.W * (int)a.page.d));
}
__device__ __forceinline__ bool is_joint(const AttnArgs& g, int n) { return n * g.G * 2 >= g.R; }

// Whole own rows that row `last` (token index within the sequence) of a tile can see.
__device__ __forceinline__ int seen_rows(const Paged& a, int b, int n, int i, int own) {
    const int64_t s = (int64_t)a.lens[b] - n + i + 1;
    return (int)(s < 0 ? 0 : s > own ? own : s);
}

// One workgroup lays out the items.  Sequences are taken 256 at a time, a thread each.
__global__ __launch_bounds__(256) void k_attn_plan(AttnArgs g) {
    __shared__ int s_scan[256];
    __shared__ int s_run[3];
    const Paged& a = g.a;
    const int tid = (int)threadIdx.x;
    const int ntp = round64(a.P);
    auto scan = [&](int v) {  // exclusive over the workgroup, the total in s_scan[255] + v of the last
        s_scan[tid] = v;
        __syncthreads();
        for (int d = 1; d < 256; d <<= 1) {
            const int o = tid >= d ? s_scan[tid - d] : 0;
            __syncthreads();
            s_scan[tid] += o;
            __syncthreads();
        }
        const int r = s_scan[tid] - v, total = s_scan[255];
        __syncthreads();
        return make_int2(r, total);
    };
    // the packed rows
    int packed = 0;
    if (a.P > 0)
        for (int b0 = 0; b0 < a.B; b0 += 256) {
            const int b = b0 + tid;
            int t0 = 0, n = 0;
            if (b < a.B) seq_tokens(a, b, t0, n);
            const bool in = n > 0 && !is_joint(g, n);
            const int2 at = scan(in ? n : 0);
            for (int i = 0; i < n; i++) {
                const int k = packed + at.x + i;
                if (in && k < a.T) g.p.packed[k] = t0 + i;
                g.p.place[t0 + i] = in && k < a.T ? k : -1;
            }
            packed += at.y;
        }
    packed = min(packed, a.T);
    const int np = packed > 0 ? (packed * g.G + g.R - 1) / g.R : 0;
    for (int i = tid; i < np; i += 256) {
        g.p.first[i] = i * ntp;
        g.p.seq[i] = -1;
        g.p.rt[i] = i;
    }
    int items = np, units = np * ntp;
    // most items there can be: overlapping sequences (offsets that decrease) stop the plan there
    const int most = np + a.B + (int)(((int64_t)a.T * g.G) / g.R);
    for (int b0 = 0; b0 < a.B; b0 += 256) {
        const int b = b0 + tid;
        int t0 = 0, n = 0;
        if (b < a.B) seq_tokens(a, b, t0, n);
        const int own = b < a.B ? own_rows(a, b) : 0;
        const int nrt = n > 0 ? (n * g.G + g.R - 1) / g.R : 0;
        const int pre = n > 0 && is_joint(g, n) ? ntp : 0;
        int mine = 0;
        for (int r = 0; r < nrt; r++)
            mine += pre + round64(seen_rows(a, b, n, min(n, ((r + 1) * g.R - 1) / g.G + 1) - 1, own));
        const int2 ai = scan(nrt), au = scan(mine);
        if (b < a.B) g.p.item0[b] = items + ai.x;
        int u = units + au.x;
        for (int r = 0; r < nrt; r++) {
            const int k = items + ai.x + r;
            if (k >= most) break;
            g.p.first[k] = u;
            g.p.seq[k] = b;
            g.p.rt[k] = r;
            u += pre + round64(seen_rows(a, b, n, min(n, ((r + 1) * g.R - 1) / g.G + 1) - 1, own));
            if (k + 1 == most) s_run[0] = u;
        }
        items += ai.y;
        units += au.y;
    }
    __syncthreads();
    if (items > most) {
        items = most;
        units = s_run[0];
    }
    if (tid == 0) {
        g.p.first[items] = units;
        g.p.info[0] = items;
        g.p.info[1] = units;
        g.p.info[2] = packed;
    }
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
    using T = typename Mfma<CT>::T;
    using V = typename Mfma<CT>::V;
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = x[i];
#pragma unroll
    for (int s = 0; s < NS; s++) {
        V v;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            v[i] = (T)r[i];
            if (s + 1 < NS) r[i] -= (float)v[i];
        }
        out[s] = __builtin_bit_cast(u32x4, v);
    }
}

// Which 16-byte chunk slot of a K row in LDS holds chunk c: rows of a 16-lane operand read
// differ in it, so that the read meets every bank once.
template <int DT>
__device__ __forceinline__ int k_slot(int row, int c) {
    return DT == 64 ? c ^ ((row >> 1) & 7) : c ^ (row & 15);
}

template <int DT>
struct Lds {
    uint4 k[2][kKeys][DT / 8];
    uint4 v[2][kKeys][DT / 8];
    float bias[2][kKeys];  // 0, or -inf for a row that is not there
};

// Whether any of 8 packed 16-bit values is an infinity or NaN.
template <int CT>
__device__ __forceinline__ bool not_finite(uint32_t d) {
    constexpr uint32_t e = CT == BPD_T_F16 ? 0x7C00u : 0x7F80u;
    return (d & e) == e || ((d >> 16) & e) == e;
}

template <int CT>
__device__ __forceinline__ uint32_t finite_or_0(uint32_t d) {
    constexpr uint32_t e = CT == BPD_T_F16 ? 0x7C00u : 0x7F80u;
    return ((d & e) == e ? 0u : d & 0xFFFFu) | (((d >> 16) & e) == e ? 0u : d & 0xFFFF0000u);
}

// 4 waves of 16 MT rows each, the units [u0, u1) of this workgroup.  Scores are taken as
// S^T = K Q^T (lane: query l % 16, keys 4 (l / 16) + r), which is the layout in which
// O^T = V^T P^T takes P: the 32 keys of two score tiles in the order 4g..4g+3, 16+4g..16+4g+3 of
// lane group g.  V's operand is read in that order of rows, 16 bytes of each, and
// transposed in registers; row c of it stands for element 8c + e of the head in product e.
template <int QT, int CT, int NS, int DT, int MT>
__global__ __launch_bounds__(256, DT == 256 ? 1 : 2) void k_attn_tile(AttnArgs g) {
    using M = Mfma<CT>;
    using T = typename M::T;
    using Q = typename Elem<QT>::type;
    constexpr int CPR = DT / 8;           // 16-byte chunks of a row
    constexpr int NI = kKeys * CPR / 256;  // chunks of K and of V that a thread moves per unit
    constexpr int KS = DT / 32;           // products of a score tile
    constexpr int NE = DT / 16;           // products of O
    constexpr int VD = DT < 128 ? 2 : 4;  // dwords of a V row in one operand read
    constexpr int VB = DT < 128 ? 1 : DT / 128;
    static_assert(NI >= 1, "a chunk per thread");
    __shared__ Lds<DT> s;
    const Paged& a = g.a;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, lg = lane >> 4;
    const int nitems = g.p.info[0];
    const int64_t U = (int64_t)g.p.info[1] * a.hkv;
    const int n_groups = (int)(U < kGroups ? U : kGroups);
    const int w = (int)blockIdx.x;
    if (w >= n_groups) return;
    int64_t u = unit_of(w, U, n_groups);
    const int64_t u1 = unit_of(w + 1, U, n_groups);
    const int per = a.D / 8;  // chunks that exist
    const float sign = g.scale > 0.f ? 1.f : g.scale < 0.f ? -1.f : 0.f;
    const float scale2 = (g.scale == 0.f ? 1.f : __builtin_fabsf(g.scale)) * kLog2e;

    while (u < u1) {
        // ---- the item of unit u
        const int per_head = (int)(u / a.hkv);
        const int item = __builtin_amdgcn_readfirstlane(count_le(g.p.first, nitems, per_head) - 1);
        const int f0 = g.p.first[item], nk = g.p.first[item + 1] - f0;
        const int64_t in = u - (int64_t)f0 * a.hkv;
        const int head = (int)(in / nk);
        int kt = (int)(in - (int64_t)head * nk);
        const int k1 = (int)(u1 - u < nk - kt ? kt + (u1 - u) : nk);
        const bool whole = kt == 0 && k1 == nk;
        const int b = g.p.seq[item], rt = g.p.rt[item];
        int t0 = 0, n = 0, own = 0, ntp = round64(a.P);
        if (b >= 0) {
            seq_tokens(a, b, t0, n);
            own = own_rows(a, b);
            if (!is_joint(g, n)) ntp = 0;
        } else {
            n = g.p.info[2];
        }
        const int64_t hoff = (int64_t)head * a.head_stride;
        const int32_t* table = b >= 0 ? a.table + (int64_t)b * a.table_stride : nullptr;

        // ---- this wave's queries
        u32x4 qf[MT][KS][NS];
        float qscale[MT];
        int lim[MT];  // own keys that the lane's query sees, -1: no query
        int tok[MT], hq[MT];
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const int row = rt * g.R + (wave * MT + m) * 16 + col;
            const int i = fdiv(g.g, row);
            hq[m] = head * g.G + (row - i * g.G);
            lim[m] = -1;
            tok[m] = -1;
            float top = 0.f;
            float x[KS][8];
            if (i < n) {
                tok[m] = b >= 0 ? t0 + i : g.p.packed[i];
                lim[m] = b >= 0 ? seen_rows(a, b, n, i, own) : 0;
                const Q* q = reinterpret_cast<const Q*>(g.q) + tok[m] * g.qs + (int64_t)hq[m] * a.D;
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    const int c = 4 * k + lg;
                    if (c < per) {
                        const Vec<Q, 8> v = *reinterpret_cast<const Vec<Q, 8>*>(q + 8 * c);
#pragma unroll
                        for (int e = 0; e < 8; e++) x[k][e] = sign == 1.f ? (float)v.v[e] : (float)v.v[e] * sign;
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e++) x[k][e] = 0.f;
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < KS; k++)
#pragma unroll
                    for (int e = 0; e < 8; e++) x[k][e] = 0.f;
            }
            qscale[m] = scale2;
            if constexpr (NS > 1 && CT == BPD_T_F16) {
                // an fp32 row scaled by a power of two to a largest element in [1, 2), so that two
                // binary16 parts keep 22 bits of that
#pragma unroll
                for (int k = 0; k < KS; k++)
#pragma unroll
                    for (int e = 0; e < 8; e++) top = fmaxf(top, __builtin_fabsf(x[k][e]));
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                int e2 = (int)((__float_as_uint(top) >> 23) & 255) - 127;
                if (top == 0.f || e2 == 128) e2 = 0;
                e2 = max(e2, -100);
#pragma unroll
                for (int k = 0; k < KS; k++)
#pragma unroll
                    for (int e = 0; e < 8; e++) x[k][e] = ldexpf(x[k][e], -e2);
                qscale[m] = ldexpf(scale2, e2);
            }
#pragma unroll
            for (int k = 0; k < KS; k++) split8<CT, NS>(x[k], qf[m][k]);
        }
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

        // ---- staging of one unit's rows: a thread moves chunk slot tid % CPR of rows tid / CPR + 256 / CPR j
        const int srow = tid / CPR, sc = tid % CPR;
        int pg[NI];
        uint4 rk[NI], rv[NI];
        bool rin[NI];
        auto key_of = [&](int t, int j, int& i, int& top) {
            const bool pre = t < ntp;
            i = (pre ? t : t - ntp) * kKeys + srow + (256 / CPR) * j;
            top = pre ? a.P : own;
            return pre ? a.prefix : table;
        };
        auto look = [&](int t) {  // the pages of unit t's rows
#pragma unroll
            for (int j = 0; j < NI; j++) {
                int i, top;
                const int32_t* tab = key_of(t, j, i, top);
                pg[j] = i < top ? tab[fdiv(a.page, i)] : -1;
            }
        };
        auto load = [&](int t) {
#pragma unroll
            for (int j = 0; j < NI; j++) {
                int i, top;
                key_of(t, j, i, top);
                rin[j] = pg[j] >= 0 && pg[j] < a.n_pages;
                rk[j] = rv[j] = make_uint4(0, 0, 0, 0);
                if (rin[j] && sc < per) {
                    const int64_t at = pg[j] * a.page_stride + (i - fdiv(a.page, i) * (int)a.page.d) * a.row_stride +
                                       hoff + 8 * sc;
                    rk[j] = *reinterpret_cast<const uint4*>(a.k + 2 * at);
                    rv[j] = *reinterpret_cast<const uint4*>(a.v + 2 * at);
                }
            }
        };
        auto store = [&](int buf) {
#pragma unroll
            for (int j = 0; j < NI; j++) {
                const int row = srow + (256 / CPR) * j;
                s.k[buf][row][k_slot<DT>(row, sc)] = rk[j];
                s.v[buf][row][sc] = rv[j];
                if (sc == 0) s.bias[buf][row] = rin[j] ? 0.f : kNegInf;
            }
        };
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
                    f32x4 sc4[2][MT];
#pragma unroll
                    for (int kk = 0; kk < 2; kk++) {
                        const int r0 = half * 32 + kk * 16;
                        const f32x4 bias = *reinterpret_cast<const f32x4*>(&s.bias[buf][r0 + 4 * lg]);
#pragma unroll
                        for (int m = 0; m < MT; m++) sc4[kk][m] = bias;
#pragma unroll
                        for (int k = 0; k < KS; k++) {
                            const u32x4 kf = __builtin_bit_cast(u32x4, s.k[buf][r0 + col][k_slot<DT>(col, 4 * k + lg)]);
#pragma unroll
                            for (int m = 0; m < MT; m++)
#pragma unroll
                                for (int x = 0; x < NS; x++) sc4[kk][m] = M::go(kf, qf[m][k][x], sc4[kk][m]);
                        }
                    }
                    bool diag = false;
                    if (kt >= ntp && b >= 0) {
                        bool d = false;
#pragma unroll
                        for (int m = 0; m < MT; m++) d |= lim[m] >= 0 && lim[m] < min(own, key0 + half * 32 + 32);
                        diag = __ballot(d) != 0;
                    }
                    u32x4 pf[MT][NS];
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        float x[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) x[e] = sc4[e >> 2][m][e & 3] * qscale[m];
                        if (diag) {
#pragma unroll
                            for (int e = 0; e < 8; e++)
                                if (key0 + half * 32 + (e >> 2) * 16 + 4 * lg + (e & 3) >= lim[m]) x[e] = kNegInf;
                        }
                        float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                                          fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
                        top = fmaxf(top, __shfl_xor(top, 16));
                        top = fmaxf(top, __shfl_xor(top, 32));
                        // weights are 2^(x - ref) with the largest met so far between 2^12 and 2^15:
                        // binary16 weights stay normal 26 binary places below it
                        const bool grow = top - 15.f > ref[m];
                        if (__ballot(grow) != 0) {
                            const float nr = grow ? top - 12.f : ref[m];
                            const float f = ref[m] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(ref[m] - nr);
                            if (grow) {
                                l[m] *= f;
#pragma unroll
                                for (int e = 0; e < NE; e++) o[m][e] *= f;
                                ref[m] = nr;
                            }
                        }
                        const float base = ref[m] == kNegInf ? 0.f : ref[m];
                        float p[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            p[e] = __builtin_amdgcn_exp2f(x[e] - base);
                            l[m] += p[e];
                        }
                        split8<CT, NS>(p, pf[m]);
                    }
                    // ---- O^T += V^T P^T
#pragma unroll
                    for (int vb = 0; vb < VB; vb++) {
                        uint32_t vr[8][VD];
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const int row = half * 32 + (j >> 2) * 16 + 4 * lg + (j & 3);
                            if constexpr (VD == 4) {
                                const uint4 t = s.v[buf][row][vb * 16 + col];
                                vr[j][0] = t.x, vr[j][1] = t.y, vr[j][2] = t.z, vr[j][3] = t.w;
                            } else {
                                const u32x2 t = reinterpret_cast<const u32x2*>(&s.v[buf][row][0])[col];
                                vr[j][0] = t[0], vr[j][1] = t[1];
                            }
                        }
                        if (diag) {
                            // an infinity or NaN in a row that some queries do not see: 0 times it is no 0.  It
                            // counts as 0 here, and is added to the rows that see it after the last unit
                            bool x = false;
#pragma unroll
                            for (int j = 0; j < 8; j++)
#pragma unroll
                                for (int d = 0; d < VD; d++) x |= not_finite<CT>(vr[j][d]);
                            if (__ballot(x) != 0) {
#pragma unroll
                                for (int j = 0; j < 8; j++)
#pragma unroll
                                    for (int d = 0; d < VD; d++) vr[j][d] = finite_or_0<CT>(vr[j][d]);
                                mend0 = min(mend0, key0 + half * 32);
                                mend1 = key0 + half * 32 + 32;
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 2 * VD; e++) {
                            const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
                            u32x4 vf;
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                vf[j] = __builtin_amdgcn_perm(vr[2 * j + 1][e >> 1], vr[2 * j][e >> 1], sel);
#pragma unroll
                            for (int m = 0; m < MT; m++)
#pragma unroll
                                for (int x = 0; x < NS; x++)
                                    o[m][vb * 8 + e] = M::go(vf, pf[m][x], o[m][vb * 8 + e]);
                        }
                    }
                }
            }
            if (kt + 1 < k1) store((kt + 1) & 1);
        }

        // the infinities and NaN of the units at the causal border
        for (int key = mend0; key < min(mend1, own); key++) {
            const int pgi = fdiv(a.page, key), page = table[pgi];
            if (page < 0 || page >= a.n_pages) continue;
            const T* v = reinterpret_cast<const T*>(a.v) + page * a.page_stride +
                         (key - pgi * (int)a.page.d) * a.row_stride + hoff;
#pragma unroll
            for (int vb = 0; vb < VB; vb++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int d = vb * 128 + 2 * VD * (4 * lg + r);
                    if (d >= a.D) continue;
                    const Vec<T, 2 * VD> x = *reinterpret_cast<const Vec<T, 2 * VD>*>(v + d);
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        if (key >= lim[m]) continue;
#pragma unroll
                        for (int e = 0; e < 2 * VD; e++) {
                            const float y = (float)x.v[e];
                            if (!(__builtin_fabsf(y) < -kNegInf)) o[m][vb * 8 + e][r] += y;
                        }
                    }
                }
        }

        // ---- the item's rows, or this workgroup's part of them
        if (busy) {
            const bool last_word = whole && b >= 0 && (ntp > 0 || a.P == 0);
            const int64_t slot = slot_of(w, item, a.hkv, head);
#pragma unroll
            for (int m = 0; m < MT; m++) {
                l[m] += __shfl_xor(l[m], 16);
                l[m] += __shfl_xor(l[m], 32);
                if (tok[m] < 0) continue;
                if (last_word) {
                    const bool any = ref[m] != kNegInf || l[m] != 0.f;
                    const float inv = any ? 1.f / l[m] : 0.f;
                    Q* out = reinterpret_cast<Q*>(g.out) + tok[m] * g.os + (int64_t)hq[m] * a.D;
#pragma unroll
                    for (int vb = 0; vb < VB; vb++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int d = vb * 128 + 2 * VD * (4 * lg + r);
                            if (d >= a.D) continue;
                            Vec<Q, 2 * VD> v;
#pragma unroll
                            for (int e = 0; e < 2 * VD; e++) v.v[e] = (Q)(o[m][vb * 8 + e][r] * inv);
                            *reinterpret_cast<Vec<Q, 2 * VD>*>(out + d) = v;
                        }
                    if (g.lse != nullptr && lg == 0)
                        g.lse[(int64_t)tok[m] * g.H + hq[m]] = any ? (ref[m] + __builtin_log2f(l[m])) * kLn2 : kNegInf;
                } else {
                    const int row = (wave * MT + m) * 16 + col;
                    float* part = g.part + (slot * g.R + row) * DT;
#pragma unroll
                    for (int vb = 0; vb < VB; vb++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            Vec<float, 2 * VD> v;
#pragma unroll
                            for (int e = 0; e < 2 * VD; e++) v.v[e] = o[m][vb * 8 + e][r];
                            *reinterpret_cast<Vec<float, 2 * VD>*>(part + vb * 128 + 2 * VD * (4 * lg + r)) = v;
                        }
                    if (lg == 0) g.ml[slot * g.R + row] = make_float2(ref[m], l[m]);
                }
            }
        }
        u += k1 - (int)(in - (int64_t)head * nk);
    }
}

// Joins what the workgroups left of each (token, query head): one wave per row, 4 elements of the
// head per lane.
template <int QT>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs g) {
    using Q = typename Elem<QT>::type;
    const Paged& a = g.a;
    const int lane = (int)threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= (int64_t)a.T * g.H) return;
    const int t = (int)(row / g.H), h = (int)(row - (int64_t)t * g.H), head = fdiv(g.g, h), gq = h - head * g.G;
    int b = t, i = 0;
    if (a.q_start != nullptr) {
        b = count_le(a.q_start, a.B + 1, t) - 1;
        if (b < 0 || b >= a.B) return;
        i = t - a.q_start[b];
    }
    int t0, n;
    seq_tokens(a, b, t0, n);
    const int nitems = g.p.info[0];
    const int64_t U = (int64_t)g.p.info[1] * a.hkv;
    const int n_groups = (int)(U < kGroups ? U : kGroups);
    const bool joint = is_joint(g, n);
    float m = kNegInf, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int which = 0; which < 2; which++) {
        int item, r;
        if (which == 0) {
            if (a.P == 0 || joint) continue;
            const int at = g.p.place[t];
            if (at < 0) continue;
            item = (at * g.G + gq) / g.R;
            r = at * g.G + gq - item * g.R;
        } else {
            const int rt = (i * g.G + gq) / g.R;
            item = g.p.item0[b] + rt;
            r = i * g.G + gq - rt * g.R;
        }
        if (item >= nitems) continue;
        const int f0 = g.p.first[item], nk = g.p.first[item + 1] - f0;
        if (nk == 0) continue;
        const int64_t ua = (int64_t)f0 * a.hkv + (int64_t)head * nk;
        const int w0 = group_of(ua, U, n_groups), w1 = group_of(ua + nk - 1, U, n_groups);
        if (which == 1 && w0 == w1 && (joint || a.P == 0)) return;  // written by k_attn_tile
        for (int w = w0; w <= w1; w++) {
            const int64_t slot = slot_of(w, item, a.hkv, head) * g.R + r;
            const float2 x = g.ml[slot];
            if (x.x == kNegInf && x.y == 0.f) continue;
            const float nm = fmaxf(m, x.x);
            const float f = m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m - nm), f2 = __builtin_amdgcn_exp2f(x.x - nm);
            m = nm;
            l = l * f + x.y * f2;
            if (4 * lane < a.D) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(g.part + slot * g.DT + 4 * lane);
#pragma unroll
                for (int c = 0; c < 4; c++) acc[c] = acc[c] * f + v[c] * f2;
            }
        }
    }
    const bool any = m != kNegInf || l != 0.f;
    const float inv = any ? 1.f / l : 0.f;
    if (4 * lane < a.D) {
        Vec<Q, 4> v;
#pragma unroll
        for (int c = 0; c < 4; c++) v.v[c] = (Q)(acc[c] * inv);
        *reinterpret_cast<Vec<Q, 4>*>(reinterpret_cast<Q*>(g.out) + t * g.os + (int64_t)h * a.D + 4 * lane) = v;
    }
    if (g.lse != nullptr && lane == 0) g.lse[row] = any ? (m + __builtin_log2f(l)) * kLn2 : kNegInf;
}

// ---------------------------------------------------------------- host

int padded(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
// Rows of a tile: 4 waves of 16 or 32.  32 where the accumulators and the parts of the queries fit the
// 256 registers of two waves per SIMD.
int rows_of(int D, int parts) { return D <= 64 || (D <= 128 && parts == 1) ? 128 : 64; }

int64_t up16(int64_t v) { return (v + 15) / 16 * 16; }

struct Sizes {
    int64_t items, slots, ints, part, ml, total;
};
Sizes sizes(int B, int T, int G, int HKV, int R, int DT) {
    Sizes s;
    const int64_t per_rows = (int64_t)T * G / R;
    s.items = per_rows + 1 + B + per_rows;  // packed, own
    s.slots = kGroups + s.items * HKV;
    s.ints = up16(4 * (4 + (s.items + 1) + 2 * s.items + B + 2 * (int64_t)T));
    s.part = s.slots * R * DT * 4;
    s.ml = s.slots * R * 8;
    s.total = s.ints + s.part + s.ml;
    return s;
}

template <int QT, int CT, int NS>
void launch_tile(const AttnArgs& g, hipStream_t s) {
    const dim3 grid(kGroups), block(256);
    if (g.DT == 64) hipLaunchKernelGGL((k_attn_tile<QT, CT, NS, 64, 2>), grid, block, 0, s, g);
    else if (g.DT == 128) hipLaunchKernelGGL((k_attn_tile<QT, CT, NS, 128, NS == 1 ? 2 : 1>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((k_attn_tile<QT, CT, NS, 256, 1>), grid, block, 0, s, g);
}

}  // namespace

int64_t attn_paged_ws(int B, int T, int H, int HKV, int D, int) {
    const int G = H / HKV, DT = padded(D);  // for either type of q
    const int64_t x = sizes(B, T, G, HKV, rows_of(D, 1), DT).total, y = sizes(B, T, G, HKV, rows_of(D, 2), DT).total;
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
    const Sizes z = sizes(a.B, a.T, g.G, a.hkv, g.R, g.DT);
    int32_t* p = static_cast<int32_t*>(ws);
    g.p.info = p;
    g.p.first = p + 4;
    g.p.seq = g.p.first + z.items + 1;
    g.p.rt = g.p.seq + z.items;
    g.p.item0 = g.p.rt + z.items;
    g.p.packed = g.p.item0 + a.B;
    g.p.place = g.p.packed + a.T;
    g.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + z.ints);
    g.ml = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(g.part) + z.part);
    hipLaunchKernelGGL(k_attn_plan, dim3(1), dim3(256), 0, s, g);
    const bool bf = cache_type == BPD_T_BF16;
    if (q_type == BPD_T_F32 && bf) launch_tile<BPD_T_F32, BPD_T_BF16, 3>(g, s);
    else if (q_type == BPD_T_F32) launch_tile<BPD_T_F32, BPD_T_F16, 2>(g, s);
    else if (bf) launch_tile<BPD_T_BF16, BPD_T_BF16, 1>(g, s);
    else launch_tile<BPD_T_F16, BPD_T_F16, 1>(g, s);
    const dim3 grid((unsigned)(((int64_t)a.T * H + 3) / 4)), block(256);
    if (q_type == BPD_T_F32) hipLaunchKernelGGL(k_attn_join<BPD_T_F32>, grid, block, 0, s, g);
    else if (bf) hipLaunchKernelGGL(k_attn_join<BPD_T_BF16>, grid, block, 0, s, g);
    else hipLaunchKernelGGL(k_attn_join<BPD_T_F16>, grid, block, 0, s, g);
}

}  // namespace bpdq
