// norm_append.hip — bpd_norm_rope_append_paged_gpu: norm every head of the new tokens' q and k, rotate it, and write k
// and v into their pages.
//
//   y_i = x_i r w_i, r = (mean x^2 + eps)^-1/2,   a' = a cos(p f) - b sin(p f),  b' = a sin(p f) + b cos(p f)
//
// in one pass.  A head's 16-byte vectors lie in a group of 2^n neighbouring lanes of one wave, which add up its squares by
// exchanging lanes.  Every element of a head is then r (x c + y s): y is the other element of its pair, and c and s, the
// weights times cosine and sine, are the same for every head that the lane meets.  The other half of a pair
// j, j + rot_dim / 2 is read a second time instead of passed between lanes: it comes from the L1, and any rot_dim keeps
// whole vectors for what is written.  Sums, scales and rotation are binary32, the angle binary64 as in
// paged_append.hip, and the result is rounded once.
// Vector instructions and latency bound it beside memory: 6,343 tokens of 32 + 2 x 8 heads of 128, bf16, 156 MB in and
// out, 36 us = 4.3 TB/s (a copy: 5.2; a version that took coefficients for every head 108 us, one with branches
// around each load 51); 64 tokens 4.8 us, 1,740 (20 + 2 x 5 heads of 80, 40 turning) 8.4.
#include <type_traits>

#include "bpdq_paged.h"

namespace bpdq {

namespace {

struct NormArgs {
    Paged a;
    const double* turns;
    int rot;
    const int32_t* pos;
    const uint8_t *q, *k, *v;
    uint8_t* qo;
    int64_t qs, ks, vs, qos;
    const uint8_t *qw, *kw;  // NULL: not normed
    int64_t qws, kws;
    float eps;
    int H;
    int lanes, shift;  // of a head: a power of two, D / 8 at least; its logarithm
    int nq, nkv;       // units of q, and of k and of v
    int waves;         // of a token, a workgroup each
};

// How elements pair up: neighbours, halves of whole 16-byte vectors, other halves.
enum { kNeighbours, kVectors, kHalves };

// The other elements of the pairs of elements e .. e + 7 of a row whose halves are `half`: element j's is j + half or
// j - half, itself behind 2 half.
template <int PAIR, typename T>
__device__ __forceinline__ Vec<T, 8> partners(const T* row, int e, int half) {
    if constexpr (PAIR == kVectors) {
        return *reinterpret_cast<const Vec<T, 8>*>(row + (e < half ? e + half : e < 2 * half ? e - half : e));
    } else {
        Vec<T, 8> v;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int j = e + i;
            v.v[i] = row[j < half ? j + half : j < 2 * half ? j - half : j];
        }
        return v;
    }
}

template <int CTRL>
__device__ __forceinline__ float plus_dpp(float x) {
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 15, 15, true));
}
// The sum over each group of `lanes` (a power of two, 32 at most) neighbouring lanes, in all of them.
__device__ __forceinline__ float group_sum(float x, int lanes) {
    if (lanes > 1) x = plus_dpp<0xB1>(x);    // lanes 1, 0, 3, 2
    if (lanes > 2) x = plus_dpp<0x4E>(x);    // 2, 3, 0, 1
    if (lanes > 4) x = plus_dpp<0x141>(x);   // a half row mirrored
    if (lanes > 8) x = plus_dpp<0x140>(x);   // a row
    if (lanes > 16) x += __shfl_xor(x, 16);
    return x;
}

// x^-1/2 to a unit, of denormal values as well
__device__ __forceinline__ float rsqrt1(float x) {
    const bool small = x < 0x1p-96f;
    const float r = __builtin_amdgcn_rsqf(small ? x * 0x1p64f : x);
    return small ? r * 0x1p32f : r;
}

// A unit is the heads of q, of k or of v that a wave takes at a time; a token's units are dealt to its waves in turn.
// Lanes without an element or a head of their own read the last one's and write nothing.
template <int XT, int CT, int WT, int PAIR>
__global__ __launch_bounds__(256) void k_norm_append(NormArgs g) {
    using X = typename Elem<XT>::type;
    using C = typename Elem<CT>::type;
    using W = typename Elem<WT>::type;
    using VX = Vec<X, 8>;
    constexpr bool NEOX = PAIR != kNeighbours;
    __shared__ float2 cs[128];
    const Paged& a = g.a;
    const int t = (int)blockIdx.x, tid = (int)threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), last = g.waves - 1;
    const int sub = lane >> g.shift, e0 = 8 * (lane & (g.lanes - 1)), e = min(e0, a.D - 8), half = g.rot >> 1;
    struct Head {
        VX x, y;
    };
    auto load = [&](const X* rows, int h, int heads, bool pairs) {
        const X* row = rows + min(h, heads - 1) * a.D;
        Head r;
        r.x = *reinterpret_cast<const VX*>(row + e);
        r.y = r.x;
        if (NEOX && pairs) r.y = partners<PAIR>(row, e, half);
        if (PAIR == kVectors && pairs && g.rot < a.D && e >= g.rot) {
#pragma unroll
            for (int j = 0; j < 8; j++) r.y.v[j] = (X)0.f;
        }
        return r;
    };
    // the wave's first unit of q, of k and of v, and its head of them; the next is `step` heads on
    const int uq = wave, uk = (wave - g.nq) & last, uv = (wave - g.nq - g.nkv) & last;
    const int hq = (uq << (6 - g.shift)) + sub, hk = (uk << (6 - g.shift)) + sub, hv = (uv << (6 - g.shift)) + sub;
    const int step = g.waves << (6 - g.shift);
    const X* q = reinterpret_cast<const X*>(g.q) + (int64_t)t * g.qs;
    const X* k = reinterpret_cast<const X*>(g.k) + (int64_t)t * g.ks;
    const X* v = reinterpret_cast<const X*>(g.v) + (int64_t)t * g.vs;
    // these are on their way while the position and its sines are looked up
    Head xq, xk, xv;
    if (uq < g.nq) xq = load(q, hq, g.H, true);
    if (uk < g.nkv) xk = load(k, hk, a.hkv, true);
    if (uv < g.nkv) xv = load(v, hv, a.hkv, false);

    int b = t;
    int64_t index;  // in the sequence's own part
    if (a.q_start != nullptr) {
        b = __builtin_amdgcn_readfirstlane(count_le(a.q_start, a.B + 1, t) - 1);
        if (b < 0 || b >= a.B) return;  // the whole workgroup: the token is no sequence's
        int t0, n;
        seq_tokens(a, b, t0, n);
        if (t < t0 || t >= t0 + n) return;  // offsets that decrease: not really the sequence's
        index = (int64_t)a.lens[b] - n + (t - t0);
    } else {
        index = (int64_t)a.lens[b] - 1;
    }
    for (int j = tid; j < half; j += 64 * g.waves) {
        const double p = g.pos != nullptr ? (double)g.pos[t] : (double)(a.P + index);
        const double r = p * g.turns[j];
        const float f = (float)(2.0 * (r - __builtin_rint(r)));  // half revolutions in [-1, 1]
        float s, c;
        sincospif(f, &s, &c);
        cs[j] = make_float2(c, s);
    }
    C *kc = nullptr, *vc = nullptr;
    if (g.nkv > 0 && index >= 0 && index < (int64_t)a.W * (int)a.page.d) {
        const int idx = (int)index, pg = fdiv(a.page, idx);
        const int page = a.table[(int64_t)b * a.table_stride + pg];
        if (page >= 0 && page < a.n_pages) {
            const int64_t at = (int64_t)page * a.page_stride + (int64_t)(idx - pg * (int)a.page.d) * a.row_stride;
            kc = reinterpret_cast<C*>(a.k) + at;
            vc = reinterpret_cast<C*>(a.v) + at;
        }
    }
    __syncthreads();
    float c0[8], s0[8], cw[8], sw[8];  // of the lane's elements and their other halves, without and with weights
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int el = e + j;
        float2 c = make_float2(1.f, 0.f);
        if (el < g.rot) c = cs[NEOX ? (el < half ? el : el - half) : el >> 1];
        c0[j] = c.x;
        s0[j] = (NEOX ? el < half : el % 2 == 0) ? -c.y : c.y;
    }
    auto weigh = [&](const W* w) {
        const Vec<W, 8> own = *reinterpret_cast<const Vec<W, 8>*>(w + e);
        Vec<W, 8> other = own;
        if (NEOX) other = partners<PAIR>(w, e, half);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            cw[j] = c0[j] * (float)own.v[j];
            sw[j] = s0[j] * (float)other.v[NEOX ? j : j ^ 1];
        }
    };
    const float per = 1.f / (float)a.D;
    // the wave's units of q or k from u on, the first of them held in r
    auto turn = [&](Head r, const X* rows, int heads, int u, int units, int h, const uint8_t* weights, int64_t ws,
                    auto* out, int64_t head_stride) {
        using Y = std::remove_pointer_t<decltype(out)>;
        const W* w = reinterpret_cast<const W*>(weights);
        if (w != nullptr && ws == 0) weigh(w);
        if (w == nullptr) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                cw[j] = c0[j];
                sw[j] = s0[j];
            }
        }
        for (; u < units; u += g.waves, h += step) {
            Head next = r;
            if (u + g.waves < units) next = load(rows, h + step, heads, true);
            float f = 1.f, x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = (float)r.x.v[j];
            if (w != nullptr) {
                if (ws != 0) weigh(w + min(h, heads - 1) * ws);
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) sum = fmaf(x[j], x[j], sum);
                f = rsqrt1(fmaf(group_sum(e0 < a.D ? sum : 0.f, g.lanes), per, g.eps));
            }
            Vec<Y, 8> y;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                // what does not turn has no other half: an infinity or NaN there is not its own
                const float z = (NEOX ? (float)r.y.v[j] : x[j ^ 1]) * sw[j];
                y.v[j] = (Y)(fmaf(x[j], cw[j], PAIR == kVectors || e + j < g.rot ? z : 0.f) * f);
            }
            if (h < heads && e0 < a.D) *reinterpret_cast<Vec<Y, 8>*>(out + (int64_t)h * head_stride + e) = y;
            r = next;
        }
    };
    turn(xq, q, g.H, uq, g.nq, hq, g.qw, g.qws, reinterpret_cast<X*>(g.qo) + (int64_t)t * g.qos, a.D);
    if (kc == nullptr) return;
    turn(xk, k, a.hkv, uk, g.nkv, hk, g.kw, g.kws, kc, a.head_stride);
    for (int u = uv, h = hv; u < g.nkv; u += g.waves, h += step) {
        if (u != uv) xv = load(v, h, a.hkv, false);
        Vec<C, 8> y;
#pragma unroll
        for (int j = 0; j < 8; j++) y.v[j] = (C)(float)xv.x.v[j];
        if (h < a.hkv && e0 < a.D) *reinterpret_cast<Vec<C, 8>*>(vc + (int64_t)h * a.head_stride + e) = y;
    }
}

template <int XT, int CT, int WT>
void launch_weights(const NormArgs& g, bool neox, hipStream_t s) {
    const dim3 grid((unsigned)g.a.T), block(64 * g.waves);
    if (!neox) hipLaunchKernelGGL((k_norm_append<XT, CT, WT, kNeighbours>), grid, block, 0, s, g);
    else if (g.rot % 16 == 0) hipLaunchKernelGGL((k_norm_append<XT, CT, WT, kVectors>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((k_norm_append<XT, CT, WT, kHalves>), grid, block, 0, s, g);
}

template <int XT, int CT>
void launch_types(const NormArgs& g, int w_type, bool neox, hipStream_t s) {
    if (w_type == BPD_T_F32) launch_weights<XT, CT, BPD_T_F32>(g, neox, s);
    else launch_weights<XT, CT, XT>(g, neox, s);
}

}  // namespace

void launch_norm_append(const Paged& a, int cache_type, const HeadNorm& n, const double* turns, int rot, bool neox,
                        const int32_t* pos, const void* q, int64_t qs, const void* k, int64_t ks, const void* v, int64_t vs,
                        void* qo, int64_t qos, int x_type, int H, hipStream_t s) {
    NormArgs g = {a, turns, rot, pos, static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(k),
                  static_cast<const uint8_t*>(v), static_cast<uint8_t*>(qo), qs, ks, vs, qos,
                  static_cast<const uint8_t*>(n.q), static_cast<const uint8_t*>(n.k), n.q_stride, n.k_stride, n.eps, H, 1};
    while (g.lanes * 8 < a.D) {
        g.lanes *= 2;
        g.shift++;
    }
    const int group = 64 / g.lanes;
    g.nq = (H + group - 1) / group;
    g.nkv = k != nullptr ? (a.hkv + group - 1) / group : 0;
    // Four waves of a token have its latency (64 tokens of 32 + 2 x 8 heads of 128, bf16: 4.8 us, two 5.8, one 7.8), fewer
    // take its sines and weights less often (6,343: 42 us, 36, 40; 1,024: 8.5, 8.7, 10.7; with 8 + 2 heads of 64, three
    // units, 4,096 tokens: 12.2, 8.5, 7.0)
    g.waves = a.T <= 1024 ? 4 : g.nq + 2 * g.nkv > 4 ? 2 : 1;
    const bool bf = cache_type == BPD_T_BF16;
    if (x_type == BPD_T_F32) bf ? launch_types<BPD_T_F32, BPD_T_BF16>(g, n.type, neox, s)
                                : launch_types<BPD_T_F32, BPD_T_F16>(g, n.type, neox, s);
    else if (x_type == BPD_T_F16) bf ? launch_types<BPD_T_F16, BPD_T_BF16>(g, n.type, neox, s)
                                     : launch_types<BPD_T_F16, BPD_T_F16>(g, n.type, neox, s);
    else bf ? launch_types<BPD_T_BF16, BPD_T_BF16>(g, n.type, neox, s)
            : launch_types<BPD_T_BF16, BPD_T_F16>(g, n.type, neox, s);
}

}  // namespace bpdq
