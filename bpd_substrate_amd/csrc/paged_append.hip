// paged_append.hip — bpd_rope_append_paged_gpu: rotate the new tokens' q and k and
// write k and v into their pages.
//
//   a' = a cos(p f) - b sin(p f),  b' = a sin(p f) + b cos(p f)
//
// p f in revolutions is a binary64 product whose whole part is dropped there: at
// position 2^20 that leaves 2^-33 revolutions, below fp32's rounding of the sine.
// Everything is read and written once.  One workgroup per token: its rot/2 sines
// are taken once and serve every head, and its row of the cache is looked up once.  Bound by
// memory where there are many tokens: 6,343 of 32 + 2 x 8 heads of 128, 156 MB in and out, 31 us = 5.0 TB/s, what a
// copy reaches; a few tokens take the latency of lengths, sines and rows one after the other, 4.5 us, and 1,740 (20 + 2
// x 5 heads of 96, 48 turning) 9.3 us where their bytes take 4: q waits for the sines, k and v for the page as well.
#include "bpdq_paged.h"

namespace bpdq {

namespace {

struct AppendArgs {
    Paged a;
    const double* turns;
    int rot;
    const int32_t* pos;
    const uint8_t *q, *k, *v;
    uint8_t* qo;
    int64_t qs, ks, vs, qos;
    int H;
    FastDiv per;   // by the vectors a head's rotated q or k is worked off in
    FastDiv perv;  // by the vectors of a head's v
};

// One unit of a head's q or k: with NEOX unit u < rot/2/N turns elements [N u, N u + N) with
// those rot/2 behind them, later ones pass N elements on; without, unit u is elements
// [N u, N u + N), turned in pairs below rot.
template <typename X, typename Y, int N, bool NEOX>
__device__ __forceinline__ void turn(const X* x, Y* y, int u, int rot, const float2* __restrict__ cs) {
    using VX = Vec<X, N>;
    using VY = Vec<Y, N>;
    if constexpr (NEOX) {
        const int half = rot >> 1;
        if (u * N < half) {
            const VX va = *reinterpret_cast<const VX*>(x + u * N);
            const VX vb = *reinterpret_cast<const VX*>(x + u * N + half);
            VY ra, rb;
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float2 t = cs[u * N + i];
                const float a = (float)va.v[i], b = (float)vb.v[i];
                ra.v[i] = (Y)(a * t.x - b * t.y);
                rb.v[i] = (Y)(a * t.y + b * t.x);
            }
            *reinterpret_cast<VY*>(y + u * N) = ra;
            *reinterpret_cast<VY*>(y + u * N + half) = rb;
        } else {
            const int e = u * N + half;
            const VX va = *reinterpret_cast<const VX*>(x + e);
            VY r;
#pragma unroll
            for (int i = 0; i < N; i++) r.v[i] = (Y)(float)va.v[i];
            *reinterpret_cast<VY*>(y + e) = r;
        }
    } else {
        const VX va = *reinterpret_cast<const VX*>(x + u * N);
        VY r;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const int e = u * N + i;
            float a = (float)va.v[i], b = (float)va.v[i + 1];
            if (e < rot) {
                const float2 t = cs[e >> 1];
                const float ra = a * t.x - b * t.y;
                b = a * t.y + b * t.x;
                a = ra;
            }
            r.v[i] = (Y)a;
            r.v[i + 1] = (Y)b;
        }
        *reinterpret_cast<VY*>(y + u * N) = r;
    }
}

template <int XT, int CT, int N, bool NEOX>
__global__ __launch_bounds__(256) void k_rope_append(AppendArgs g) {
    using X = typename Elem<XT>::type;
    using C = typename Elem<CT>::type;
    __shared__ float2 cs[128];
    const Paged& a = g.a;
    const int t = (int)blockIdx.x;
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
    for (int j = (int)threadIdx.x; j < (g.rot >> 1); j += 256) {
        const double p = g.pos != nullptr ? (double)g.pos[t] : (double)(a.P + index);
        const double r = p * g.turns[j];
        const float f = (float)(2.0 * (r - __builtin_rint(r)));  // half revolutions in [-1, 1]
        float s, c;
        sincospif(f, &s, &c);
        cs[j] = make_float2(c, s);
    }
    __syncthreads();
    C *kc = nullptr, *vc = nullptr;
    if (g.k != nullptr && index >= 0 && index < (int64_t)a.W * (int)a.page.d) {
        const int idx = (int)index, pg = fdiv(a.page, idx);
        const int page = a.table[(int64_t)b * a.table_stride + pg];
        if (page >= 0 && page < a.n_pages) {
            const int64_t at = (int64_t)page * a.page_stride + (int64_t)(idx - pg * (int)a.page.d) * a.row_stride;
            kc = reinterpret_cast<C*>(a.k) + at;
            vc = reinterpret_cast<C*>(a.v) + at;
        }
    }
    const X* q = reinterpret_cast<const X*>(g.q) + (int64_t)t * g.qs;
    X* qo = reinterpret_cast<X*>(g.qo) + (int64_t)t * g.qos;
    const int nq = g.H * (int)g.per.d;
    for (int i = (int)threadIdx.x; i < nq; i += 256) {
        const int h = fdiv(g.per, i);
        turn<X, X, N, NEOX>(q + h * a.D, qo + h * a.D, i - h * (int)g.per.d, g.rot, cs);
    }
    if (kc == nullptr) return;
    const X* k = reinterpret_cast<const X*>(g.k) + (int64_t)t * g.ks;
    const X* v = reinterpret_cast<const X*>(g.v) + (int64_t)t * g.vs;
    const int nk = a.hkv * (int)g.per.d, nv = a.hkv * (int)g.perv.d;
    for (int i = (int)threadIdx.x; i < nk; i += 256) {
        const int h = fdiv(g.per, i);
        turn<X, C, N, NEOX>(k + h * a.D, kc + (int64_t)h * a.head_stride, i - h * (int)g.per.d, g.rot, cs);
    }
    for (int i = (int)threadIdx.x; i < nv; i += 256) {
        const int h = fdiv(g.perv, i);
        turn<X, C, 8, false>(v + h * a.D, vc + (int64_t)h * a.head_stride, i - h * (int)g.perv.d, 0, cs);
    }
}

template <int XT, int CT>
void launch_types(const AppendArgs& g, bool neox, bool wide, hipStream_t s) {
    const dim3 grid((unsigned)g.a.T), block(256);
    if (!neox) hipLaunchKernelGGL((k_rope_append<XT, CT, 8, false>), grid, block, 0, s, g);
    else if (wide) hipLaunchKernelGGL((k_rope_append<XT, CT, 8, true>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((k_rope_append<XT, CT, 1, true>), grid, block, 0, s, g);
}

}  // namespace

void launch_rope_append(const Paged& a, int cache_type, const double* turns, int rot, bool neox, const int32_t* pos,
                        const void* q, int64_t qs, const void* k, int64_t ks, const void* v, int64_t vs, void* qo,
                        int64_t qos, int x_type, int H, hipStream_t s) {
    // halves of whole 16-byte vectors turn 8 pairs at a time, others pair by pair
    const bool wide = rot % 16 == 0;
    const int n = neox && !wide ? 1 : 8;
    AppendArgs g = {a, turns, rot, pos, static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(k),
                    static_cast<const uint8_t*>(v), static_cast<uint8_t*>(qo), qs, ks, vs, qos, H,
                    fast_div((neox ? a.D - rot / 2 : a.D) / n), fast_div(a.D / 8)};
    const bool bf = cache_type == BPD_T_BF16;
    if (x_type == BPD_T_F32) bf ? launch_types<BPD_T_F32, BPD_T_BF16>(g, neox, wide, s)
                                : launch_types<BPD_T_F32, BPD_T_F16>(g, neox, wide, s);
    else if (x_type == BPD_T_F16) bf ? launch_types<BPD_T_F16, BPD_T_BF16>(g, neox, wide, s)
                                     : launch_types<BPD_T_F16, BPD_T_F16>(g, neox, wide, s);
    else bf ? launch_types<BPD_T_BF16, BPD_T_BF16>(g, neox, wide, s)
            : launch_types<BPD_T_BF16, BPD_T_F16>(g, neox, wide, s);
}

}  // namespace bpdq
