// norm_append.hip — bpd_norm_rope_append_paged_gpu: norm every head of the new tokens' q and k, rotate it, and write k
// and v into their pages.
//
//   y_i = x_i (mean x^2 + eps)^-1/2 w_i,   a' = a cos(p f) - b sin(p f),  b' = a sin(p f) + b cos(p f)
//
// in one pass: a head's 16-byte vectors lie in a group of 2^n neighbouring lanes of one wave, which add up its squares by
// exchanging lanes.  The other half of each turning pair is read a second time instead of passed between lanes: it
// comes from the L1, and any rot_dim then keeps whole vectors for what is written.  Sums, scales and rotation are
// binary32, the angle binary64 as in paged_append.hip, and the result is rounded once.
#include "bpdq_paged.h"

namespace bpdq {

namespace {

constexpr int kAhead = 3;  // heads of a lane whose loads are under way together

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
    int lanes;  // of a head: a power of two, D / 8 at least
};

// 8 elements, in binary32.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    const Vec<T, 8> v = *reinterpret_cast<const Vec<T, 8>*>(p);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)v.v[i];
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    Vec<T, 8> v;
#pragma unroll
    for (int i = 0; i < 8; i++) v.v[i] = (T)x[i];
    *reinterpret_cast<Vec<T, 8>*>(p) = v;
}

// The partners of elements e .. e + 7 of a row in halves of `half`: element j's is j + half or j - half, none at 2 half
// and behind.
template <typename T>
__device__ __forceinline__ void load_partners(const T* row, int e, int half, float (&x)[8]) {
    if (half % 8 == 0) {
        if (e < 2 * half) load8(row + (e < half ? e + half : e - half), x);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int j = e + i;
        x[i] = j < 2 * half ? (float)row[j < half ? j + half : j - half] : 0.f;
    }
}

template <int XT, int CT, int WT, bool NEOX>
__global__ __launch_bounds__(256) void k_norm_append(NormArgs g) {
    using X = typename Elem<XT>::type;
    using C = typename Elem<CT>::type;
    using W = typename Elem<WT>::type;
    __shared__ float2 cs[128];
    const Paged& a = g.a;
    const int t = (int)blockIdx.x, tid = (int)threadIdx.x;
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
    for (int j = tid; j < (g.rot >> 1); j += 256) {
        const double p = g.pos != nullptr ? (double)g.pos[t] : (double)(a.P + index);
        const double r = p * g.turns[j];
        const float f = (float)(2.0 * (r - __builtin_rint(r)));  // half revolutions in [-1, 1]
        float s, c;
        sincospif(f, &s, &c);
        cs[j] = make_float2(c, s);
    }
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
    __syncthreads();
    const int sub = tid & (g.lanes - 1), e = 8 * sub, half = g.rot >> 1;
    const int step = 256 / g.lanes, heads = g.H + (kc != nullptr ? 2 * a.hkv : 0);
    const bool mine = e < a.D;
    const float per = 1.f / (float)a.D;
    // the whole wave stays in the loop: its lanes exchange sums
    for (int h0 = tid / g.lanes; h0 - tid / g.lanes < heads; h0 += step * kAhead) {
        float x[kAhead][8], y[kAhead][8], w[kAhead][8], wy[kAhead][8];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int h = h0 + i * step;
            if (!mine || h >= heads) continue;
            const bool is_q = h < g.H, is_v = h >= g.H + a.hkv;
            const X* row = is_q ? reinterpret_cast<const X*>(g.q) + (int64_t)t * g.qs + (int64_t)h * a.D
                           : is_v ? reinterpret_cast<const X*>(g.v) + (int64_t)t * g.vs + (int64_t)(h - g.H - a.hkv) * a.D
                                  : reinterpret_cast<const X*>(g.k) + (int64_t)t * g.ks + (int64_t)(h - g.H) * a.D;
            load8(row + e, x[i]);
            if (is_v) continue;
            if (NEOX) load_partners(row, e, half, y[i]);
            const W* wr = reinterpret_cast<const W*>(is_q ? g.qw : g.kw);
            if (wr == nullptr) continue;
            wr += is_q ? h * g.qws : (h - g.H) * g.kws;
            load8(wr + e, w[i]);
            if (NEOX) load_partners(wr, e, half, wy[i]);
        }
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int h = h0 + i * step;
            const bool is_q = h < g.H, is_v = h >= g.H + a.hkv, on = mine && h < heads;
            const bool normed = on && !is_v && (is_q ? g.qw : g.kw) != nullptr;
            float sum = 0.f;
            if (normed) {
#pragma unroll
                for (int j = 0; j < 8; j++) sum = fmaf(x[i][j], x[i][j], sum);
            }
            for (int d = 1; d < g.lanes; d <<= 1) sum += __shfl_xor(sum, d);
            if (!on) continue;
            if (normed) {
                const float f = 1.f / sqrtf(fmaf(sum, per, g.eps));
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    x[i][j] = x[i][j] * f * w[i][j];
                    if (NEOX) y[i][j] = y[i][j] * f * wy[i][j];
                }
            }
            if (!is_v) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if constexpr (NEOX) {
                        const int el = e + j;
                        if (el >= g.rot) break;
                        const bool low = el < half;
                        const float2 c = cs[low ? el : el - half];
                        x[i][j] = low ? x[i][j] * c.x - y[i][j] * c.y : y[i][j] * c.y + x[i][j] * c.x;
                    } else if (j % 2 == 0 && e + j < g.rot) {
                        const float2 c = cs[(e + j) >> 1];
                        const float u = x[i][j], v = x[i][j + 1];
                        x[i][j] = u * c.x - v * c.y;
                        x[i][j + 1] = u * c.y + v * c.x;
                    }
                }
            }
            if (is_q) store8(reinterpret_cast<X*>(g.qo) + (int64_t)t * g.qos + (int64_t)h * a.D + e, x[i]);
            else if (is_v) store8(vc + (int64_t)(h - g.H - a.hkv) * a.head_stride + e, x[i]);
            else store8(kc + (int64_t)(h - g.H) * a.head_stride + e, x[i]);
        }
    }
}

template <int XT, int CT, int WT>
void launch_weights(const NormArgs& g, bool neox, hipStream_t s) {
    const dim3 grid((unsigned)g.a.T), block(256);
    if (neox) hipLaunchKernelGGL((k_norm_append<XT, CT, WT, true>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((k_norm_append<XT, CT, WT, false>), grid, block, 0, s, g);
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
    while (g.lanes * 8 < a.D) g.lanes *= 2;
    const bool bf = cache_type == BPD_T_BF16;
    if (x_type == BPD_T_F32) bf ? launch_types<BPD_T_F32, BPD_T_BF16>(g, n.type, neox, s)
                                : launch_types<BPD_T_F32, BPD_T_F16>(g, n.type, neox, s);
    else if (x_type == BPD_T_F16) bf ? launch_types<BPD_T_F16, BPD_T_BF16>(g, n.type, neox, s)
                                     : launch_types<BPD_T_F16, BPD_T_F16>(g, n.type, neox, s);
    else bf ? launch_types<BPD_T_BF16, BPD_T_BF16>(g, n.type, neox, s)
            : launch_types<BPD_T_BF16, BPD_T_F16>(g, n.type, neox, s);
}

}  // namespace bpdq
