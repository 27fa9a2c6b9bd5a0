// paged_attn.hip — bpd_attn_paged_gpu: attention over a paged cache.
//
//   s_i = scale q.k_i,  out = sum_i exp(s_i - m) v_i / sum_i exp(s_i - m),  m = max s_i,
//   lse = m + log sum_i exp(s_i - m)
//
// in one pass over the keys with the running maximum and sum of each row.
#include "bpdq_paged.h"

namespace bpdq {

namespace {

struct AttnArgs {
    Paged a;
    const uint8_t* q;
    uint8_t* out;
    int64_t qs, os;
    float* lse;
    int H, G;  // query heads, and of each kv head
    float scale;
};

// The plain form: one wave per (token, head), a lane per key for the scores and a lane per
// four elements for the sums.
template <int QT, int CT>
__global__ __launch_bounds__(64) void k_attn_plain(AttnArgs g) {
    using Q = typename Elem<QT>::type;
    using C = typename Elem<CT>::type;
    __shared__ float qf[256];
    const Paged& a = g.a;
    const int t = (int)blockIdx.x, h = (int)blockIdx.y, lane = (int)threadIdx.x;
    int b = t, seen;
    if (a.q_start != nullptr) {
        b = count_le(a.q_start, a.B + 1, t) - 1;
        if (b < 0 || b >= a.B) return;
        seen = a.lens[b] - (a.q_start[b + 1] - a.q_start[b]) + (t - a.q_start[b]) + 1;
    } else {
        seen = a.lens[b];
    }
    seen = max(0, min(seen, a.W * (int)a.page.d));
    const Q* q = reinterpret_cast<const Q*>(g.q) + t * g.qs + h * a.D;
    for (int e = lane; e < a.D; e += 64) qf[e] = (float)q[e] * g.scale;
    __syncthreads();
    float m = -__builtin_inff(), l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    const int64_t head = (int64_t)(h / g.G) * a.head_stride;
    for (int part = 0; part < 2; part++) {
        const int32_t* table = part == 0 ? a.prefix : a.table + (int64_t)b * a.table_stride;
        const int n = part == 0 ? a.P : seen;
        for (int i0 = 0; i0 < n; i0 += 64) {
            const int i = i0 + lane;
            int64_t at = -1;
            if (i < n) {
                const int pg = fdiv(a.page, i), page = table[pg];
                if (page >= 0 && page < a.n_pages)
                    at = page * a.page_stride + (i - pg * (int)a.page.d) * a.row_stride + head;
            }
            float s = -__builtin_inff();
            if (at >= 0) {
                const C* k = reinterpret_cast<const C*>(a.k) + at;
                s = 0.f;
                for (int e = 0; e < a.D; e++) s = fmaf(qf[e], (float)k[e], s);
            }
            float top = s;
            for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
            const float mn = fmaxf(m, top);
            if (mn == -__builtin_inff()) continue;
            const float keep = expf(m - mn);
            float p = at >= 0 ? expf(s - mn) : 0.f;
            float sum = p;
            for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
            l = l * keep + sum;
            m = mn;
            for (int c = 0; c < 4; c++) acc[c] *= keep;
            for (int j = 0; j < 64; j++) {
                const int64_t vat = __shfl(at, j);
                const float pj = __shfl(p, j);
                if (vat < 0 || 4 * lane >= a.D) continue;
                const C* v = reinterpret_cast<const C*>(a.v) + vat + 4 * lane;
                for (int c = 0; c < 4; c++) acc[c] = fmaf(pj, (float)v[c], acc[c]);
            }
        }
    }
    Q* out = reinterpret_cast<Q*>(g.out) + t * g.os + h * a.D;
    if (4 * lane < a.D)
        for (int c = 0; c < 4; c++) out[4 * lane + c] = (Q)(l > 0.f || l != l ? acc[c] / l : 0.f);
    if (g.lse != nullptr && lane == 0) g.lse[(int64_t)t * g.H + h] = l > 0.f || l != l ? m + logf(l) : -__builtin_inff();
}

}  // namespace

int64_t attn_paged_ws(int, int, int, int, int, int) { return 16; }

void launch_attn_paged(const Paged& a, int cache_type, const void* q, int64_t qs, void* out, int64_t os, float* lse,
                       int q_type, int H, float scale, void*, hipStream_t s) {
    AttnArgs g = {a, static_cast<const uint8_t*>(q), static_cast<uint8_t*>(out), qs, os, lse, H, H / a.hkv, scale};
    const dim3 grid((unsigned)a.T, (unsigned)H), block(64);
    const bool bf = cache_type == BPD_T_BF16;
    if (q_type == BPD_T_F32 && bf) hipLaunchKernelGGL((k_attn_plain<BPD_T_F32, BPD_T_BF16>), grid, block, 0, s, g);
    else if (q_type == BPD_T_F32) hipLaunchKernelGGL((k_attn_plain<BPD_T_F32, BPD_T_F16>), grid, block, 0, s, g);
    else if (bf) hipLaunchKernelGGL((k_attn_plain<BPD_T_BF16, BPD_T_BF16>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((k_attn_plain<BPD_T_F16, BPD_T_F16>), grid, block, 0, s, g);
}

}  // namespace bpdq
