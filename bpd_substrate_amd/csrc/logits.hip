// logits.hip — bpd_adjust_logits_gpu: penalties for repeated tokens, biases and masks on rows of logits.
//
// A workgroup takes a slice of one row's vocabulary.  The row's history is read once per slice and counted in LDS, a
// word for each of the slice's tokens: the tokens of a history are few beside a row and repeat, and integer counts do
// not depend on the order of their atomics.  Then the slice's logits are read, changed and written in one pass, 8 at a
// time.  Of a token that stands several times in the bias list the last entry counts: the largest of its indices.
// Memory bounds it, then the history's latency before a slice's logits can change: 256 x 128,256 binary16 to fp32 with
// 1,000 tokens and a mask each, 202 MB, 47.5 us = 4.25 TB/s (a copy: 5.1); 64 x 128,256 fp32 with up to 16,384 tokens, 300
// biases, some masks, 68 MB, 18 us (with the logits read behind the counts and 4-byte reads of the history: 36).  In place,
// where the counts say what to read, 18 us for the 64, with penalties alone 15.6 (a new tensor 19.2).  Measured
// and left: stores past the caches, 43 us for the 256, but 5 to 6 more for the sampling that reads them; slices of 4,096 or
// 16,384 and workgroups of 256 or 1,024 (48 to 56 us).
#include "bpdq_paged.h"

namespace bpdq {

namespace {

constexpr int kThreads = 512;
constexpr int kSlice = 8192;
constexpr int kVecs = kSlice / (8 * kThreads);  // of 8 logits, a thread's
constexpr uint32_t kMet = 0x80000000u;          // of a count: the token stands in the history, the prompt included

// 8 (4) elements at any address that is aligned to one
template <typename T>
struct Any8 {
    typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};
typedef int32_t i32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Clears the words of n tokens: of whole vectors of 8, as they are read.
__device__ __forceinline__ void clear(uint32_t* lds, int n) {
    for (int i = 4 * (int)threadIdx.x; i < ((n + 7) & ~7); i += 4 * kThreads)
        *reinterpret_cast<u32x4*>(lds + i) = u32x4{0, 0, 0, 0};
}

// LITE: neither history nor biases, and so no LDS.  SELF: out is the logits, and what stays as it is is neither read nor written.
template <int XT, int YT, bool LITE, bool SELF>
__global__ __launch_bounds__(kThreads) void k_adjust(AdjustArgs g) {
    using X = typename Elem<XT>::type;
    using Y = typename Elem<YT>::type;
    using VX = typename Any8<X>::type;
    using VY = typename Any8<Y>::type;
    __shared__ __attribute__((aligned(16))) uint32_t count[LITE ? 4 : kSlice];
    const int tid = (int)threadIdx.x, b = (int)(blockIdx.x / (unsigned)g.slices);
    const int lo = ((int)blockIdx.x - b * g.slices) * g.slice, n = min(g.slice, g.V - lo);
    const uint8_t* bits = nullptr;
    if (g.mask != nullptr) {
        const int m = g.mask_row != nullptr ? g.mask_row[b] : b;
        if (m >= 0 && m < g.n_masks) bits = reinterpret_cast<const uint8_t*>(g.mask + (int64_t)m * g.mask_stride);
    }
    int len = 0, prompt = 0, e0 = 0, e1 = 0;
    if (!LITE && g.tokens != nullptr) {
        len = g.lens != nullptr ? max(0, min(g.lens[b], g.width)) : g.width;
        prompt = g.prompt != nullptr ? max(0, min(g.prompt[b], len)) : 0;
    }
    if (!LITE && g.bias_start != nullptr) {
        e0 = max(0, min(g.bias_start[b], g.n_bias));
        e1 = max(0, min(g.bias_start[b + 1], g.n_bias));
    }
    const bool history = len > 0, biased = e1 > e0;
    const X* x = reinterpret_cast<const X*>(g.x) + (int64_t)b * g.xs + lo;
    Y* y = reinterpret_cast<Y*>(g.y) + (int64_t)b * g.ys + lo;
    uint32_t keep[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; k++) {
        const int i = 8 * (tid + k * kThreads);
        keep[k] = i < n && bits != nullptr ? bits[(lo + i) >> 3] : 255u;  // lo is a multiple of 8
    }
    // the history's first tokens and the logits are on their way while the counts are cleared
    constexpr int A = 4;  // vectors of tokens under way
    const int32_t* t = g.tokens + (int64_t)b * g.token_stride;
    const int whole = len & ~3;
    i32x4 w[A];
    auto ask = [&](int i0) {
#pragma unroll
        for (int k = 0; k < A; k++) {
            const int i = i0 + 4 * k * kThreads;
            w[k] = i32x4{-1, -1, -1, -1};  // no token
            if (i < whole) w[k] = *reinterpret_cast<const i32x4*>(t + i);
        }
    };
    if (history) {
        ask(4 * tid);
        clear(count, n);
    }
    VX v[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; k++) {
        const int i = 8 * (tid + k * kThreads);
        v[k] = VX{};
        if (!SELF && i + 8 <= n && keep[k] != 0) v[k] = *reinterpret_cast<const VX*>(x + i);
    }
    if (history) {
        __syncthreads();
        auto met = [&](int token, int i) {
            const uint32_t at = (uint32_t)token - (uint32_t)lo;
            if (at >= (uint32_t)n) return;
            if (i < prompt) atomicOr(&count[at], kMet);
            else atomicAdd(&count[at], 1u);
        };
        for (int i0 = 4 * tid; i0 < whole; i0 += 4 * A * kThreads) {
            if (i0 != 4 * tid) ask(i0);
#pragma unroll
            for (int k = 0; k < A; k++)
#pragma unroll
                for (int j = 0; j < 4; j++) met(w[k][j], i0 + 4 * k * kThreads + j);
        }
        if (tid < len - whole) met(t[whole + tid], whole + tid);
        __syncthreads();
    }
    const float rep = g.repetition != nullptr ? g.repetition[b] : 1.f;
    const float freq = g.frequency != nullptr ? g.frequency[b] : 0.f;
    const float pres = g.presence != nullptr ? g.presence[b] : 0.f;
    float f[kVecs][8];
    uint32_t change[kVecs];  // bit j: logit j is another than before
#pragma unroll
    for (int k = 0; k < kVecs; k++) {
        const int i = 8 * (tid + k * kThreads);
        change[k] = ~keep[k] & 255u;
        if (i >= n) continue;
        uint32_t c[8] = {};
        if (history) {
            const u32x4 c0 = *reinterpret_cast<const u32x4*>(count + i), c1 = *reinterpret_cast<const u32x4*>(count + i + 4);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                c[j] = j < 4 ? c0[j & 3] : c1[j & 3];
                if (c[j] != 0) change[k] |= 1u << j;
            }
        }
        if (SELF && i + 8 <= n && keep[k] != 0 && (change[k] != 0 || biased)) v[k] = *reinterpret_cast<const VX*>(x + i);
        if (i + 8 > n) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i + j < n) v[k][j] = x[i + j];
        }
#pragma unroll
        for (int j = 0; j < 8; j++) f[k][j] = (float)v[k][j];
        if ((change[k] & keep[k]) != 0) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (c[j] == 0) continue;
                f[k][j] = f[k][j] > 0.f ? f[k][j] / rep : f[k][j] * rep;
                if (c[j] & ~kMet) f[k][j] = f[k][j] - freq * (float)(c[j] & ~kMet) - pres;
            }
        }
    }
    if (biased) {  // the same words, now the index + 1 of each token's last entry
        if (history) __syncthreads();
        clear(count, n);
        __syncthreads();
        for (unsigned i = (unsigned)(e0 + tid); i < (unsigned)e1; i += kThreads) {
            const uint32_t at = (uint32_t)g.bias_token[i] - (uint32_t)lo;
            if (at < (uint32_t)n) atomicMax(&count[at], i + 1u);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kVecs; k++) {
            const int i = 8 * (tid + k * kThreads);
            if (i >= n) continue;
            const u32x4 c0 = *reinterpret_cast<const u32x4*>(count + i), c1 = *reinterpret_cast<const u32x4*>(count + i + 4);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t c = j < 4 ? c0[j & 3] : c1[j & 3];
                if (c == 0) continue;
                f[k][j] += g.bias_value[c - 1];
                change[k] |= 1u << j;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < kVecs; k++) {
        const int i = 8 * (tid + k * kThreads);
        if (i >= n || (SELF && change[k] == 0)) continue;
        VY r;
#pragma unroll
        for (int j = 0; j < 8; j++) r[j] = (keep[k] >> j) & 1u ? (Y)f[k][j] : (Y)-__builtin_inff();
        if (i + 8 <= n) {
            *reinterpret_cast<VY*>(y + i) = r;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i + j < n) y[i + j] = r[j];
        }
    }
}

template <int XT, int YT, bool SELF>
void launch_rules(const AdjustArgs& g, hipStream_t s) {
    const dim3 grid((unsigned)g.B * (unsigned)g.slices), block(kThreads);
    if (g.tokens == nullptr && g.bias_start == nullptr) hipLaunchKernelGGL((k_adjust<XT, YT, true, SELF>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((k_adjust<XT, YT, false, SELF>), grid, block, 0, s, g);
}

template <int T>
void launch_types(const AdjustArgs& g, int out_type, hipStream_t s) {
    if (g.x == g.y) launch_rules<T, T, true>(g, s);
    else if (out_type == T) launch_rules<T, T, false>(g, s);
    else launch_rules<T, BPD_T_F32, false>(g, s);
}

}  // namespace

void launch_adjust(const AdjustArgs& a, int type, int out_type, hipStream_t s) {
    AdjustArgs g = a;
    g.slice = kSlice;  // 32 KB of counts: four workgroups on a CU, all that its waves allow
    // smaller while the slices do not fill the chip twice
    while (g.slice > 1024 && (int64_t)g.B * ((g.V + g.slice - 1) / g.slice) < 512) g.slice >>= 1;
    g.slices = (g.V + g.slice - 1) / g.slice;
    if (type == BPD_T_F32) launch_types<BPD_T_F32>(g, out_type, s);
    else if (type == BPD_T_F16) launch_types<BPD_T_F16>(g, out_type, s);
    else launch_types<BPD_T_BF16>(g, out_type, s);
}

}  // namespace bpdq
