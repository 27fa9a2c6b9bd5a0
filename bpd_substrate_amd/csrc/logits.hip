// logits.hip — bpd_adjust_logits_gpu: penalties for repeated tokens, biases and masks on rows of logits.
//
// A workgroup takes a slice of one row's vocabulary.  The row's history is read once per slice and counted in LDS, a
// word for each of the slice's tokens: the tokens of a history are few beside a row and repeat, and integer counts do
// not depend on the order of their atomics.  Then the slice's logits are read, changed and written in one pass, 8 at a
// time.  Of a token that stands several times in the bias list the last entry counts: the largest of its indices.
#include "bpdq_paged.h"

namespace bpdq {

namespace {

constexpr int kThreads = 512;
constexpr uint32_t kMet = 0x80000000u;  // of a count: the token stands in the history, the prompt included

// 8 elements at any address that is aligned to one
template <typename T>
struct Any8 {
    typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

template <int XT, int YT>
__global__ __launch_bounds__(kThreads) void k_adjust(AdjustArgs g) {
    using X = typename Elem<XT>::type;
    using Y = typename Elem<YT>::type;
    extern __shared__ uint32_t lds[];
    const int tid = (int)threadIdx.x, b = (int)(blockIdx.x / (unsigned)g.slices);
    const int lo = ((int)blockIdx.x - b * g.slices) * g.slice, n = min(g.slice, g.V - lo);
    uint32_t* count = lds;
    int len = 0, prompt = 0, e0 = 0, e1 = 0;
    if (g.tokens != nullptr) {
        len = g.lens != nullptr ? max(0, min(g.lens[b], g.width)) : g.width;
        prompt = g.prompt != nullptr ? max(0, min(g.prompt[b], len)) : 0;
    }
    if (g.bias_start != nullptr) {
        e0 = max(0, min(g.bias_start[b], g.n_bias));
        e1 = max(0, min(g.bias_start[b + 1], g.n_bias));
    }
    const bool history = len > 0, biased = e1 > e0;
    uint32_t* entry = lds + (g.tokens != nullptr ? g.slice : 0);  // index + 1 of the token's last bias
    for (int i = tid; i < n; i += kThreads) {
        if (history) count[i] = 0;
        if (biased) entry[i] = 0;
    }
    if (history || biased) __syncthreads();
    if (history) {
        const int32_t* t = g.tokens + (int64_t)b * g.token_stride;
        for (int i = tid; i < len; i += kThreads) {
            const uint32_t at = (uint32_t)t[i] - (uint32_t)lo;
            if (at >= (uint32_t)n) continue;
            if (i < prompt) atomicOr(&count[at], kMet);
            else atomicAdd(&count[at], 1u);
        }
    }
    if (biased)
        for (int i = e0 + tid; i < e1; i += kThreads) {
            const uint32_t at = (uint32_t)g.bias_token[i] - (uint32_t)lo;
            if (at < (uint32_t)n) atomicMax(&entry[at], (uint32_t)i + 1u);
        }
    if (history || biased) __syncthreads();
    const float rep = g.repetition != nullptr ? g.repetition[b] : 1.f;
    const float freq = g.frequency != nullptr ? g.frequency[b] : 0.f;
    const float pres = g.presence != nullptr ? g.presence[b] : 0.f;
    const uint8_t* bits = nullptr;
    if (g.mask != nullptr) {
        const int m = g.mask_row != nullptr ? g.mask_row[b] : b;
        if (m >= 0 && m < g.n_masks) bits = reinterpret_cast<const uint8_t*>(g.mask + (int64_t)m * g.mask_stride);
    }
    const X* x = reinterpret_cast<const X*>(g.x) + (int64_t)b * g.xs + lo;
    Y* y = reinterpret_cast<Y*>(g.y) + (int64_t)b * g.ys + lo;
    auto one = [&](float v, int i) {
        if (history) {
            const uint32_t c = count[i];
            if (c != 0) {
                v = v > 0.f ? v / rep : v * rep;
                if (c & ~kMet) v = v - freq * (float)(c & ~kMet) - pres;
            }
        }
        if (biased) {
            const uint32_t c = entry[i];
            if (c != 0) v += g.bias_value[c - 1];
        }
        return v;
    };
    for (int i = 8 * tid; i < n; i += 8 * kThreads) {
        const uint32_t keep = bits != nullptr ? bits[(lo + i) >> 3] : 255u;  // lo is a multiple of 8
        if (i + 8 <= n) {
            using VX = typename Any8<X>::type;
            using VY = typename Any8<Y>::type;
            VX v = {};
            if (keep != 0) v = *reinterpret_cast<const VX*>(x + i);
            VY r;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float f = one((float)v[j], i + j);
                r[j] = (keep >> j) & 1u ? (Y)f : (Y)-__builtin_inff();
            }
            *reinterpret_cast<VY*>(y + i) = r;
        } else {
            for (int j = 0; i + j < n; j++)
                y[i + j] = (keep >> j) & 1u ? (Y)one((float)x[i + j], i + j) : (Y)-__builtin_inff();
        }
    }
}

template <int XT, int YT>
void launch(const AdjustArgs& g, hipStream_t s) {
    const size_t words = (g.tokens != nullptr) + (g.bias_start != nullptr);
    hipLaunchKernelGGL((k_adjust<XT, YT>), dim3((unsigned)g.B * (unsigned)g.slices), dim3(kThreads), words * 4 * g.slice, s,
                       g);
}

}  // namespace

void launch_adjust(const AdjustArgs& a, int type, int out_type, hipStream_t s) {
    AdjustArgs g = a;
    g.slice = 8192;  // 64 KB of counts and entries: two workgroups on a CU
    // smaller while the slices do not fill the chip twice
    while (g.slice > 1024 && (int64_t)g.B * ((g.V + g.slice - 1) / g.slice) < 512) g.slice >>= 1;
    g.slices = (g.V + g.slice - 1) / g.slice;
    if (type == BPD_T_F32) launch<BPD_T_F32, BPD_T_F32>(g, s);
    else if (type == BPD_T_F16) out_type == BPD_T_F32 ? launch<BPD_T_F16, BPD_T_F32>(g, s)
                                                      : launch<BPD_T_F16, BPD_T_F16>(g, s);
    else out_type == BPD_T_F32 ? launch<BPD_T_BF16, BPD_T_F32>(g, s) : launch<BPD_T_BF16, BPD_T_BF16>(g, s);
}

}  // namespace bpdq
