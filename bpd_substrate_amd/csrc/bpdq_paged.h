// bpdq_paged.h — what the kernels of include/bpdq_serve.h share: the batch as a
// kernel argument, the element types, the sequence of a token.  Callers have
// validated the host side of every argument; device contents (lengths, indices,
// pages) are checked where a kernel uses them.
#pragma once
#include <hip/hip_bfloat16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/bpdq_serve.h"
#include "bpdq_paged_plan.h"

namespace bpdq {

struct Paged {
    uint8_t *k, *v;
    int n_pages, hkv, D;
    FastDiv page;  // by the page size
    int page_stride, row_stride, head_stride;  // below 2^30: elements of a product with a page or row fit 61 bits
    const int32_t* table;
    int64_t table_stride;
    int W;
    const int32_t* lens;
    const int32_t* q_start;
    int B, T;
    const int32_t* prefix;
    int P;
};

#ifdef __HIPCC__
// How many of the values p[0..n), not decreasing, are <= t: a search over 64 places at a
// time, one load for up to 64 values.  The whole wave calls it with the same arguments.
// Values that do decrease give some number in 0..n.
__device__ __forceinline__ int count_le(const int32_t* __restrict__ p, int n, int t) {
    const int lane = (int)(threadIdx.x & 63);
    int lo = 0, hi = n;
    while (lo < hi) {
        const int step = (hi - lo + 63) >> 6;
        const int i = lo + lane * step;
        const int c = __popcll(__ballot(i < hi && p[i < hi ? i : lo] <= t));
        if (c == 0) return lo;
        if (step == 1) return lo + c;
        hi = min(hi, lo + c * step);
        lo = lo + (c - 1) * step + 1;
    }
    return lo;
}

// The first and one past the last new token of sequence b, within [0, T].
__device__ __forceinline__ void seq_tokens(const Paged& a, int b, int& t0, int& n) {
    if (a.q_start == nullptr) {
        t0 = b;
        n = 1;
        return;
    }
    clamp_tokens(a.q_start[b], a.q_start[b + 1], a.T, t0, n);
}

template <int TYPE>
struct Elem;
template <>
struct Elem<BPD_T_F32> {
    using type = float;
};
template <>
struct Elem<BPD_T_F16> {
    using type = _Float16;
};
template <>
struct Elem<BPD_T_BF16> {
    using type = __bf16;
};

template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Vec {
    T v[N];
};
#endif

// Host launchers.
void launch_rope_append(const Paged& a, int cache_type, const double* turns, int rot, bool neox, const int32_t* pos,
                        const void* q, int64_t qs, const void* k, int64_t ks, const void* v, int64_t vs, void* qo,
                        int64_t qos, int x_type, int H, hipStream_t s);
struct HeadNorm {
    const void *q, *k;
    int type;
    int64_t q_stride, k_stride;
    float eps;
};
void launch_norm_append(const Paged& a, int cache_type, const HeadNorm& n, const double* turns, int rot, bool neox,
                        const int32_t* pos, const void* q, int64_t qs, const void* k, int64_t ks, const void* v, int64_t vs,
                        void* qo, int64_t qos, int x_type, int H, hipStream_t s);
int64_t attn_paged_ws(const int32_t* q_start, int B, int T, int H, int HKV, int D, int P);
void launch_attn_paged(const Paged& a, int cache_type, const void* q, int64_t qs, void* out, int64_t os, float* lse,
                       int q_type, int H, float scale, void* ws, hipStream_t s);
void launch_attn_window(const Paged& a, int cache_type, const void* q, int64_t qs, void* out, int64_t os, float* lse,
                        int q_type, int H, float scale, int window, int sinks, void* ws, hipStream_t s);
int64_t attn_window_ws(const Paged& a, int q_type, int H, int window, int sinks);
int64_t sample_ws(int n_rows, int vocab);
struct SampleArgs {
    const void* logits;
    int64_t stride;
    int B, V;
    const float* temperature;
    const int32_t* top_k;
    const float *top_p, *min_p, *u;
    int32_t* token;
    float* logprob;
    int32_t* kept;
};
void launch_sample(const SampleArgs& a, int type, void* ws, hipStream_t s);
struct AdjustArgs {
    const void* x;
    int64_t xs;
    void* y;
    int64_t ys;
    int B, V;
    const int32_t* tokens;
    int64_t token_stride;
    int width;
    const int32_t *lens, *prompt;
    const float *repetition, *frequency, *presence;
    const int32_t *bias_start, *bias_token;
    const float* bias_value;
    int n_bias;
    const int32_t* mask;
    int64_t mask_stride;
    int n_masks;
    const int32_t* mask_row;
    int slice, slices;  // the launcher's
};
void launch_adjust(const AdjustArgs& a, int type, int out_type, hipStream_t s);
struct PoolArgs {
    int32_t* table;
    int64_t table_stride;
    int W;
    int32_t *lens, *gone, *free_pages, *n_free;
    int n_rows, n_pages;
    FastDiv page;
    const int32_t *rows, *add, *keep;
    int B, T;
    int32_t* table_out;
    int64_t table_out_stride;
    int32_t *lens_out, *q_start, *slots, *pos, *refused;
    int prefix_len, window, sinks;
    int parts;  // the launcher's
};
void launch_pages_extend(const PoolArgs& a, hipStream_t s);
void launch_pages_release(const PoolArgs& a, hipStream_t s);

}  // namespace bpdq
