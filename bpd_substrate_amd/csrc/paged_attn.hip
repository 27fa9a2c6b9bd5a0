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
#include "bpdq_attn.h"

namespace bpdq {

namespace {

// ---------------------------------------------------------------- host

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
    if (g.planned) hipLaunchKernelGGL(k_attn_plan<false>, dim3(1), dim3(1024), 0, s, g);
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

void launch_attn_paged(const Paged& a, int cache_type, const void* q, int64_t qs, void* out, int64_t os, float* lse,
                       int q_type, int H, float scale, void* ws, hipStream_t s) {
    const AttnArgs g = attn_args(a, cache_type, q, qs, out, os, lse, q_type, H, scale, a.n_pages == 0 ? 0 : a.P, ws);
    const bool bf = cache_type == BPD_T_BF16;
    if (q_type == BPD_T_F32 && bf) launch_types<BPD_T_F32, BPD_T_BF16, 3>(g, s);
    else if (q_type == BPD_T_F32) launch_types<BPD_T_F32, BPD_T_F16, 2>(g, s);
    else if (bf) launch_types<BPD_T_BF16, BPD_T_BF16, 1>(g, s);
    else launch_types<BPD_T_F16, BPD_T_F16, 1>(g, s);
}

}  // namespace bpdq
