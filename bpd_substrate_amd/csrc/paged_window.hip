// paged_window.hip — bpd_attn_window_paged_gpu: attention over a sliding window and the first rows of a paged cache.
//
// A token at position p sees the rows at positions j <= p with j > p - window or j < sinks.  The kernels are those of
// paged_attn.hip with the units that no token of an item sees left out (span_of): at most four runs, the first
// rows and the window's in the prefix and in the sequence's own part.  Every sequence reads the prefix's rows that it sees
// for itself, as a window passes the prefix soon: its tokens are not packed.
#include "bpdq_attn.h"

namespace bpdq {

namespace {

template <int QT, int CT, int NS, int DT, int MT, int NW, bool UNI>
void launch_dim(const AttnArgs& g, hipStream_t s) {
    if (g.planned)
        hipLaunchKernelGGL((k_attn_tile<QT, CT, NS, DT, MT, NW, UNI, true>), dim3((unsigned)g.groups), dim3(64 * NW), 0, s,
                           g);
    else if (g.a.W > 0 || g.a.P > 0)
        hipLaunchKernelGGL((k_attn_wave<QT, CT, NS, DT, UNI, true>), dim3((unsigned)(g.waves / 4)), dim3(256), 0, s, g);
}

template <int QT, int CT, int NS, bool UNI>
void launch_uni(const AttnArgs& g, hipStream_t s) {
    if (g.DT == 64) launch_dim<QT, CT, NS, 64, 2, 8, UNI>(g, s);
    else if (g.DT == 128) launch_dim<QT, CT, NS, 128, NS == 1 ? 2 : 1, 8, UNI>(g, s);
    else launch_dim<QT, CT, NS, 256, 1, 4, UNI>(g, s);
}

template <int QT, int CT, int NS>
void launch_types(const AttnArgs& g, hipStream_t s) {
    if (g.planned) hipLaunchKernelGGL(k_attn_plan<true>, dim3(1), dim3(1024), 0, s, g);
    if (g.a.page.d % 16 == 0 && g.a.row_stride < 1 << 26) launch_uni<QT, CT, NS, true>(g, s);
    else launch_uni<QT, CT, NS, false>(g, s);
    // one head per wave while that fills the chip twice at most, more where most rows are done
    if ((int64_t)g.a.T * g.H <= 32768)
        hipLaunchKernelGGL((k_attn_join<QT, 1, true>), dim3((unsigned)g.a.T, (unsigned)((g.H + 3) / 4)), dim3(256), 0, s, g);
    else
        hipLaunchKernelGGL((k_attn_join<QT, 8, true>), dim3((unsigned)g.a.T, (unsigned)((g.H + 31) / 32)), dim3(256), 0, s,
                           g);
}

}  // namespace

void launch_attn_window(const Paged& a, int cache_type, const void* q, int64_t qs, void* out, int64_t os, float* lse,
                        int q_type, int H, float scale, int window, int sinks, void* ws, hipStream_t s) {
    AttnArgs g = attn_args(a, cache_type, q, qs, out, os, lse, q_type, H, scale, 0, ws);
    g.window = window;
    g.sinks = sinks;
    const bool bf = cache_type == BPD_T_BF16;
    if (q_type == BPD_T_F32 && bf) launch_types<BPD_T_F32, BPD_T_BF16, 3>(g, s);
    else if (q_type == BPD_T_F32) launch_types<BPD_T_F32, BPD_T_F16, 2>(g, s);
    else if (bf) launch_types<BPD_T_BF16, BPD_T_BF16, 1>(g, s);
    else launch_types<BPD_T_F16, BPD_T_F16, 1>(g, s);
}

}  // namespace bpdq
