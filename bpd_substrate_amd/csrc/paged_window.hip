// paged_window.hip — bpd_attn_window_paged_gpu: attention over a sliding window and the first rows of a paged cache.
//
// A token at position p sees the rows at positions j <= p with j > p - window or j < sinks.  The kernels are those of
// paged_attn.hip with the units that no token of an item sees left out (span_of): at most four runs, the first
// rows and the window's in the prefix and in the sequence's own part.  Every sequence reads the prefix's rows that it sees
// for itself, as a window passes the prefix soon: its tokens are not packed.  Windows bound what a token sees, so the host
// knows the work of most batches: up to a few thousand rows they take one launch of k_attn_head, a workgroup for each
// (sequence, kv head) or each 16 rows of a few tokens.
//
// Measured (H 32, 8 kv heads, D 128, bf16 unless said; calls back to back):
//   64 sequences of one token, windows of 1,024, 268 MB    47 us   5.7 TB/s (reads alone: 7.1): 8 waves of a CU and what
//                                                                  they hold of the next two units
//   3,049 tokens in 8 chunks, windows of 4,096            317 us   553 TFLOP/s of the 175 GFLOP asked for, 624 of the 198
//                                                                  that tiles of 64 tokens take (an 8192^3 product: 1,200); plan 5,
//                                                                  join 20 of it.  A unit of 64 keys takes a wave 6,800 clocks, of
//                                                                  which it issues 2,600 (283 vector, 228 scalar instructions)
//   17 sequences, fp32 q, 5 heads of 96, pages of 21, 2,500    33 us   2.5 TB/s: waves with one unit in flight wait for it
//                                                                  half of their time
//   the chunks with fp32 queries, f16 / bf16 pages       487 / 595 us   two and three products for each
//   1 sequence, D 64, f16, 512                              9 us   latency of one workgroup
// Measured and left: 64 rows a wave with 4 waves and all 512 registers (433 us for the chunks, 822 with accumulation
// registers); one lookup for units in one page (313, but 47 -> 51 for 64 sequences behind 8,192 shared keys, which share
// that code).
#include "bpdq_attn.h"

namespace bpdq {

namespace {

constexpr int64_t kMostItems = 1 << 22;  // workgroups of 512 threads in a launch
// Rows that one workgroup may have to take for 16 rows of queries, where there are no more workgroups than these.
constexpr int64_t kMostRows = 8192, kManyItems = 512;

bool whole_pages(const Paged& a) { return a.page.d % 16 == 0 && a.row_stride < 1 << 26; }

// Waves of a workgroup so that `items` workgroups are on the chip at once.  With few rows a wave's time is latency that more
// waves do not shorten, and a second round of workgroups doubles it.  Measured (us, 4 / 2 / 1 waves; 4 query heads to each
// kv head, 128 wide, bf16; lengths from a quarter of the rows to all): 512 items, 132 rows 10.7, 11.0, 12.5; 600 15.4, 11.7,
// 13.3; 1,024 17.8, 14.3, 15.0; 1,408 24.1, 21.0, 17.8; 2,048 items, 68 / 260 / 516 rows 29.2, 20.2, 14.7 / 50.6, 41.6,
// 37.4 / 66.6, 61.0, 60.8, but 2,052 rows 227, 235, 234, where memory bounds it; heads of 256, 1,024 items, 132 rows 37.2,
// 28.3, 22.2; fp32 queries, 480 items, pages of 21, 132 / 520 rows 8.7, 10.8, 14.0 / 19.5, 28.5, 42.7.
int chip_waves(int DT) { return DT == 256 ? 1024 : 2048; }  // that the registers hold
bool few_rows(int DT, bool single, int64_t rows) { return rows <= (single || DT == 256 ? 320 : 640); }
int waves_at_once(int most, int64_t items, int64_t waves) {
    while (most > 1 && items * most > waves) most >>= 1;
    return most;
}

// Waves of a workgroup for each (sequence, head), or 0: the units dealt to all waves of the chip, and a second launch.
// `rows` is what a token sees at most, `items` sequences times kv heads.  One launch spares the dealing and the join, 6 to
// 9 us, and costs where few items with many rows leave CUs idle.  Measured (us, one launch with 8 and with 4 waves,
// two launches; 8 kv heads of 128, bf16):
//   8 items, 132 / 2,052 / 4,100 rows      7.7, 8.3, 13.1 / 19.2, 25.5, 20.4 / 31.9, 45.4, 29.7
//   128, 1,028 / 4,100                     18.1, 19.5, 27.1 / 62.7, 66.6, 68.6
//   512, 1,028 / 4,100                     52.0, 46.6, 64.6 / 172.7, 170.5, 182.8
// The lengths are on the device, and one sequence may have most of the rows: beyond 4,096, where dealing and join are little
// beside them, they are dealt unless more than 4,096 items keep the chip busy beside it (one launch, two; all lengths the
// same, a quarter of the rows to all, one sequence of all and the others of 512):
//   512, 4,100 / 16,388    179, 182 / 679, 641    135, 129 / 431, 392    65, 38 / 196, 50
//   128, 4,100 / 16,388    52, 54 / 199, 171      45, 39 / 161, 109      44, 32 / 148, 47
//   128 of 256, 4,100      110, 116               98, 95                 83, 62
//   2,048, 4,100 / 16,388  -                      421, 421 / 1,698, 1,549    99, 107 / 229, 117
//   8,192, 4,100 / 16,388  -                      1,706, 1,744 / 6,942, 6,854    367, 395 / 382, 402
// Waves with one unit in flight (`single`: fp32 queries, pages that are no multiple of 16 rows) take more than twice as
// long for a row (5 heads of 96, page 21, 5 items, 516 / 1,028 rows: 14.7, 18.4, 14.2 / 21.7, 30.0, 15.8; 320 items:
// 30.8, 23.8, 27.8 / 49.0, 41.6, 40.5).  Heads of 256 fill the registers with 4 waves (2 heads, 2 items, 516 / 1,028 rows:
// -, 17.0, 17.8 / -, 24.0, 21.0; 128 items: -, 21.3, 43.6 / -, 37.0, 56.0).
int head_waves(int DT, bool single, int64_t items, int64_t rows) {
    if (rows > 4096 && items <= 4096) return 0;
    if (DT == 256 ? items < 128 && rows > 640 : single ? rows > 640 : items < 128 && rows > 2304) return 0;
    const int most = DT == 256 ? 4 : 8;
    if (few_rows(DT, single, rows)) return waves_at_once(most, items, chip_waves(DT));
    return items <= 256 ? most : 4;
}

// Rows that a token sees at most.
int64_t rows_seen(const Paged& a, int window, int sinks) {
    const int64_t all = (int64_t)a.W * a.page.d + a.P, seen = (int64_t)window + sinks;
    return seen < all ? seen : all;
}
// Tiles of R rows that the tokens make at most, and where every sequence has as many of them.
int64_t tiles_of(const Paged& a, int G, int R) { return (int64_t)a.T * G / R + a.B; }
int64_t even_tiles(const Paged& a, int G, int R) {
    const int64_t n = a.B > 0 ? ((int64_t)a.T + a.B - 1) / a.B : 0, even = a.B * ((n * G + R - 1) / R);
    return even < tiles_of(a, G, R) ? even : tiles_of(a, G, R);
}

// The same for several tokens of a sequence, whose rows go 16 to a workgroup or by k_attn_plan, k_attn_tile and k_attn_join.
// Those have 20 us of launches (few workgroups) to 40 (uneven shares), and read the keys once for R rows; the cost of a
// unit, all CUs working, is in ns.  Measured (us, 16 rows to a workgroup / tiles; 8 kv heads of 128, 4 query heads each, bf16):
//   64 sequences, 516 rows, 2 / 4 / 8 / 16 / 32 tokens    35, 81 / 36, 83 / 54, 90 / 82, 106 / 142, 109
//   64, 2,052 rows, 4 / 8 / 16                            92, 172 / 152, 180 / 238, 196
//   8, 516 and 2,052 rows, 64                             35, 57 and 86, 74
//   1, 2,052 rows, 128                                    20, 42
// heads of 64 (5 to a kv head), 64 sequences, 2,052 rows, 8 / 32: 103, 135 / 240, 149; of 256 (2 kv heads, 8 each), 4 / 8:
// 76, 98 / 147, 104.
// Fewer of them than CUs take as long as one per CU would, and nearly the same for each row however few they are (one
// sequence of 1 / 4 tokens: 2,052 rows 24.5, 24.5 / 25.3, 27.9; 4,100 38.9, 26.0 / 39.6, 29.5; 16,388 165, 40 / 166, 43;
// 131,076 1,724, 150 / 1,730, 153; 2,052 and 4,100 rows with fp32 queries 23.5, 22.2 and 36.5, 24.1, in pages of 21
// 27.2, 24.0 and 45.0, 26.7; heads of 256, 1,028 and 4,100 27.4, 25.4 and 75.0, 34.6).
// The lengths are on the device: a workgroup may get all the rows and the others few, while tiles deal what is there.
// Beyond kMostRows that risk is taken only where more than kManyItems workgroups keep the chip busy beside it, which tiles
// of few rows do worse (sequences of one token, 8 workgroups to each; 8,196 and 16,388 rows; lengths from a quarter of the
// rows to all / one of all and the others of 512:
//   64 sequences     301, 355 and 548, 613 / 65 of two tokens, 19,264 rows 473, 94
//   128              514, 682 and 999, 1,223 / 212, 125 and 411, 134
//   256              981, 1,324 and 1,869, 2,489 / 234, 215 and 425, 222
//   1,024            3,587, 5,241 and 7,064, 9,914 / 462, 743 and 500, 747).
// Of the workgroups up to one per sequence has no tokens and ends at once: the chip is taken for a quarter larger (us, 4 / 2 / 1
// waves; 64 sequences, 516 rows, up to 4 and 8 tokens 31.1, 28.0, 40.7 and 40.2, 37.2, 43.9; 107, heads of 64, 122 rows, 6
// tokens 29.3, 19.5, 15.3; 128, 132 rows, 4 tokens 30.2, 24.9, 21.7).
int rows_waves(const Paged& a, int G, int R, bool single, int64_t rows) {
    const int DT = padded(a.D);
    const double head = DT == 64 ? 0.95 : DT == 128 ? 1.6 : 4.2, tile = DT == 64 ? 6 : DT == 128 ? 9 : 14;
    const int64_t items = even_tiles(a, G, 16) * a.hkv;
    const double one = head * (double)(items > kGroups ? items : kGroups) * (double)((rows + 63) / 32);
    const double plan = 40e3 + tile * (double)(even_tiles(a, G, R) * a.hkv) * (double)((rows + 127) / 64);
    if ((rows > kMostRows && items <= kManyItems) || one >= plan || tiles_of(a, G, 16) * a.hkv > kMostItems) return 0;
    const int most = DT == 256 ? 4 : 8;
    if (few_rows(DT, single, rows)) return waves_at_once(most, tiles_of(a, G, 16) * a.hkv, chip_waves(DT) * 5 / 4);
    return items <= 256 ? most : 4;
}

// head_waves or rows_waves of a call.
int waves_of(const Paged& a, int q_type, int G, int window, int sinks) {
    const int DT = padded(a.D);
    const int64_t rows = rows_seen(a, window, sinks);
    const bool single = !whole_pages(a) || (q_type == BPD_T_F32 && DT > 64);
    if (planned_way(a.q_start, G)) return rows_waves(a, G, rows_of(a.D, q_type == BPD_T_F32 ? 2 : 1), single, rows);
    const int64_t items = (int64_t)a.B * a.hkv;
    if (items > kMostItems) return 0;
    return head_waves(DT, single, items, rows);
}

template <int QT, int CT, int NS, int DT, bool UNI, int NW>
void launch_head(const AttnArgs& g, hipStream_t s) {
    const dim3 block(64 * NW);
    if (g.planned)
        hipLaunchKernelGGL((k_attn_head<QT, CT, NS, DT, UNI, NW, true>),
                           dim3((unsigned)(tiles_of(g.a, g.G, 16) * g.a.hkv)), block, 0, s, g);
    else
        hipLaunchKernelGGL((k_attn_head<QT, CT, NS, DT, UNI, NW, false>), dim3((unsigned)(g.a.B * g.a.hkv)), block, 0, s, g);
}

template <int QT, int CT, int NS, int DT, int MT, int NW, bool UNI>
void launch_dim(const AttnArgs& g, hipStream_t s) {
    if (DT < 256 && g.waves == 8)
        launch_head<QT, CT, NS, DT, UNI, DT < 256 ? 8 : 4>(g, s);
    else if (g.waves == 4)
        launch_head<QT, CT, NS, DT, UNI, 4>(g, s);
    else if (g.waves == 2)
        launch_head<QT, CT, NS, DT, UNI, 2>(g, s);
    else if (g.waves == 1)
        launch_head<QT, CT, NS, DT, UNI, 1>(g, s);
    else if (g.planned)
        hipLaunchKernelGGL((k_attn_tile<QT, CT, NS, DT, MT, NW, UNI, true>), dim3((unsigned)g.groups), dim3(64 * NW), 0, s,
                           g);
    else
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
    const bool one = g.waves <= 8;  // one launch: the workgroups join their waves
    if (g.planned && !one) hipLaunchKernelGGL(k_attn_plan<true>, dim3(1), dim3(1024), 0, s, g);
    if (whole_pages(g.a)) launch_uni<QT, CT, NS, true>(g, s);
    else launch_uni<QT, CT, NS, false>(g, s);
    if (one) return;
    // one head per wave while that fills the chip twice at most, more where most rows are done
    if ((int64_t)g.a.T * g.H <= 32768)
        hipLaunchKernelGGL((k_attn_join<QT, 1, true>), dim3((unsigned)g.a.T, (unsigned)((g.H + 3) / 4)), dim3(256), 0, s, g);
    else
        hipLaunchKernelGGL((k_attn_join<QT, 8, true>), dim3((unsigned)g.a.T, (unsigned)((g.H + 31) / 32)), dim3(256), 0, s,
                           g);
}

}  // namespace

int64_t attn_window_ws(const Paged& a, int q_type, int H, int window, int sinks) {
    const int G = H / a.hkv, DT = padded(a.D);
    if (waves_of(a, q_type, G, window, sinks) > 0) return 0;
    return sizes(planned_way(a.q_start, G), a.B, a.T, G, a.hkv, rows_of(a.D, q_type == BPD_T_F32 ? 2 : 1), DT, 0).total;
}

void launch_attn_window(const Paged& a, int cache_type, const void* q, int64_t qs, void* out, int64_t os, float* lse,
                        int q_type, int H, float scale, int window, int sinks, void* ws, hipStream_t s) {
    AttnArgs g = attn_args(a, cache_type, q, qs, out, os, lse, q_type, H, scale, 0, ws);
    g.window = window;
    g.sinks = sinks;
    const int n = waves_of(a, q_type, g.G, window, sinks);  // as the workspace's size goes by
    if (n > 0) g.waves = n;
    // as k_attn_wave's
    g.past_mall = (int64_t)a.B * a.hkv * rows_seen(g.a, window, sinks) * a.D * 4 > (int64_t)256 << 20;
    const bool bf = cache_type == BPD_T_BF16;
    if (q_type == BPD_T_F32 && bf) launch_types<BPD_T_F32, BPD_T_BF16, 3>(g, s);
    else if (q_type == BPD_T_F32) launch_types<BPD_T_F32, BPD_T_F16, 2>(g, s);
    else if (bf) launch_types<BPD_T_BF16, BPD_T_BF16, 1>(g, s);
    else launch_types<BPD_T_F16, BPD_T_F16, 1>(g, s);
}

}  // namespace bpdq
