// sample.hip — bpd_sample_gpu: one token per row of logits.
//
// A logit's place is its order key: the binary32 bits, sign-folded so that unsigned order is
// the logits' order, 0 for what is never chosen.  All weights are
// W = rint(2^shift exp((l - max) / t)), taken in binary64: their sums are exact in 64 bits,
// so no sum depends on its order.  Every filter keeps a head of the list sorted by
// (logit, index), so it is one cut, found in four steps:
//   max    largest and smallest logit, how many there are
//   hist   in each of kBuckets ranges of logits, counted from the largest, with top-k how many there are,
//          else how much they weigh
//   pick   (k_cut, k_pick) the buckets in which the cut can fall (top-k: all up to it) go to a list; what stands before
//          them stays
//   draw   the list sorted, the cut, the slice in which the draw falls, the token
// k_sample_row takes them in turn with one workgroup for a row; k_max, k_hist and k_pick with one per
// slice of a row, and k_cut and k_draw with one per row.  A row whose list is too long (thousands of equal
// logits at the cut) is searched digit by digit instead.
//
// Measured (calls back to back): 1 row of 32,000, top-k and top-p, 18 us, one launch, latency; 64 rows of 128,256
// (fp32, mixed settings) 51-54 us; 256 rows of 128,256 (binary16, top-p) 97 us, and of 128,257, whose rows lie at no
// 16-byte border and are read by element, 145.  Traced apart the five launches of those 256 rows take 101 us: max 15 (66
// MB at 4.4 TB/s), hist 32 (28 vector instructions a logit, which keep their units busy 93 % of it), cut 8, pick 22, draw
// 25 (latency of a workgroup).  Left: a slice's first loads ahead of its row's settings (their registers cost a
// workgroup of four per CU: hist 34 -> 37 us).
#include "bpdq_paged.h"

namespace bpdq {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;  // of a row's workgroup
constexpr int kRow = 32768;  // elements of a row that its workgroup holds in registers
constexpr int kSliceThreads = 512;
constexpr int kBuckets = 1024;
constexpr int kList = 4096;  // entries of a list that is sorted
constexpr int kMaxSlice = 16384;  // elements of a slice at most: 32 for a thread, marked in one word
constexpr int kSlices = 256;  // of a row at most
static_assert((int64_t)kSlices * kMaxSlice >= 1 << 22, "the largest vocab");
typedef unsigned long long u64;

__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);  // -0 becomes +0: they are equal
    const uint32_t k = (u >> 31) ? ~u : u | 0x80000000u;
    return x != x || x == -__builtin_inff() ? 0u : k;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float((key >> 31) ? key & 0x7FFFFFFFu : ~key);
}

// Buckets and weights go by the distance from the largest logit, d = (max - l) scale in binary64, b = d rounded:
//   exp((l - max) / t) = exp(-b c) exp(-(d - b) c),  c = 1 / (scale t) <= 1 / 32,
// the first from a table of the buckets (2^shift times it), the second by 6 terms of its series: 2^-54 of it is left
// out.
struct Row {
    float top;            // the largest logit
    double max, scale;    // top, buckets per unit of logit
    double k[6];          // (-c)^j / j!
    double c, t;
    int shift;            // weights are multiples of 2^-shift
    const double* table;  // in LDS, kBuckets of them
    // x up to max.  Grows as logits fall, up to the last bucket's, where only logits are that weigh nothing, -infinity
    // and NaN
    __device__ __forceinline__ double distance(double x) const {
        return __builtin_fmin((max - x) * scale, kBuckets - 0.6);
    }
    __device__ __forceinline__ int bucket(double x) const {
        return (int)(uint32_t)__double_as_longlong(distance(x) + 6755399441055744.0);  // 1.5 2^52: rounds, low bits
    }
    // 2^shift exp((x - top) / t) up to some units of 2^-52 of it, exactly 2^shift for the largest logit; 0 in
    // the last bucket
    __device__ __forceinline__ double power(float x, int& b) const {
        const double magic = 6755399441055744.0, d = distance((double)x), to = d + magic, r = d - (to - magic);
        b = (int)(uint32_t)__double_as_longlong(to);
        double p = __builtin_fma(r, k[5], k[4]);
        p = __builtin_fma(r, p, k[3]);
        p = __builtin_fma(r, p, k[2]);
        p = __builtin_fma(r, p, k[1]);
        p = __builtin_fma(r, p, k[0]);
        p = __builtin_fma(r, p, 1.0);
        return p * table[b];
    }
    // at most 2^44: adding 2^52 rounds to an integer and leaves it in the low bits
    __device__ __forceinline__ u64 weight(float x, int& b) const {
        return (u64)__double_as_longlong(power(x, b) + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
    }
    __device__ __forceinline__ u64 weight(float x) const {
        int b;
        return weight(x, b);
    }
    // where the largest may be infinite
    __device__ __forceinline__ u64 weight_of(uint32_t key) const {
        return logit_of(key) == top ? 1ull << shift : weight(logit_of(key));
    }
    // min-p's rule; above 1 no weight reaches it, and the first of the largest logits is the caller's to keep
    __device__ __forceinline__ bool passes(uint32_t key, float min_p) const {
        const float x = logit_of(key);
        if (!(min_p > 0.f)) return true;
        if (x == top) return min_p <= 1.f;
        if (!(min_p < 1.f)) return false;
        if (!(min_p > 0x1p-45f)) return exp(((double)x - max) / t) >= (double)min_p;  // beyond the table
        int b;
        return power(x, b) >= (double)min_p * (double)(1ull << shift);
    }
    template <int THREADS>
    __device__ __forceinline__ void fill(double* to) const {
        for (int b = (int)threadIdx.x; b < kBuckets; b += THREADS)
            to[b] = b < kBuckets - 1 ? exp(-(double)b * c) * (double)(1ull << shift) : 0.0;
    }
};

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// Exclusive sum over the workgroup, the total in `all`.
template <int THREADS, typename T>
__device__ __forceinline__ T scan_block(T v, T& all, T* s_part) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    T run = v;
    for (int d = 1; d < 64; d <<= 1) {
        const T o = __shfl_up(run, d);
        if (lane >= d) run += o;
    }
    __syncthreads();
    if (lane == 63) s_part[wave] = run;
    __syncthreads();
    constexpr int W = THREADS / 64;
    T sums = s_part[lane & (W - 1)];
    for (int d = 1; d < W; d <<= 1) {
        const T o = __shfl_up(sums, d);
        if (lane >= d) sums += o;
    }
    all = __shfl(sums, W - 1);
    const T before = __shfl(sums, (wave + 63) & 63);  // of the waves before this one
    return (wave > 0 ? before : 0) + run - v;
}

// The settings of a row.
struct Set {
    float t, p, m, u;
    int k;
    bool greedy;
};
__device__ __forceinline__ Set settings(const SampleArgs& g, int row) {
    Set s;
    s.t = g.temperature != nullptr ? g.temperature[row] : 1.f;
    s.greedy = !(s.t > 0.f);
    s.p = g.top_p != nullptr ? g.top_p[row] : 1.f;
    s.m = g.min_p != nullptr ? g.min_p[row] : 0.f;
    s.k = g.top_k != nullptr ? g.top_k[row] : 0;
    s.u = g.u[row];
    return s;
}

enum Mode { kWeights, kTopK, kGreedy, kNone, kSearch };

struct Max {
    float top, low;  // largest and smallest logit
    uint32_t n;      // how many
};
// What stays of a slice whatever the list says, and the entries of its list.
struct Sum {
    u64 w;
    uint32_t n, list;
};
// The buckets [0, first) stay, logits from x1 on; those below from x2 on are listed; top-p: weight to be reached
// within the list.
struct Pick {
    u64 want;
    int first;
    float x1, x2;
};
struct Work {
    int S, len;  // slices, elements of one
    int shift;
    Max* max;        // [row][S]
    Sum* sum;        // [row][S]
    Pick* pick;      // [row]
    u64* weight;     // [row][S][kBuckets], or in the same place
    uint32_t* count; // [row][S][2 kBuckets], the first half used
    uint16_t* list;  // [row][S][len]: indices within the slice
};

// Each element of [lo, hi) of a row, 16 bytes at a time and thread, four of those under way at once.
template <typename X, int THREADS, typename F>
__device__ __forceinline__ void each(const X* __restrict__ x, int lo, int hi, F&& f) {
    constexpr int N = 16 / (int)sizeof(X), STEP = THREADS * N;
    const bool aligned = ((uintptr_t)(x + lo) & 15) == 0;
    if (aligned && (hi - lo) % (4 * STEP) == 0) {  // nothing to check
        for (int i0 = lo; i0 < hi; i0 += 4 * STEP) {
            Vec<X, N> v[4];
#pragma unroll
            for (int c = 0; c < 4; c++)
                v[c] = *reinterpret_cast<const Vec<X, N>*>(x + i0 + c * STEP + (int)threadIdx.x * N);
#pragma unroll
            for (int c = 0; c < 4; c++)
#pragma unroll
                for (int j = 0; j < N; j++) f(i0 + c * STEP + (int)threadIdx.x * N + j, (float)v[c].v[j]);
        }
        return;
    }
    for (int i0 = lo + (int)threadIdx.x * N; i0 < hi; i0 += 4 * STEP) {
        Vec<X, N> v[4];
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const int i = i0 + c * STEP;
            if (aligned && i + N <= hi) {
                v[c] = *reinterpret_cast<const Vec<X, N>*>(x + i);
            } else {
#pragma unroll
                for (int j = 0; j < N; j++) v[c].v[j] = i + j < hi ? x[i + j] : (X)-__builtin_inff();
            }
        }
#pragma unroll
        for (int c = 0; c < 4; c++) {
            if (i0 + c * STEP >= hi) break;
#pragma unroll
            for (int j = 0; j < N; j++) f(i0 + c * STEP + j, (float)v[c].v[j]);  // -infinity behind the end
        }
    }
}

__device__ __forceinline__ void join(Max& a, float top, float low, uint32_t n) {
    a.top = fmaxf(a.top, top);
    a.low = fminf(a.low, low);
    a.n += n;
}
__device__ __forceinline__ void join_wave(Max& a) {
    for (int d = 1; d < 64; d <<= 1) join(a, __shfl_xor(a.top, d), __shfl_xor(a.low, d), __shfl_xor(a.n, d));
}

// ---- max: in every thread, and what the thread itself met
// (visit(f) calls f(index, logit) for a thread's part of the elements)
template <int THREADS, typename VISIT>
__device__ __forceinline__ Max part_max(VISIT&& visit, Max* s_part, float& mine) {
    Max m = {-__builtin_inff(), __builtin_inff(), 0u};
    visit([&](int, float v) {
        const bool is = v > -__builtin_inff();
        m.top = fmaxf(m.top, v);
        m.low = is ? fminf(m.low, v) : m.low;
        m.n += is;
    });
    mine = m.top;
    join_wave(m);
    if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = m;
    __syncthreads();
    m = s_part[0];
    for (int i = 1; i < THREADS / 64; i++) join(m, s_part[i].top, s_part[i].low, s_part[i].n);
    m.top += 0.f;  // -0 is 0
    return m;
}

__device__ __forceinline__ Row row_of(const Set& set, const Max& m, int shift, const double* table) {
    Row r;
    r.top = m.top;
    r.max = (double)m.top;
    r.t = (double)set.t;
    // 32 to a unit of (l - max) / t, which weighs nothing beyond kBuckets of them; a smaller range of logits
    // is cut finer, up to the bucket before the last
    r.scale = __builtin_fmin(__builtin_fmax(32.0 / r.t, (kBuckets - 2) / (r.max - (double)m.low)), 1e300);
    r.c = __builtin_fmin(1.0 / (r.scale * r.t), 1.0 / 32);
    r.k[0] = -r.c;
    r.k[1] = r.c * r.c * (1.0 / 2);
    r.k[2] = r.k[1] * r.c * (-1.0 / 3);
    r.k[3] = r.k[2] * r.c * (-1.0 / 4);
    r.k[4] = r.k[3] * r.c * (-1.0 / 5);
    r.k[5] = r.k[4] * r.c * (-1.0 / 6);
    r.shift = shift;
    r.table = table;
    return r;
}

__device__ __forceinline__ Mode mode_of(const Set& s, const Max& m) {
    if (m.n == 0) return kNone;
    if (s.greedy) return kGreedy;
    if (m.top == __builtin_inff()) return kSearch;
    if (s.k > 0 && (uint32_t)s.k < m.n) return s.k > kList ? kSearch : kTopK;
    return kWeights;
}

// ---- hist: into hw (kTopK: counts in its first half), cleared before; ends with a barrier
template <typename VISIT>
__device__ __forceinline__ void part_hist(VISIT&& visit, const Row& r, Mode mode, u64* hw) {
    if (mode == kTopK) {
        uint32_t* hc = reinterpret_cast<uint32_t*>(hw);
        visit([&](int, float v) {
            // the last bucket's are what the others leave, and not asked for
            const int b = r.bucket((double)v);
            if (b < kBuckets - 1) atomicAdd(&hc[b], 1u);
        });
    } else {
        visit([&](int, float v) {  // in the last bucket few weigh anything
            int b;
            const u64 w = r.weight(v, b);
            if (w != 0) atomicAdd(&hw[b], w);
        });
    }
    __syncthreads();
}

// Weight that top-p has to reach of a total.
__device__ __forceinline__ u64 reach(float p, u64 total) {
    const double need = __builtin_ceil((double)(p > 0.f ? p : 0.f) * (double)total);
    const u64 want = need >= (double)total ? total : (u64)need;
    return want == 0 ? 1 : want;
}

// The smallest finite logit in the buckets before `end`, 1 or more; the lowest of all at kBuckets.  The whole wave.
__device__ __forceinline__ float lowest_before(const Row& r, int end) {
    constexpr uint32_t kLowest = 0x00800000u;  // the key of -FLT_MAX
    uint32_t lo = kLowest - 1, hi = end < kBuckets ? key_of(r.top) : kLowest;  // in (lo, hi]
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 63) >> 6, k = lo + (((uint32_t)threadIdx.x & 63) + 1) * step;
        const int l = __builtin_ctzll(__ballot(k >= hi || r.bucket((double)logit_of(k)) < end));  // the last lane's is
        hi = min(hi, lo + (uint32_t)(l + 1) * step);
        lo += (uint32_t)l * step;
    }
    return logit_of(hi);
}

// ---- pick, first half: which logits, from the row's histogram of S slices, `stride` apart (of T); every thread
template <typename T>
struct FindLds {
    T part[kWaves], before;
    int bucket;
    float x[2];
};
template <typename T>
__device__ __forceinline__ Pick find_buckets(const T* hist, int stride, int S, const Row& r, const Set& set, Mode mode,
                                             FindLds<T>& s) {
    static_assert(kBuckets == kThreads, "a thread for each");
    const int tid = (int)threadIdx.x;
    T v = 0, total;
#pragma unroll 8
    for (int i = 0; i < S; i++) v += hist[(int64_t)i * stride + tid];
    if (tid == 0) s.bucket = kBuckets - 1;
    const T before = scan_block<kThreads>(v, total, s.part);
    const bool by_p = mode == kWeights && set.p < 1.f;
    const T need = mode == kTopK ? (T)set.k : by_p ? (T)reach(set.p, (u64)total) : 0;
    if (before < need && before + v >= need) s.bucket = tid;  // one thread, or none
    __syncthreads();
    Pick p = {~0ull, 0, __builtin_inff(), 0.f};
    int last = s.bucket;
    if (mode != kTopK) {
        p.first = last = by_p ? last : kBuckets;
        if (set.m > 0.f) {
            // min-p's own cut lies between the logits x + off and x - off
            const double x = r.max + log((double)fminf(set.m, 1.f)) * r.t;
            const double off = 1e-6 * (__builtin_fabs(r.max) + __builtin_fabs(x)) + 1e-30;
            p.first = min(p.first, r.bucket(__builtin_fmin(x + off, r.max)));
            last = min(last, r.bucket(x - off));
        }
        if (by_p && tid == p.first) s.before = before;
    }
    if (tid < 128) {
        const int end = __builtin_amdgcn_readfirstlane(tid < 64 ? p.first : last < kBuckets - 1 ? last + 1 : kBuckets);
        const float x = end > 0 ? lowest_before(r, end) : __builtin_inff();
        if ((tid & 63) == 0) s.x[tid >> 6] = x;
    }
    __syncthreads();
    p.x1 = s.x[0];
    p.x2 = s.x[1];
    if (by_p) p.want = (u64)need - (u64)s.before;
    return p;
}

// ---- pick, second half: bit k of `listed` for the k-th element that visit shows the thread, 32 at most; returns
// how many stay, by thread
template <typename VISIT>
__device__ __forceinline__ uint32_t part_pick(VISIT&& visit, const Pick& p, uint32_t& listed) {
    uint32_t n = 0, bit = 1;
    listed = 0;
    visit([&](int, float v) {
        const bool stays = v >= p.x1;
        n += stays;
        listed |= v >= p.x2 && !stays ? bit : 0u;
        bit <<= 1;
    });
    return n;
}
// Weight of the buckets before `first`, by thread.
template <int THREADS>
__device__ __forceinline__ u64 staying(const u64* hw, const Pick& p) {
    u64 w = 0;
    for (int i = (int)threadIdx.x; i < min(p.first, kBuckets); i += THREADS) w += hw[i];
    return w;
}

__device__ __forceinline__ void answer(const SampleArgs& g, int row, int token, float logprob, uint32_t kept) {
    g.token[row] = token;
    if (g.logprob != nullptr) g.logprob[row] = logprob;
    if (g.kept != nullptr) g.kept[row] = (int32_t)kept;
}

// Weight that the cumulated sum has to exceed.
__device__ __forceinline__ u64 draw_target(float u, u64 total) {
    const double at = (u > 0.f ? (u < 1.f ? (double)u : 1.0) : 0.0) * (double)total;
    return at >= (double)total ? total - 1 : (u64)at;
}

// The row digit by digit, a pass for every question, by one workgroup.  The cut is a key and how many that
// equal it, from the first index on, stay.
struct SearchLds {
    uint32_t hc[256];
    u64 hw[256];
    u64 part[kWaves];
    uint32_t ties[kWaves];
    uint32_t key, cnt;
    u64 w;
};
template <typename X>
__device__ __forceinline__ void search_row(const SampleArgs& g, int row, const X* x, const Row& r, const Set& set,
                                           uint32_t n, SearchLds& s) {
    auto& hc = s.hc;
    auto& ties = s.ties;
    auto& hw = s.hw;
    auto& part = s.part;
    auto &s_key = s.key, &s_cnt = s.cnt;
    auto& s_w = s.w;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int V = g.V;
    auto key_at = [&](int i) { return key_of((float)x[i]); };
    const int kk = set.k;
    const float pf = set.p, mf = set.m;
    uint32_t cut = 1, tie = 0xFFFFFFFFu, kept = n;  // all keys above 0
    // The cut at which count (by_weight: weight) of keys from the largest down first reaches `need`.
    auto select = [&](bool by_weight, u64 need, uint32_t& above, u64& wabove) {
        uint32_t prefix = 0;
        above = 0;
        wabove = 0;
        for (int bit = 24; bit >= 0; bit -= 8) {
            if (tid < 256) hc[tid] = 0, hw[tid] = 0;
            __syncthreads();
            for (int i = tid; i < V; i += kThreads) {
                const uint32_t k = key_at(i);
                if (k < cut || (bit < 24 && (k >> (bit + 8)) != prefix)) continue;
                atomicAdd(&hc[(k >> bit) & 255], 1u);
                // ties beyond the cut's number weigh nothing: taken off below
                if (by_weight) atomicAdd(&hw[(k >> bit) & 255], (u64)r.weight_of(k));
            }
            __syncthreads();
            if (by_weight && tid == 0 && cut > 1 && (bit == 24 || (cut >> (bit + 8)) == prefix)) {
                // count the ties in this digit's bucket only up to `tie`
                hw[(cut >> bit) & 255] -= s_w;
                hc[(cut >> bit) & 255] -= s_cnt;
            }
            __syncthreads();
            if (tid == 0) {
                int d = 255;
                for (; d > 0; d--) {
                    const u64 have = by_weight ? wabove + hw[d] : (u64)above + hc[d];
                    if (have >= need) break;
                    above += hc[d];
                    wabove += hw[d];
                }
                s_key = (prefix << 8) | (uint32_t)d;
                part[0] = above;
                part[1] = wabove;
            }
            __syncthreads();
            prefix = s_key;
            above = (uint32_t)part[0];
            wabove = part[1];
            __syncthreads();
        }
        return prefix;
    };
    auto count_ties = [&](uint32_t key) {
        __syncthreads();
        if (tid == 0) s_cnt = 0;
        __syncthreads();
        uint32_t c = 0;
        for (int i = tid; i < V; i += kThreads) c += key_at(i) == key;
        c = wave_sum(c);
        if (lane == 0 && c) atomicAdd(&s_cnt, c);
        __syncthreads();
        const uint32_t all = s_cnt;
        __syncthreads();
        return all;
    };
    {
        if (kk > 0 && (uint32_t)kk < n) {
            uint32_t above;
            u64 w;
            cut = select(false, (u64)kk, above, w);
            tie = (uint32_t)kk - above;
            kept = (uint32_t)kk;
        }
        if (pf < 1.f) {
            const uint32_t more = tie == 0xFFFFFFFFu ? 0 : count_ties(cut) - tie;  // ties that top_k left out
            if (tid == 0) s_cnt = more, s_w = more * r.weight_of(cut);
            __syncthreads();
            u64 total = 0;
            for (int i = tid; i < V; i += kThreads) {
                const uint32_t k = key_at(i);
                if (k >= cut) total += r.weight_of(k);
            }
            total = wave_sum(total);
            if (lane == 0) part[wave] = total;
            __syncthreads();
            total = 0;
            for (int w = 0; w < kWaves; w++) total += part[w];
            total -= s_w;
            __syncthreads();
            const u64 want = reach(pf, total);
            uint32_t above;
            u64 wabove;
            const uint32_t key = select(true, want, above, wabove);
            const uint64_t each = r.weight_of(key);
            const uint32_t num = each == 0 ? 1 : (uint32_t)((want - wabove + each - 1) / each);
            cut = key;
            tie = num;
            kept = above + num;
        }
        if (mf > 1.f) {  // the first of the largest alone
            cut = key_of(r.top);
            tie = kept = 1;
        } else if (mf > 0.f) {  // weights fall with the key: the cut moves up to the last key at or above min_p
            __syncthreads();
            if (tid == 0) s_cnt = 0, s_key = 0xFFFFFFFFu;
            __syncthreads();
            uint32_t c = 0, low = 0xFFFFFFFFu;
            for (int i = tid; i < V; i += kThreads) {
                const uint32_t k = key_at(i);
                if (k < cut || !r.passes(k, mf)) continue;
                low = min(low, k);
                c += k > cut;
            }
            c = wave_sum(c);
            for (int d = 1; d < 64; d <<= 1) low = min(low, (uint32_t)__shfl_xor(low, d));
            if (lane == 0) atomicAdd(&s_cnt, c), atomicMin(&s_key, low);
            __syncthreads();
            const uint32_t l = s_key, cc = s_cnt;
            __syncthreads();
            if (l > cut || cut == 1) {
                cut = l;
                tie = 0xFFFFFFFFu;
                kept = cc;
                if (cut == 1) kept = n;
            } else {
                kept = cc + min(tie, count_ties(cut));
            }
        }
    }
    // The draw.  Wave w owns indices [w seg, w seg + seg): weights above the cut and ties of each
    // segment, then the segment, then the place in it.
    const int seg = (V + kWaves * 64 - 1) / (kWaves * 64) * 64;
    const int lo = min(V, wave * seg), hi = min(V, lo + seg);
    const uint64_t wc = r.weight_of(cut);
    u64 w = 0;
    uint32_t tc = 0;
    for (int i = lo + lane; i < hi; i += 64) {
        const uint32_t k = key_at(i);
        if (k > cut) w += r.weight_of(k);
        tc += k == cut;
    }
    w = wave_sum(w);
    tc = wave_sum(tc);
    __syncthreads();
    if (lane == 0) part[wave] = w, ties[wave] = tc;
    __syncthreads();
    u64 total = 0, before = 0;
    uint32_t tb = 0;
    for (int i = 0; i < kWaves; i++) {
        const uint32_t took = min(ties[i], tie > tb ? tie - tb : 0u);
        total += part[i] + took * wc;
        tb += ties[i];
    }
    const u64 target = draw_target(g.u[row], total);  // chosen: sum > target
    tb = 0;
    int chosen = 0;
    uint32_t left = 0;
    for (int i = 0; i < kWaves; i++) {
        left = tie > tb ? tie - tb : 0u;
        const u64 mine = part[i] + min(ties[i], left) * wc;
        if (before + mine > target) {
            chosen = i;
            break;
        }
        before += mine;
        tb += ties[i];
    }
    if (wave != chosen) return;
    for (int i0 = lo; i0 < hi; i0 += 64) {
        const int i = i0 + lane;
        const uint32_t k = i < hi ? key_at(i) : 0;
        const uint64_t same = __ballot(i < hi && k == cut);
        const bool in = i < hi && (k > cut || (k == cut && (uint32_t)__popcll(same & ((1ull << lane) - 1)) < left));
        const u64 mine = in ? r.weight_of(k) : 0;
        u64 run = mine;
        for (int d = 1; d < 64; d <<= 1) {
            const u64 o = __shfl_up(run, d);
            if (lane >= d) run += o;
        }
        const uint64_t over = __ballot(before + run > target);
        if (over != 0) {
            if (lane == __ffsll((u64)over) - 1) {
                answer(g, row, i, (float)log((double)mine / (double)total), kept);
            }
            return;
        }
        before += __shfl(run, 63);
        const uint32_t used = (uint32_t)__popcll(same);
        left = left > used ? left - used : 0u;
    }
}

// Sorts n different values of LDS, falling.  Up to 256 find their places by counting those above them, four threads
// each (1.6 us against 2.9); more go through a bitonic network: up to 1024 each thread holds one, and
// partners less than 64 apart are asked by shuffles.
__device__ __forceinline__ void sort_falling(u64* a, int n, uint32_t* s_rank) {
    const int tid = (int)threadIdx.x;
    if (n <= kThreads / 4) {
        const int e = tid & 255, j0 = (tid >> 8) * ((n + 3) >> 2), j1 = min(n, j0 + ((n + 3) >> 2));
        if (tid < 256) s_rank[tid] = 0;
        __syncthreads();
        const u64 v = e < n ? a[e] : 0;
        uint32_t rank = 0;
        if ((e & ~63) < n) {
#pragma unroll 8
            for (int j = j0; j < j1; j++) rank += a[j] > v;
        }
        if (e < n && rank != 0) atomicAdd(&s_rank[e], rank);
        __syncthreads();
        if (tid < n) a[s_rank[tid]] = v;
        __syncthreads();
        return;
    }
    if (n <= kThreads) {
        u64 v = tid < n ? a[tid] : 0;
        for (int k = 2; k < 2 * n; k <<= 1)
            for (int j = k >> 1; j > 0; j >>= 1) {
                u64 o;
                if (j >= 64) {
                    __syncthreads();
                    a[tid] = v;
                    __syncthreads();
                    o = a[tid ^ j];
                } else {
                    o = __shfl_xor(v, j);
                }
                const bool larger = ((tid & k) == 0) == ((tid & j) == 0);
                v = (v > o) == larger ? v : o;
            }
        __syncthreads();
        a[tid] = v;
        __syncthreads();
        return;
    }
    int n2 = 2 * kThreads;
    while (n2 < n) n2 <<= 1;
    for (int i = n + tid; i < n2; i += kThreads) a[i] = 0;
    __syncthreads();
    for (int k = 2; k <= n2; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int i = tid; i < n2 / 2; i += kThreads) {
                const int x = 2 * i - (i & (j - 1)), y = x + j;  // x has bit j clear
                const u64 p = a[x], q = a[y];
                if ((p < q) == ((x & k) == 0)) a[x] = q, a[y] = p;
            }
            __syncthreads();
        }
}

struct DrawLds {
    u64 list[kList];  // (key, ~index), later (~index, key)
    u64 part[kWaves];
    u64 slice[kSlices];
    uint32_t rank[kThreads / 4];
    u64 before;
    uint32_t n, kept;
    int chosen;
};

// ---- draw: from the list (n_list entries, in LDS), n_stay logits that stay whatever it says and the slices'
// weights of those; S slices of len elements.  kThreads threads.
template <typename X>
__device__ __forceinline__ void draw_row(const SampleArgs& g, int row, const X* x, const Row& r, const Set& set,
                                         Mode mode, const Pick& pick, const Sum* sums, int S, int len, uint32_t n_list,
                                         uint32_t n_stay, DrawLds& s) {
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    sort_falling(s.list, (int)n_list, s.rank);  // by logit, equal ones by index
    // how many of the list stay.  Every loop here is kept rolled: a row's workgroup runs through this code
    // once, and waits for its instructions more than for its data
    const int n_ranked = mode == kTopK ? min((int)n_list, set.k) : (int)n_list;
    u64 total = 0, want = pick.want;
    if (mode == kTopK && set.p < 1.f) {  // the total of the top-k first
        u64 mine = 0;
#pragma unroll 1
        for (int i = tid; i < n_ranked; i += kThreads) mine += r.weight_of((uint32_t)(s.list[i] >> 32));
        scan_block<kThreads>(mine, total, s.part);
        want = reach(set.p, total);
    }
    u64 run0 = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < n_ranked; i0 += kThreads) {
        const int i = i0 + tid;
        const uint32_t k = i < n_ranked ? (uint32_t)(s.list[i] >> 32) : 0;
        u64 all = 0, run = run0;
        if (want != ~0ull) run += scan_block<kThreads>(i < n_ranked ? r.weight_of(k) : 0, all, s.part);
        // what stands before it falls short of what is wanted
        const bool largest = i == 0 && n_stay == 0;  // min-p leaves it in any case
        const uint64_t stay = __ballot(i < n_ranked && run < want && (largest || r.passes(k, set.m)));
        if (lane == 0 && stay != 0) atomicAdd(&s.kept, (uint32_t)__popcll(stay));
        run0 += all;
    }
    __syncthreads();
    const uint32_t kept_list = s.kept, kept = kept_list + n_stay;

    if (mode == kTopK) {
        // all that stays is in the list: sorted by index, the draw
        for (int i = tid; i < (int)kept_list; i += kThreads) {
            const u64 e = s.list[i];
            s.list[i] = e << 32 | e >> 32;
        }
        __syncthreads();
        sort_falling(s.list, (int)kept_list, s.rank);  // ~index falls
        for (int pass = 0; pass < 2; pass++) {  // the total, then the place
            const u64 target = pass == 0 ? 0 : draw_target(set.u, total);
            run0 = 0;
#pragma unroll 1
            for (int i0 = 0; i0 < (int)kept_list; i0 += kThreads) {
                const int i = i0 + tid;
                const u64 e = i < (int)kept_list ? s.list[i] : 0, v = i < (int)kept_list ? r.weight_of((uint32_t)e) : 0;
                u64 all;
                const u64 run = run0 + scan_block<kThreads>(v, all, s.part);
                run0 += all;
                if (pass == 0 && kept_list > (uint32_t)kThreads) continue;
                const u64 t = kept_list > (uint32_t)kThreads ? target : draw_target(set.u, all);
                const u64 sum = pass == 0 ? all : total;
                if (run <= t && run + v > t)
                    answer(g, row, (int)~(uint32_t)(e >> 32), (float)log((double)v / (double)sum), kept);
            }
            total = run0;
            if (kept_list <= (uint32_t)kThreads) break;  // one round said it all
        }
        return;
    }
    // a head of the list stays, up to this one; where none does, the buckets before it alone
    const u64 cut = kept_list > 0 ? s.list[kept_list - 1] : 0;
    // the slice: what stays of each is its sum and its part of the list
    if (tid < kSlices) s.slice[tid] = tid < S ? sums[tid].w : 0;
    __syncthreads();
    for (int i = tid; i < (int)kept_list; i += kThreads)
        atomicAdd(&s.slice[S == 1 ? 0 : (int)(~(uint32_t)s.list[i]) / len], r.weight_of((uint32_t)(s.list[i] >> 32)));
    __syncthreads();
    {
        const u64 w = tid < kSlices ? s.slice[tid] : 0, at = scan_block<kThreads>(w, total, s.part);
        const u64 target = draw_target(set.u, total);
        if (at <= target && at + w > target) {
            s.chosen = tid;
            s.before = at;
        }
    }
    __syncthreads();
    // the place in the slice: a thread weighs some elements in a row, then a wave those of the thread that it falls to
    const u64 target = draw_target(set.u, total);
    constexpr int N = 16 / (int)sizeof(X);
    const int lo = s.chosen * len, hi = min(g.V, lo + len);
    const int per = (min(len, g.V) + 8 * kThreads - 1) / (8 * kThreads) * 8;  // 32 at most
    auto weight_at = [&](float f, int i) -> u64 {
        const bool in = f >= pick.x1 || (cut != 0 && ((u64)key_of(f) << 32 | (uint32_t)~(uint32_t)i) >= cut);
        return in ? r.weight(f) : 0;
    };
    const bool aligned = ((uintptr_t)(x + lo) & 15) == 0;
    const int a0 = lo + tid * per;
    u64 mine = 0;
#pragma unroll 1
    for (int i0 = a0; i0 < min(hi, a0 + per); i0 += 16) {
        Vec<X, N> v[16 / N];
#pragma unroll
        for (int c = 0; c < 16 / N; c++) {
            const int i = i0 + c * N, end = min(hi, a0 + per);
            if (aligned && i + N <= end) {
                v[c] = *reinterpret_cast<const Vec<X, N>*>(x + i);
            } else {
#pragma unroll
                for (int j = 0; j < N; j++) v[c].v[j] = i + j < end ? x[i + j] : (X)-__builtin_inff();
            }
        }
#pragma unroll
        for (int c = 0; c < 16 / N; c++)
#pragma unroll
            for (int j = 0; j < N; j++) mine += weight_at((float)v[c].v[j], i0 + c * N + j);
    }
    auto up_to = [&](u64 sum) {  // over the lanes up to this one
        for (int d = 1; d < 64; d <<= 1) {
            const u64 o = __shfl_up(sum, d);
            if (lane >= d) sum += o;
        }
        return sum;
    };
    const u64 run = up_to(mine);
    __syncthreads();
    if (lane == 63) s.part[wave] = run;
    __syncthreads();
    u64 before = s.before;
    int chosen = 0;
    for (; chosen < kWaves - 1 && before + s.part[chosen] <= target; chosen++) before += s.part[chosen];
    if (wave != chosen) return;
    const uint64_t past = __ballot(before + run > target);
    if (past == 0) return;
    const int who = __builtin_ctzll(past);
    before += __shfl(run - mine, who);
    const int i = lo + (wave * 64 + who) * per + lane;
    const u64 v = lane < per && i < hi ? weight_at((float)x[i], i) : 0;
    const uint64_t over = __ballot(before + up_to(v) > target);
    if (over != 0 && lane == __builtin_ctzll(over)) answer(g, row, i, (float)log((double)v / (double)total), kept);
}

// The first index of the largest logit, which [lo, hi) holds.
template <typename X>
__device__ __forceinline__ void greedy_row(const SampleArgs& g, int row, const X* x, int lo, int hi, float top,
                                           uint32_t* s_at) {
    if (threadIdx.x == 0) *s_at = 0xFFFFFFFFu;
    __syncthreads();
    uint32_t at = 0xFFFFFFFFu;
    each<X, kThreads>(x, lo, hi, [&](int i, float v) {
        if (v == top) at = min(at, (uint32_t)i);
    });
    if (at != 0xFFFFFFFFu) atomicMin(s_at, at);
    __syncthreads();
    if (threadIdx.x == 0) answer(g, row, (int)*s_at, 0.f, 1);
}

union RowLds {
    DrawLds draw;
    SearchLds search;
};

// ---- one workgroup per row
template <int TYPE>
__global__ __launch_bounds__(kThreads) void k_sample_row(SampleArgs g, int shift) {
    using X = typename Elem<TYPE>::type;
    __shared__ double table[kBuckets];
    __shared__ u64 hw[kBuckets];
    __shared__ Max s_max[kWaves];
    __shared__ u64 s_part[kWaves];
    __shared__ union {
        FindLds<u64> w;
        FindLds<uint32_t> n;
    } s_find;
    __shared__ Sum s_sum;
    __shared__ RowLds s;
    const int row = (int)blockIdx.x, tid = (int)threadIdx.x;
    const Set set = settings(g, row);
    const X* x = reinterpret_cast<const X*>(g.logits) + (int64_t)row * g.stride;
    hw[tid] = 0;
    if (tid == 0) s.draw.n = s.draw.kept = 0;
    // the row's kRow elements at most stay in registers
    constexpr int N = 16 / (int)sizeof(X), NV = kRow / (kThreads * N);
    Vec<X, N> held[NV];
    const bool aligned = ((uintptr_t)x & 15) == 0;
#pragma unroll
    for (int c = 0; c < NV; c++) {
        const int i = (c * kThreads + tid) * N;
        if (aligned && i + N <= g.V) {
            held[c] = *reinterpret_cast<const Vec<X, N>*>(x + i);
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) held[c].v[j] = i + j < g.V ? x[i + j] : (X)-__builtin_inff();
        }
    }
    auto visit = [&](auto&& f) {
#pragma unroll
        for (int c = 0; c < NV; c++) {
            if (c * kThreads * N >= g.V) break;
#pragma unroll
            for (int j = 0; j < N; j++) f((c * kThreads + tid) * N + j, (float)held[c].v[j]);
        }
    };
    float mine;
    const Max m = part_max<kThreads>(visit, s_max, mine);
    const Mode mode = mode_of(set, m);
    if (mode == kNone) {
        if (tid == 0) answer(g, row, -1, __builtin_nanf(""), 0);
        return;
    }
    if (mode == kGreedy) {
        greedy_row(g, row, x, 0, g.V, m.top, &s.search.key);
        return;
    }
    const Row r = row_of(set, m, shift, table);
    r.fill<kThreads>(table);
    __syncthreads();
    if (mode != kSearch) {
        // top-k of few: where k threads' largest logits stand, k logits stand, so that these alone are counted (the
        // histogram of all 32,000: 2.8 us)
        if (mode == kTopK && 2 * set.k <= min(kThreads, g.V / N)) part_hist([&](auto&& f) { f(0, mine); }, r, mode, hw);
        else part_hist(visit, r, mode, hw);
        const uint32_t* hc = reinterpret_cast<const uint32_t*>(hw);
        const Pick pick = mode == kTopK ? find_buckets(hc, 0, 1, r, set, mode, s_find.n)
                                        : find_buckets(hw, 0, 1, r, set, mode, s_find.w);
        uint32_t n_stay = m.n, n_list = 0;
        if (pick.first < kBuckets) {
            uint32_t listed;
            const uint32_t n = part_pick(visit, pick, listed);
            u64 both;  // staying above, listed below
            const u64 at = scan_block<kThreads>((u64)n << 32 | (uint32_t)__popc(listed), both, s_part);
            n_stay = (uint32_t)(both >> 32);
            n_list = (uint32_t)both;
            if (n_list <= (uint32_t)kList && listed != 0) {
                uint32_t to = (uint32_t)at, bit = 1;
                visit([&](int i, float v) {
                    if (listed & bit) s.draw.list[to++] = (u64)key_of(v) << 32 | (uint32_t)~(uint32_t)i;
                    bit <<= 1;
                });
            }
        }
        __syncthreads();
        if (n_list <= (uint32_t)kList) {
            u64 w_stay = 0;
            if (mode == kWeights) scan_block<kThreads>(staying<kThreads>(hw, pick), w_stay, s_part);
            if (tid == 0) s_sum.w = w_stay;
            __syncthreads();
            draw_row(g, row, x, r, set, mode, pick, &s_sum, 1, g.V, n_list, n_stay, s.draw);
            return;
        }
        __syncthreads();
    }
    search_row(g, row, x, r, set, m.n, s.search);
}

// ---- one workgroup per slice
// The row's from its slices, in every wave.
__device__ __forceinline__ Max row_max(const Work& w, int row) {
    Max m = {-__builtin_inff(), __builtin_inff(), 0u};
    for (int i = (int)threadIdx.x & 63; i < w.S; i += 64) {
        const Max o = w.max[(int64_t)row * w.S + i];
        join(m, o.top, o.low, o.n);
    }
    join_wave(m);
    return m;
}

template <int TYPE>
__global__ __launch_bounds__(kSliceThreads) void k_max(SampleArgs g, Work w) {
    using X = typename Elem<TYPE>::type;
    __shared__ Max part[kSliceThreads / 64];
    const int row = (int)(blockIdx.x / (unsigned)w.S), slice = (int)(blockIdx.x % (unsigned)w.S);
    const int lo = slice * w.len, hi = min(g.V, lo + w.len);
    const X* x = reinterpret_cast<const X*>(g.logits) + (int64_t)row * g.stride;
    float mine;
    const Max m = part_max<kSliceThreads>([&](auto&& f) { each<X, kSliceThreads>(x, lo, hi, f); }, part, mine);
    if (threadIdx.x == 0) w.max[blockIdx.x] = m;
}

template <int TYPE>
__global__ __launch_bounds__(kSliceThreads) void k_hist(SampleArgs g, Work w) {
    using X = typename Elem<TYPE>::type;
    __shared__ double table[kBuckets];
    __shared__ u64 hw[kBuckets];
    const int row = (int)(blockIdx.x / (unsigned)w.S), slice = (int)(blockIdx.x % (unsigned)w.S);
    const int tid = (int)threadIdx.x;
    const Set set = settings(g, row);
    const Max m = row_max(w, row);
    const Mode mode = mode_of(set, m);
    if (mode != kWeights && mode != kTopK) return;
    const Row r = row_of(set, m, w.shift, table);
    if (mode == kWeights) r.fill<kSliceThreads>(table);
    for (int i = tid; i < kBuckets; i += kSliceThreads) hw[i] = 0;
    __syncthreads();
    const int lo = slice * w.len, hi = min(g.V, lo + w.len);
    const X* x = reinterpret_cast<const X*>(g.logits) + (int64_t)row * g.stride;
    part_hist([&](auto&& f) { each<X, kSliceThreads>(x, lo, hi, f); }, r, mode, hw);
    const int64_t at = (int64_t)blockIdx.x * kBuckets;
    const int n = mode == kTopK ? kBuckets / 2 : kBuckets;
    for (int i = tid; i < n; i += kSliceThreads) w.weight[at + i] = hw[i];
}

__global__ __launch_bounds__(kThreads) void k_cut(SampleArgs g, Work w) {
    __shared__ union {
        FindLds<u64> w;
        FindLds<uint32_t> n;
    } s;
    const int row = (int)blockIdx.x;
    const Set set = settings(g, row);
    const Max m = row_max(w, row);
    const Mode mode = mode_of(set, m);
    if (mode != kWeights && mode != kTopK) return;
    const Row r = row_of(set, m, w.shift, nullptr);  // no weights here
    const int64_t at = (int64_t)row * w.S;
    const Pick pick = mode == kTopK ? find_buckets(w.count + at * 2 * kBuckets, 2 * kBuckets, w.S, r, set, mode, s.n)
                                    : find_buckets(w.weight + at * kBuckets, kBuckets, w.S, r, set, mode, s.w);
    if (threadIdx.x == 0) w.pick[row] = pick;
}

template <int TYPE>
__global__ __launch_bounds__(kSliceThreads) void k_pick(SampleArgs g, Work w) {
    using X = typename Elem<TYPE>::type;
    constexpr int T = kSliceThreads;
    __shared__ u64 s_part[T / 64];
    const int row = (int)(blockIdx.x / (unsigned)w.S), slice = (int)(blockIdx.x % (unsigned)w.S);
    const int tid = (int)threadIdx.x;
    const Set set = settings(g, row);
    const Max m = row_max(w, row);
    const Mode mode = mode_of(set, m);
    if (mode != kWeights && mode != kTopK) return;
    const Pick pick = w.pick[row];
    const int lo = slice * w.len, hi = min(g.V, lo + w.len);
    uint16_t* list = w.list + (int64_t)blockIdx.x * w.len;
    uint32_t n_all = w.max[blockIdx.x].n, n_list = 0;
    if (pick.first < kBuckets) {
        const X* x = reinterpret_cast<const X*>(g.logits) + (int64_t)row * g.stride;
        uint32_t listed;
        const uint32_t n = part_pick([&](auto&& f) { each<X, T>(x, lo, hi, f); }, pick, listed);
        u64 both;  // staying above, listed below
        const u64 at = scan_block<T>((u64)n << 32 | (uint32_t)__popc(listed), both, s_part);
        n_all = (uint32_t)(both >> 32);
        n_list = (uint32_t)both;
        constexpr int N = 16 / (int)sizeof(X);
        for (uint32_t to = (uint32_t)at; listed != 0; listed &= listed - 1) {
            const int k = __builtin_ctz(listed);
            list[to++] = (uint16_t)((k / N * T + tid) * N + k % N);
        }
    }
    u64 w_all = 0;
    if (mode == kWeights) scan_block<T>(staying<T>(w.weight + (int64_t)blockIdx.x * kBuckets, pick), w_all, s_part);
    __syncthreads();
    if (tid == 0) w.sum[blockIdx.x] = {w_all, n_all, n_list};
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void k_draw(SampleArgs g, Work w) {
    using X = typename Elem<TYPE>::type;
    __shared__ double table[kBuckets];
    __shared__ RowLds s;
    const int row = (int)blockIdx.x, tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Set set = settings(g, row);
    const Max m = row_max(w, row);
    const Mode mode = mode_of(set, m);
    const X* x = reinterpret_cast<const X*>(g.logits) + (int64_t)row * g.stride;
    if (mode == kNone) {
        if (tid == 0) answer(g, row, -1, __builtin_nanf(""), 0);
        return;
    }
    if (mode == kGreedy) {
        int slice = w.S;  // the first with the largest logit
        for (int i = lane; i < w.S; i += 64)
            if (w.max[(int64_t)row * w.S + i].top == m.top) slice = min(slice, i);
        for (int d = 1; d < 64; d <<= 1) slice = min(slice, __shfl_xor(slice, d));
        greedy_row(g, row, x, slice * w.len, min(g.V, (slice + 1) * w.len), m.top, &s.search.key);
        return;
    }
    if (tid == 0) s.draw.n = s.draw.kept = 0;
    const Row r = row_of(set, m, w.shift, table);
    r.fill<kThreads>(table);
    const Sum* sums = w.sum + (int64_t)row * w.S;
    __syncthreads();
    uint32_t n_list = 0, n_stay = 0;
    if (mode != kSearch) {
        for (int i = lane; i < w.S; i += 64) n_list += sums[i].list, n_stay += sums[i].n;
        n_list = wave_sum(n_list);
        n_stay = wave_sum(n_stay);
    }
    if (mode == kSearch || n_list > (uint32_t)kList) {
        search_row(g, row, x, r, set, m.n, s.search);
        return;
    }
    for (int i = wave; i < w.S; i += kWaves) {
        const uint32_t n = sums[i].list;
        const uint16_t* from = w.list + ((int64_t)row * w.S + i) * w.len;
        uint32_t at = 0;
        if (lane == 0 && n > 0) at = atomicAdd(&s.draw.n, n);
        at = __shfl(at, 0);
        for (uint32_t j = lane; j < n; j += 64) {
            const uint32_t idx = (uint32_t)(i * w.len) + from[j];
            s.draw.list[at + j] = (u64)key_of((float)x[idx]) << 32 | (uint32_t)~idx;
        }
    }
    __syncthreads();
    draw_row(g, row, x, r, set, mode, w.pick[row], sums, w.S, w.len, n_list, n_stay, s.draw);
}

int shift_of(int V) {
    int bits = 0;
    while (((int64_t)1 << bits) < V) bits++;
    return bits <= 18 ? 44 : 62 - bits;
}

// Elements of a slice: enough workgroups for the chip, but no more slices of a row than k_draw has sums for.
int slice_len(int B, int V) {
    auto slices = [&](int len) { return (V + len - 1) / len; };
    int len = kMaxSlice;
    while (len > 2048 && (int64_t)B * slices(len) < 1024 && slices(len / 2) <= kSlices) len >>= 1;
    return len;
}

// Whether rows take one workgroup each or one per slice: as long as a workgroup holds them.  Measured at 32,000 logits:
// 1 row 29 us against 33, with top-k 18 against 29; 256 rows 37 against 55.
bool by_row(int V) { return V <= kRow; }

struct Layout {
    int64_t max, sum, pick, weight, list, total;
    int S, len;
};
Layout layout(int B, int V) {
    Layout l = {};
    if (by_row(V)) {
        l.total = 16;
        return l;
    }
    l.len = slice_len(B, V);
    l.S = (V + l.len - 1) / l.len;
    const int64_t n = (int64_t)B * l.S;
    l.sum = up16(n * (int64_t)sizeof(Max));
    l.pick = l.sum + up16(n * (int64_t)sizeof(Sum));
    l.weight = l.pick + up16(B * (int64_t)sizeof(Pick));
    l.list = l.weight + n * kBuckets * 8;
    l.total = l.list + up16(n * l.len * 2);
    return l;
}

template <int TYPE>
void launch_type(const SampleArgs& a, const Work& w, hipStream_t s) {
    if (by_row(a.V)) {
        hipLaunchKernelGGL(k_sample_row<TYPE>, dim3((unsigned)a.B), dim3(kThreads), 0, s, a, w.shift);
        return;
    }
    const dim3 grid((unsigned)w.S * (unsigned)a.B), block(kSliceThreads);
    hipLaunchKernelGGL(k_max<TYPE>, grid, block, 0, s, a, w);
    hipLaunchKernelGGL(k_hist<TYPE>, grid, block, 0, s, a, w);
    hipLaunchKernelGGL(k_cut, dim3((unsigned)a.B), dim3(kThreads), 0, s, a, w);
    hipLaunchKernelGGL(k_pick<TYPE>, grid, block, 0, s, a, w);
    hipLaunchKernelGGL(k_draw<TYPE>, dim3((unsigned)a.B), dim3(kThreads), 0, s, a, w);
}

}  // namespace

int64_t sample_ws(int n_rows, int vocab) { return layout(n_rows, vocab).total; }

void launch_sample(const SampleArgs& a, int type, void* ws, hipStream_t s) {
    const Layout l = layout(a.B, a.V);
    uint8_t* p = static_cast<uint8_t*>(ws);
    Work w;
    w.S = l.S;
    w.len = l.len;
    w.shift = shift_of(a.V);
    w.max = reinterpret_cast<Max*>(p);
    w.sum = reinterpret_cast<Sum*>(p + l.sum);
    w.pick = reinterpret_cast<Pick*>(p + l.pick);
    w.weight = reinterpret_cast<u64*>(p + l.weight);
    w.count = reinterpret_cast<uint32_t*>(p + l.weight);
    w.list = reinterpret_cast<uint16_t*>(p + l.list);
    if (type == BPD_T_F32) launch_type<BPD_T_F32>(a, w, s);
    else if (type == BPD_T_F16) launch_type<BPD_T_F16>(a, w, s);
    else launch_type<BPD_T_BF16>(a, w, s);
}

}  // namespace bpdq
