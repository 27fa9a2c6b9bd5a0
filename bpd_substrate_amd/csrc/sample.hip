// sample.hip — bpd_sample_gpu: one token per row of logits.
//
// A logit's place is its order key: the binary32 bits, sign-folded so that unsigned order is
// the logits' order, 0 for what is never chosen.  All weights are
// W = rint(2^shift exp((l - max) / t)), taken in binary64: their sums are exact in 64 bits,
// so no sum depends on its order.  Every filter keeps a head of the list sorted by
// (logit, index), so it is one cut.
//
// A row is worked on by one workgroup per slice, in four launches:
//   k_max    largest and smallest logit, how many there are
//   k_hist   top-k: how many logits, top-p: how much weight, in each of kBuckets ranges of logits
//            counted from the largest
//   k_pick   the bucket in which the cut falls (top-k: all up to it) goes to a list; what stands
//            before it is added up per slice
//   k_draw   one workgroup per row: the list sorted, the cut, the slice in which the draw falls, the
//            token
// Three of them read the row; what does not fit into the first cache comes from the MALL after the first.
// A row whose list is too long (thousands of equal logits at the cut) is searched digit by digit
// in k_draw instead.
#include "bpdq_paged.h"

namespace bpdq {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;  // k_draw
constexpr int kSliceThreads = 512;
constexpr int kBuckets = 1024;
constexpr int kList = 4096;  // entries of a list that k_draw sorts
constexpr int kTable = 64;

__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);  // -0 becomes +0: they are equal
    const uint32_t k = (u >> 31) ? ~u : u | 0x80000000u;
    return x != x || x == -__builtin_inff() ? 0u : k;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float((key >> 31) ? key & 0x7FFFFFFFu : ~key);
}

// 2^(i / 64), for exp by table and polynomial (Tang 1989): 2^y = 2^e 2^(i/64) e^(r ln 2), y = e + i/64 + r.
__device__ __forceinline__ void fill_table(double* table) {
    if (threadIdx.x < kTable) table[threadIdx.x] = exp2((double)threadIdx.x / kTable);
}

struct Row {
    float top;            // the largest logit
    double per;           // log2(e) / temperature
    int shift;            // weights are multiples of 2^-shift
    float buckets;        // buckets per unit of logit
    const double* table;  // in LDS
    // 2^((x - top) per) up to some units of 2^-52, times 2^up
    __device__ __forceinline__ double weight_real(float x, int up) const {
        if (x == top) return __builtin_ldexp(1.0, up);
        const double y = ((double)x - (double)top) * per;
        if (!(y > -1000.0)) return 0.0;  // also where top is +inf
        const double n = __builtin_rint(y * kTable);
        const double r = __builtin_fma(n, -1.0 / kTable, y) * 0.693147180559945309417;
        double p = __builtin_fma(r, 1.0 / 120, 1.0 / 24);
        p = __builtin_fma(r, p, 1.0 / 6);
        p = __builtin_fma(r, p, 0.5);
        p = __builtin_fma(r, p, 1.0);
        p = __builtin_fma(r, p, 1.0);
        const int k = (int)n;
        return __builtin_ldexp(table[k & (kTable - 1)] * p, (k >> 6) + up);
    }
    __device__ __forceinline__ uint64_t weight(uint32_t key) const {
        // at most 2^44: adding 2^52 rounds to an integer and leaves it in the low bits
        const double v = weight_real(logit_of(key), shift) + 4503599627370496.0;
        return (uint64_t)__double_as_longlong(v) & 0xFFFFFFFFFFFFFull;
    }
    __device__ __forceinline__ bool passes(uint32_t key, float min_p) const {
        return !(min_p > 0.f) || logit_of(key) == top || weight_real(logit_of(key), 0) >= (double)(min_p < 1.f ? min_p : 1.f);
    }
    // Not falling with the distance from the largest logit.
    __device__ __forceinline__ int bucket(uint32_t key) const {
        const float x = logit_of(key), d = (top - x) * buckets;
        return x == top ? 0 : d < (float)(kBuckets - 1) ? (int)d : kBuckets - 1;
    }
};

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// The settings of a row.
struct Set {
    float t, p, m;
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
    return s;
}

enum Mode { kAll, kTopP, kTopK, kGreedy, kNone, kSearch };

// What k_max leaves of a slice, what k_pick leaves of it, and of a row.
struct SliceMax {
    uint32_t top, low, n, at;  // largest key, smallest, how many, first index of the largest
};
struct SliceSum {
    unsigned long long w;  // weights that stay whatever the list says
    uint32_t n, list;      // how many those are, entries of the slice's list
};
struct RowInfo {
    unsigned long long want;  // top-p: weight to be reached within the list
    int mode;
};
struct Work {
    int S, len;  // slices, elements of one
    int shift;
    SliceMax* max;   // [row][S]
    SliceSum* sum;   // [row][S]
    RowInfo* info;   // [row]
    unsigned long long* weight;  // [row][S][kBuckets], or in the same place
    uint32_t* count;             // [row][S][2 kBuckets], the first half used
    uint16_t* list;              // [row][S][len]: indices within the slice
};

// Key and index of each element of [lo, hi) of a row, 16 bytes at a time and thread.
template <typename X, int THREADS, typename F>
__device__ __forceinline__ void each(const X* __restrict__ x, int lo, int hi, F&& f) {
    constexpr int N = 16 / (int)sizeof(X);
    const bool aligned = ((uintptr_t)(x + lo) & 15) == 0;
    for (int i = lo + (int)threadIdx.x * N; i < hi; i += THREADS * N) {
        Vec<X, N> v;
        const int m = min(N, hi - i);
        if (aligned && m == N) {
            v = *reinterpret_cast<const Vec<X, N>*>(x + i);
#pragma unroll
            for (int j = 0; j < N; j++) f(i + j, key_of((float)v.v[j]));
        } else {
            for (int j = 0; j < m; j++) f(i + j, key_of((float)x[i + j]));
        }
    }
}

template <int TYPE>
__global__ __launch_bounds__(kSliceThreads) void k_max(SampleArgs g, Work w) {
    using X = typename Elem<TYPE>::type;
    __shared__ SliceMax part[kSliceThreads / 64];
    const int row = (int)(blockIdx.x / (unsigned)w.S), slice = (int)(blockIdx.x % (unsigned)w.S), tid = (int)threadIdx.x;
    const int lo = slice * w.len, hi = min(g.V, lo + w.len);
    SliceMax s = {0u, 0xFFFFFFFFu, 0u, 0xFFFFFFFFu};
    each<X, kSliceThreads>(reinterpret_cast<const X*>(g.logits) + (int64_t)row * g.stride, lo, hi, [&](int i, uint32_t k) {
        if (k > s.top) s.top = k, s.at = (uint32_t)i;
        s.low = min(s.low, k - 1u);  // 0 is no logit: it wraps to the largest
        s.n += k != 0;
    });
    auto join = [](SliceMax& a, uint32_t top, uint32_t low, uint32_t n, uint32_t at) {
        if (top > a.top || (top == a.top && at < a.at)) a.top = top, a.at = at;
        a.low = min(a.low, low);
        a.n += n;
    };
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t t = __shfl_xor(s.top, d), l = __shfl_xor(s.low, d), n = __shfl_xor(s.n, d), at = __shfl_xor(s.at, d);
        join(s, t, l, n, at);
    }
    if ((tid & 63) == 0) part[tid >> 6] = s;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < kSliceThreads / 64; i++) join(s, part[i].top, part[i].low, part[i].n, part[i].at);
        w.max[(int64_t)row * w.S + slice] = s;
    }
}

// The row's largest and smallest logit and number from its slices, in every wave.
__device__ __forceinline__ SliceMax row_max(const Work& w, int row) {
    SliceMax s = {0u, 0xFFFFFFFFu, 0u, 0xFFFFFFFFu};
    for (int i = (int)threadIdx.x & 63; i < w.S; i += 64) {
        const SliceMax o = w.max[(int64_t)row * w.S + i];
        if (o.top > s.top || (o.top == s.top && o.at < s.at)) s.top = o.top, s.at = o.at;
        s.low = min(s.low, o.low);
        s.n += o.n;
    }
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t t = __shfl_xor(s.top, d), at = __shfl_xor(s.at, d);
        if (t > s.top || (t == s.top && at < s.at)) s.top = t, s.at = at;
        s.low = min(s.low, (uint32_t)__shfl_xor(s.low, d));
        s.n += __shfl_xor(s.n, d);
    }
    return s;
}

__device__ __forceinline__ Row row_of(const Set& set, const SliceMax& m, int shift, const double* table) {
    Row r;
    r.top = logit_of(m.top);
    r.per = 1.4426950408889634074 / (double)set.t;
    r.shift = shift;
    r.table = table;
    // 32 to a unit of (l - max) / t, which weighs nothing beyond kBuckets of them; fewer logits' range is cut
    // finer
    r.buckets = fmaxf(32.f / set.t, 0.999f * (float)kBuckets / (r.top - logit_of(m.low + 1u)));
    return r;
}

__device__ __forceinline__ Mode mode_of(const Set& s, const SliceMax& m) {
    if (m.n == 0) return kNone;
    if (s.greedy) return kGreedy;
    if (s.k > 0 && (uint32_t)s.k < m.n) return s.k > kList ? kSearch : kTopK;
    return s.p < 1.f ? kTopP : kAll;
}

template <int TYPE>
__global__ __launch_bounds__(kSliceThreads) void k_hist(SampleArgs g, Work w) {
    using X = typename Elem<TYPE>::type;
    __shared__ double table[kTable];
    __shared__ unsigned long long hw[kBuckets];
    uint32_t* hc = reinterpret_cast<uint32_t*>(hw);
    const int row = (int)(blockIdx.x / (unsigned)w.S), slice = (int)(blockIdx.x % (unsigned)w.S), tid = (int)threadIdx.x;
    const Set set = settings(g, row);
    const SliceMax m = row_max(w, row);
    const Mode mode = mode_of(set, m);
    if (mode != kTopP && mode != kTopK) return;
    fill_table(table);
    for (int i = tid; i < kBuckets; i += kSliceThreads) hw[i] = 0;
    __syncthreads();
    const Row r = row_of(set, m, w.shift, table);
    const int lo = slice * w.len, hi = min(g.V, lo + w.len);
    const X* x = reinterpret_cast<const X*>(g.logits) + (int64_t)row * g.stride;
    const int64_t at = ((int64_t)row * w.S + slice) * kBuckets;
    if (mode == kTopK) {
        // the last bucket's are what the others leave, and not asked for
        each<X, kSliceThreads>(x, lo, hi, [&](int, uint32_t k) {
            const int b = r.bucket(k);
            if (k != 0 && b < kBuckets - 1) atomicAdd(&hc[b], 1u);
        });
        __syncthreads();
        for (int i = tid; i < kBuckets; i += kSliceThreads) w.count[2 * at + i] = hc[i];
    } else {
        unsigned long long rest = 0;  // the last bucket's, by thread
        each<X, kSliceThreads>(x, lo, hi, [&](int, uint32_t k) {
            if (k == 0) return;
            const int b = r.bucket(k);
            const unsigned long long v = r.weight(k);
            if (b == kBuckets - 1) rest += v;
            else if (v != 0) atomicAdd(&hw[b], v);
        });
        rest = wave_sum(rest);
        if ((tid & 63) == 0 && rest != 0) atomicAdd(&hw[kBuckets - 1], rest);
        __syncthreads();
        for (int i = tid; i < kBuckets; i += kSliceThreads) w.weight[at + i] = hw[i];
    }
}

// Sums of a row's histogram over its slices and the first bucket at which they reach `need`, with the sum
// before it; kBuckets - 1 if none before does.
template <typename T>
struct Cut {
    T before, total;
    int bucket;
};
template <typename T, typename NEED>
__device__ __forceinline__ Cut<T> find_bucket(const T* hist, int stride, int S, NEED&& need_of, T* s_part, Cut<T>* s_cut) {
    constexpr int PER = kBuckets / kSliceThreads, W = kSliceThreads / 64;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    T v[PER], mine = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) v[j] = 0;
    for (int s = 0; s < S; s++)
#pragma unroll
        for (int j = 0; j < PER; j++) v[j] += hist[(int64_t)s * stride + tid * PER + j];
#pragma unroll
    for (int j = 0; j < PER; j++) mine += v[j];
    T run = mine;
    for (int d = 1; d < 64; d <<= 1) {
        const T o = __shfl_up(run, d);
        if (lane >= d) run += o;
    }
    if (lane == 63) s_part[wave] = run;
    __syncthreads();
    T before = run - mine, total = 0;
    for (int i = 0; i < W; i++) {
        if (i < wave) before += s_part[i];
        total += s_part[i];
    }
    const T need = need_of(total);
    if (tid == kSliceThreads - 1) {
        s_cut->bucket = kBuckets - 1;
        s_cut->before = total - v[PER - 1];
        s_cut->total = total;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; j++) {
        if (before < need && before + v[j] >= need) {  // one thread's one bucket
            s_cut->bucket = tid * PER + j;
            s_cut->before = before;
        }
        before += v[j];
    }
    __syncthreads();
    return *s_cut;
}

// Weight that top-p has to reach of a total.
__device__ __forceinline__ unsigned long long reach(float p, unsigned long long total) {
    const double need = __builtin_ceil((double)(p > 0.f ? p : 0.f) * (double)total);
    const unsigned long long want = need >= (double)total ? total : (unsigned long long)need;
    return want == 0 ? 1 : want;
}

template <int TYPE>
__global__ __launch_bounds__(kSliceThreads) void k_pick(SampleArgs g, Work w) {
    using X = typename Elem<TYPE>::type;
    constexpr int W = kSliceThreads / 64;
    __shared__ double table[kTable];
    __shared__ unsigned long long s_part[W];
    __shared__ Cut<unsigned long long> s_cut;
    __shared__ Cut<uint32_t> s_cutn;
    __shared__ uint32_t s_n[W], s_list;
    const int row = (int)(blockIdx.x / (unsigned)w.S), slice = (int)(blockIdx.x % (unsigned)w.S), tid = (int)threadIdx.x;
    const Set set = settings(g, row);
    const SliceMax m = row_max(w, row);
    Mode mode = mode_of(set, m);
    fill_table(table);
    if (tid == 0) s_list = 0;
    __syncthreads();
    const Row r = row_of(set, m, w.shift, table);
    int first = 0, last = -1;  // buckets [0, first) stay, [first, last] are listed
    RowInfo info = {0, mode};
    if (mode == kTopP) {
        const auto c = find_bucket<unsigned long long>(
            w.weight + (int64_t)row * w.S * kBuckets, kBuckets, w.S, [&](unsigned long long total) { return reach(set.p, total); },
            s_part, &s_cut);
        first = last = c.bucket;
        info.want = reach(set.p, c.total) - c.before;
    } else if (mode == kTopK) {
        const auto c = find_bucket<uint32_t>(w.count + (int64_t)row * w.S * 2 * kBuckets, 2 * kBuckets, w.S,
                                             [&](uint32_t) { return (uint32_t)set.k; }, reinterpret_cast<uint32_t*>(s_part),
                                             &s_cutn);
        first = 0;
        last = c.bucket;
    } else if (mode == kAll) {
        first = kBuckets;
    }
    if (slice == 0 && tid == 0) w.info[row] = info;
    if (mode == kGreedy || mode == kNone || mode == kSearch) return;
    const int lo = slice * w.len, hi = min(g.V, lo + w.len);
    uint16_t* list = w.list + ((int64_t)row * w.S + slice) * w.len;
    unsigned long long sum = 0;
    uint32_t n = 0;
    each<X, kSliceThreads>(reinterpret_cast<const X*>(g.logits) + (int64_t)row * g.stride, lo, hi, [&](int i, uint32_t k) {
        if (k == 0) return;
        const int b = r.bucket(k);
        if (b < first) {
            if (r.passes(k, set.m)) {
                sum += r.weight(k);
                n++;
            }
        } else if (b <= last) {
            list[atomicAdd(&s_list, 1u)] = (uint16_t)(i - lo);
        }
    });
    sum = wave_sum(sum);
    n = wave_sum(n);
    __syncthreads();
    if ((tid & 63) == 0) s_part[tid >> 6] = sum, s_n[tid >> 6] = n;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < W; i++) sum += s_part[i], n += s_n[i];
        w.sum[(int64_t)row * w.S + slice] = {sum, n, s_list};
    }
}

__device__ __forceinline__ void answer(const SampleArgs& g, int row, int token, float logprob, uint32_t kept) {
    g.token[row] = token;
    if (g.logprob != nullptr) g.logprob[row] = logprob;
    if (g.kept != nullptr) g.kept[row] = (int32_t)kept;
}

// Weight that the cumulated sum has to exceed.
__device__ __forceinline__ unsigned long long draw_target(float u, unsigned long long total) {
    const double at = (u > 0.f ? (u < 1.f ? (double)u : 1.0) : 0.0) * (double)total;
    return at >= (double)total ? total - 1 : (unsigned long long)at;
}

// The row digit by digit, a pass for every question, by one workgroup.  The cut is a key and how many that
// equal it, from the first index on, stay.
struct SearchLds {
    uint32_t hc[256];
    unsigned long long hw[256];
    unsigned long long part[kWaves];
    uint32_t ties[kWaves];
    uint32_t key, cnt;
    unsigned long long w;
};
template <int TYPE>
__device__ void search_row(const SampleArgs& g, const Row& r, const Set& set, uint32_t n, int row, SearchLds& s) {
    using X = typename Elem<TYPE>::type;
    auto& hc = s.hc;
    auto& ties = s.ties;
    auto& hw = s.hw;
    auto& part = s.part;
    auto &s_key = s.key, &s_cnt = s.cnt;
    auto& s_w = s.w;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const X* x = reinterpret_cast<const X*>(g.logits) + (int64_t)row * g.stride;
    const int V = g.V;
    auto key_at = [&](int i) { return key_of((float)x[i]); };
    const int kk = set.k;
    const float pf = set.p, mf = set.m;
    uint32_t cut = 1, tie = 0xFFFFFFFFu, kept = n;  // all keys above 0
    // The cut at which count (by_weight: weight) of keys from the largest down first reaches `need`.
    auto select = [&](bool by_weight, unsigned long long need, uint32_t& above, unsigned long long& wabove) {
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
                if (by_weight) atomicAdd(&hw[(k >> bit) & 255], (unsigned long long)r.weight(k));
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
                    const unsigned long long have = by_weight ? wabove + hw[d] : (unsigned long long)above + hc[d];
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
            unsigned long long w;
            cut = select(false, (unsigned long long)kk, above, w);
            tie = (uint32_t)kk - above;
            kept = (uint32_t)kk;
        }
        if (pf < 1.f) {
            const uint32_t more = tie == 0xFFFFFFFFu ? 0 : count_ties(cut) - tie;  // ties that top_k left out
            if (tid == 0) s_cnt = more, s_w = more * r.weight(cut);
            __syncthreads();
            unsigned long long total = 0;
            for (int i = tid; i < V; i += kThreads) {
                const uint32_t k = key_at(i);
                if (k >= cut) total += r.weight(k);
            }
            total = wave_sum(total);
            if (lane == 0) part[wave] = total;
            __syncthreads();
            total = 0;
            for (int w = 0; w < kWaves; w++) total += part[w];
            total -= s_w;
            __syncthreads();
            const unsigned long long want = reach(pf, total);
            uint32_t above;
            unsigned long long wabove;
            const uint32_t key = select(true, want, above, wabove);
            const uint64_t each = r.weight(key);
            const uint32_t num = each == 0 ? 1 : (uint32_t)((want - wabove + each - 1) / each);
            cut = key;
            tie = num;
            kept = above + num;
        }
        if (mf > 0.f) {  // weights fall with the key: the cut moves up to the last key at or above min_p
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
    const uint64_t wc = r.weight(cut);
    unsigned long long w = 0;
    uint32_t tc = 0;
    for (int i = lo + lane; i < hi; i += 64) {
        const uint32_t k = key_at(i);
        if (k > cut) w += r.weight(k);
        tc += k == cut;
    }
    w = wave_sum(w);
    tc = wave_sum(tc);
    __syncthreads();
    if (lane == 0) part[wave] = w, ties[wave] = tc;
    __syncthreads();
    unsigned long long total = 0, before = 0;
    uint32_t tb = 0;
    for (int i = 0; i < kWaves; i++) {
        const uint32_t took = min(ties[i], tie > tb ? tie - tb : 0u);
        total += part[i] + took * wc;
        tb += ties[i];
    }
    const unsigned long long target = draw_target(g.u[row], total);  // chosen: sum > target
    tb = 0;
    int chosen = 0;
    uint32_t left = 0;
    for (int i = 0; i < kWaves; i++) {
        left = tie > tb ? tie - tb : 0u;
        const unsigned long long mine = part[i] + min(ties[i], left) * wc;
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
        const unsigned long long mine = in ? r.weight(k) : 0;
        unsigned long long run = mine;
        for (int d = 1; d < 64; d <<= 1) {
            const unsigned long long o = __shfl_up(run, d);
            if (lane >= d) run += o;
        }
        const uint64_t over = __ballot(before + run > target);
        if (over != 0) {
            if (lane == __ffsll((unsigned long long)over) - 1) {
                answer(g, row, i, (float)log((double)mine / (double)total), kept);
            }
            return;
        }
        before += __shfl(run, 63);
        const uint32_t used = (uint32_t)__popcll(same);
        left = left > used ? left - used : 0u;
    }
}

// Sorts n (a power of two) values of LDS, falling.
__device__ __forceinline__ void sort_falling(unsigned long long* a, int n) {
    for (int k = 2; k <= n; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int i = (int)threadIdx.x; i < n / 2; i += kThreads) {
                const int x = 2 * i - (i & (j - 1)), y = x + j;  // x has bit j clear
                const unsigned long long p = a[x], q = a[y];
                if ((p < q) == ((x & k) == 0)) a[x] = q, a[y] = p;
            }
            __syncthreads();
        }
}

// Exclusive sum over the workgroup, the total in `all`.
__device__ __forceinline__ unsigned long long scan_block(unsigned long long v, unsigned long long& all,
                                                         unsigned long long* s_part) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    unsigned long long run = v;
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned long long o = __shfl_up(run, d);
        if (lane >= d) run += o;
    }
    __syncthreads();
    if (lane == 63) s_part[wave] = run;
    __syncthreads();
    unsigned long long before = run - v;
    all = 0;
    for (int i = 0; i < kWaves; i++) {
        if (i < wave) before += s_part[i];
        all += s_part[i];
    }
    return before;
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void k_draw(SampleArgs g, Work w) {
    using X = typename Elem<TYPE>::type;
    __shared__ double table[kTable];
    __shared__ unsigned long long list[kList];  // (key, ~index), later (~index, place)
    __shared__ unsigned long long s_part[kWaves];
    __shared__ unsigned long long s_before;
    __shared__ uint32_t s_n, s_kept;
    __shared__ int s_slice;
    __shared__ SearchLds search;
    const int row = (int)blockIdx.x, tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Set set = settings(g, row);
    const SliceMax m = row_max(w, row);
    const X* x = reinterpret_cast<const X*>(g.logits) + (int64_t)row * g.stride;
    if (m.n == 0 || set.greedy) {
        if (tid == 0) m.n == 0 ? answer(g, row, -1, __builtin_nanf(""), 0) : answer(g, row, (int)m.at, 0.f, 1);
        return;
    }
    fill_table(table);
    if (tid == 0) s_n = 0, s_kept = 0, s_before = 0, s_slice = -1;
    const Row r = row_of(set, m, w.shift, table);
    const RowInfo info = w.info[row];
    const SliceSum* sums = w.sum + (int64_t)row * w.S;
    __syncthreads();
    // the list
    uint32_t n_list = 0, n_stay = 0;
    if (info.mode != kSearch) {
        for (int s = lane; s < w.S; s += 64) n_list += sums[s].list, n_stay += sums[s].n;
        n_list = wave_sum(n_list);
        n_stay = wave_sum(n_stay);
    }
    if (info.mode == kSearch || n_list > (uint32_t)kList) {
        search_row<TYPE>(g, r, set, m.n, row, search);
        return;
    }
    for (int s = wave; s < w.S; s += kWaves) {
        const uint32_t n = sums[s].list;
        const uint16_t* from = w.list + ((int64_t)row * w.S + s) * w.len;
        uint32_t at = 0;
        if (lane == 0 && n > 0) at = atomicAdd(&s_n, n);
        at = __shfl(at, 0);
        for (uint32_t i = lane; i < n; i += 64) {
            const uint32_t idx = (uint32_t)(s * w.len) + from[i];
            list[at + i] = (unsigned long long)key_of((float)x[idx]) << 32 | (uint32_t)~idx;
        }
    }
    int n2 = 1;
    while (n2 < (int)n_list) n2 <<= 1;
    __syncthreads();
    for (int i = (int)n_list + tid; i < n2; i += kThreads) list[i] = 0;
    __syncthreads();
    sort_falling(list, n2);  // by logit, equal ones by index
    // how many of the list stay: top-k, top-p, min-p
    constexpr int PER = kList / kThreads;
    unsigned long long v[PER], mine = 0, total_list;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int i = tid * PER + j;
        v[j] = i < (int)n_list && (info.mode != kTopK || i < set.k) ? r.weight((uint32_t)(list[i] >> 32)) : 0;
        mine += v[j];
    }
    unsigned long long run = scan_block(mine, total_list, s_part);
    unsigned long long want = info.want;
    if (info.mode == kTopK) want = set.p < 1.f ? reach(set.p, total_list) : total_list + 1;
    uint32_t stay = 0;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int i = tid * PER + j;
        // what stands before it falls short of what is wanted
        if (i < (int)n_list && (info.mode != kTopK || i < set.k) && run < want && r.passes((uint32_t)(list[i] >> 32), set.m))
            stay++;
        run += v[j];
    }
    stay = wave_sum(stay);
    if (lane == 0 && stay) atomicAdd(&s_kept, stay);
    __syncthreads();
    const uint32_t kept_list = s_kept, kept = kept_list + n_stay;
    // a head of the list stays, up to this one; where none does, min-p alone decides
    const uint64_t cut = kept_list > 0 ? list[kept_list - 1] : 0;

    if (info.mode == kTopK) {
        // all that stays is in the list: in the order of the vocabulary, the draw
        __syncthreads();
        n2 = 1;
        while (n2 < (int)kept_list) n2 <<= 1;
        for (int i = tid; i < n2; i += kThreads) {
            const unsigned long long e = i < (int)kept_list ? list[i] : 0;
            list[i] = e << 32 | e >> 32;
        }
        __syncthreads();
        sort_falling(list, n2);  // ~index falling
        mine = 0;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int i = tid * PER + j;
            v[j] = i < (int)kept_list ? r.weight((uint32_t)list[i]) : 0;
            mine += v[j];
        }
        unsigned long long total;
        run = scan_block(mine, total, s_part);
        const unsigned long long target = draw_target(g.u[row], total);
#pragma unroll
        for (int j = 0; j < PER; j++) {
            if (run <= target && run + v[j] > target)
                answer(g, row, (int)~(uint32_t)(list[tid * PER + j] >> 32), (float)log((double)v[j] / (double)total), kept);
            run += v[j];
        }
        return;
    }
    // the slice: what stays of each is its sum and its part of the list
    unsigned long long* slice_w = search.hw;  // 256 at most at a time
    unsigned long long total = 0;
    for (int pass = 0; pass < 2; pass++) {  // the total, then the slice
        unsigned long long before = 0;
        const unsigned long long target = pass == 0 ? 0 : draw_target(g.u[row], total);
        for (int s0 = 0; s0 < w.S; s0 += 256) {
            __syncthreads();
            if (tid < 256) slice_w[tid] = s0 + tid < w.S ? sums[s0 + tid].w : 0;
            __syncthreads();
            for (int i = tid; i < (int)kept_list; i += kThreads) {
                const int s = (int)(~(uint32_t)list[i]) / w.len - s0;
                if (s >= 0 && s < 256) atomicAdd(&slice_w[s], (unsigned long long)r.weight((uint32_t)(list[i] >> 32)));
            }
            __syncthreads();
            const unsigned long long ws = tid < 256 ? slice_w[tid] : 0;
            unsigned long long all;
            const unsigned long long at = before + scan_block(ws, all, s_part);
            if (pass == 1 && at <= target && at + ws > target) {
                s_slice = s0 + tid;
                s_before = at;
            }
            before += all;
        }
        total = before;
    }
    __syncthreads();
    // the place in the slice: wave by wave, then step by step
    const unsigned long long target = draw_target(g.u[row], total);
    const int lo = s_slice * w.len, hi = min(g.V, lo + w.len), seg = (w.len + kWaves - 1) / kWaves;
    const int wlo = min(hi, lo + wave * seg), whi = min(hi, wlo + seg);
    auto weight_at = [&](int i) -> unsigned long long {
        if (i >= whi) return 0;
        const uint32_t k = key_of((float)x[i]);
        return k != 0 && ((uint64_t)k << 32 | (uint32_t)~(uint32_t)i) >= cut && r.passes(k, set.m) ? r.weight(k) : 0;
    };
    mine = 0;
    for (int i = wlo + lane; i < whi; i += 64) mine += weight_at(i);
    mine = wave_sum(mine);
    __syncthreads();
    if (lane == 0) s_part[wave] = mine;
    __syncthreads();
    unsigned long long before = s_before;
    int chosen = 0;
    for (; chosen < kWaves - 1 && before + s_part[chosen] <= target; chosen++) before += s_part[chosen];
    if (wave != chosen) return;
    for (int i0 = wlo; i0 < whi; i0 += 64) {
        const unsigned long long v1 = weight_at(i0 + lane);
        unsigned long long sum = v1;
        for (int d = 1; d < 64; d <<= 1) {
            const unsigned long long o = __shfl_up(sum, d);
            if (lane >= d) sum += o;
        }
        const uint64_t over = __ballot(before + sum > target);
        if (over != 0) {
            if (lane == __builtin_ctzll(over)) answer(g, row, i0 + lane, (float)log((double)v1 / (double)total), kept);
            return;
        }
        before += __shfl(sum, 63);
    }
}

int shift_of(int V) {
    int bits = 0;
    while (((int64_t)1 << bits) < V) bits++;
    return bits <= 18 ? 44 : 62 - bits;
}

// Elements of a slice: enough workgroups for the chip, up to 16384 (16-bit places in a slice's list).
int slice_len(int B, int V) {
    int len = 16384;
    while (len > 2048 && (int64_t)B * ((V + len - 1) / len) < 1024) len >>= 1;
    return len;
}

int64_t up16(int64_t v) { return (v + 15) / 16 * 16; }

struct Layout {
    int64_t max, sum, info, weight, list, total;
    int S, len;
};
Layout layout(int B, int V) {
    Layout l;
    l.len = slice_len(B, V);
    l.S = V > 0 ? (V + l.len - 1) / l.len : 0;
    const int64_t n = (int64_t)B * l.S;
    l.max = 0;
    l.sum = l.max + up16(n * (int64_t)sizeof(SliceMax));
    l.info = l.sum + up16(n * (int64_t)sizeof(SliceSum));
    l.weight = l.info + up16(B * (int64_t)sizeof(RowInfo));
    l.list = l.weight + n * kBuckets * 8;
    l.total = l.list + up16(n * l.len * 2) + 16;
    return l;
}

template <int TYPE>
void launch_type(const SampleArgs& a, const Work& w, hipStream_t s) {
    const dim3 grid((unsigned)w.S * (unsigned)a.B), block(kSliceThreads);
    if (w.S > 0) {
        hipLaunchKernelGGL(k_max<TYPE>, grid, block, 0, s, a, w);
        if (a.top_p != nullptr || a.top_k != nullptr) hipLaunchKernelGGL(k_hist<TYPE>, grid, block, 0, s, a, w);
        hipLaunchKernelGGL(k_pick<TYPE>, grid, block, 0, s, a, w);
    }
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
    w.max = reinterpret_cast<SliceMax*>(p + l.max);
    w.sum = reinterpret_cast<SliceSum*>(p + l.sum);
    w.info = reinterpret_cast<RowInfo*>(p + l.info);
    w.count = reinterpret_cast<uint32_t*>(p + l.weight);
    w.weight = reinterpret_cast<unsigned long long*>(p + l.weight);
    w.list = reinterpret_cast<uint16_t*>(p + l.list);
    if (type == BPD_T_F32) launch_type<BPD_T_F32>(a, w, s);
    else if (type == BPD_T_F16) launch_type<BPD_T_F16>(a, w, s);
    else launch_type<BPD_T_BF16>(a, w, s);
}

}  // namespace bpdq
