// sample.hip — bpd_sample_gpu: one token per row of logits.
//
// A logit's place is its order key: the binary32 bits, sign-folded so that unsigned order is
// the logits' order, 0 for what is never chosen.  All weights are
// W = rint(2^shift exp((l - max) / t)), taken in binary64: their sums are exact in 64 bits,
// so no sum depends on its order.  Every filter keeps a head of the list sorted by
// (logit, index), so it is one cut: a key c and a number r, keeping all keys above c and
// the first r in index order that equal c.
#include "bpdq_paged.h"

namespace bpdq {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;

__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);  // -0 becomes +0: they are equal
    const uint32_t k = (u >> 31) ? ~u : u | 0x80000000u;
    return x != x || x == -__builtin_inff() ? 0u : k;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float((key >> 31) ? key & 0x7FFFFFFFu : ~key);
}

struct Row {
    float top;    // the largest logit
    double t;     // temperature
    double unit;  // 2^shift
    __device__ __forceinline__ uint64_t weight(uint32_t key) const {
        const float x = logit_of(key);
        if (x == top) return (uint64_t)unit;
        const double z = ((double)x - (double)top) / t;
        const double w = exp(z) * unit;
        return w >= 0.5 ? (uint64_t)(int64_t)__builtin_rint(w) : 0;  // also 0 where z is no number (top = +inf)
    }
};

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// The plain form: one workgroup per row, a pass over the row for every question.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void k_sample_row(SampleArgs g, int shift) {
    using X = typename Elem<TYPE>::type;
    __shared__ uint32_t hc[256];
    __shared__ unsigned long long hw[256];
    __shared__ unsigned long long part[kWaves];
    __shared__ uint32_t ties[kWaves];
    __shared__ uint32_t s_key, s_cnt;
    __shared__ unsigned long long s_w;
    const int row = (int)blockIdx.x, tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const X* x = reinterpret_cast<const X*>(g.logits) + (int64_t)row * g.stride;
    const int V = g.V;
    auto key_at = [&](int i) { return key_of((float)x[i]); };
    if (tid == 0) s_key = 0, s_cnt = 0;
    __syncthreads();
    uint32_t mk = 0, n = 0;
    for (int i = tid; i < V; i += kThreads) {
        const uint32_t k = key_at(i);
        mk = max(mk, k);
        n += k != 0;
    }
    for (int d = 1; d < 64; d <<= 1) mk = max(mk, (uint32_t)__shfl_xor(mk, d));
    n = wave_sum(n);
    if (lane == 0) atomicMax(&s_key, mk), atomicAdd(&s_cnt, n);
    __syncthreads();
    mk = s_key;
    n = s_cnt;
    __syncthreads();
    if (mk == 0) {
        if (tid == 0) {
            g.token[row] = -1;
            if (g.logprob != nullptr) g.logprob[row] = __builtin_nanf("");
            if (g.kept != nullptr) g.kept[row] = 0;
        }
        return;
    }
    Row r;
    r.top = logit_of(mk);
    const float tf = g.temperature != nullptr ? g.temperature[row] : 1.f;
    const bool greedy = !(tf > 0.f);
    r.t = greedy ? 1.0 : (double)tf;
    r.unit = (double)(1ull << shift);
    const int kk = g.top_k != nullptr ? g.top_k[row] : 0;
    const float pf = g.top_p != nullptr ? g.top_p[row] : 1.f, mf = g.min_p != nullptr ? g.min_p[row] : 0.f;
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
    if (greedy) {
        cut = mk;
        tie = 1;
        kept = 1;
    } else {
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
            double need = __builtin_ceil((double)(pf > 0.f ? pf : 0.f) * (double)total);
            unsigned long long want = need >= (double)total ? total : (unsigned long long)need;
            if (want == 0) want = 1;
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
            const double least = mf < 1.f ? (double)mf : 1.0;
            auto passes = [&](uint32_t k) {
                const float v = logit_of(k);
                return v == r.top || exp(((double)v - (double)r.top) / r.t) >= least;
            };
            __syncthreads();
            if (tid == 0) s_cnt = 0, s_key = 0xFFFFFFFFu;
            __syncthreads();
            uint32_t c = 0, low = 0xFFFFFFFFu;
            for (int i = tid; i < V; i += kThreads) {
                const uint32_t k = key_at(i);
                if (k < cut || !passes(k)) continue;
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
    const float uf = g.u[row];
    double at = (uf > 0.f ? (uf < 1.f ? (double)uf : 1.0) : 0.0) * (double)total;
    unsigned long long target = at >= (double)total ? total - 1 : (unsigned long long)at;  // chosen: sum > target
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
                g.token[row] = i;
                if (g.logprob != nullptr) g.logprob[row] = (float)log((double)mine / (double)total);
                if (g.kept != nullptr) g.kept[row] = (int32_t)kept;
            }
            return;
        }
        before += __shfl(run, 63);
        const uint32_t used = (uint32_t)__popcll(same);
        left = left > used ? left - used : 0u;
    }
}

int shift_of(int V) {
    int bits = 0;
    while (((int64_t)1 << bits) < V) bits++;
    return bits <= 18 ? 44 : 62 - bits;
}

}  // namespace

int64_t sample_ws(int, int) { return 16; }

void launch_sample(const SampleArgs& a, int type, void*, hipStream_t s) {
    const dim3 grid((unsigned)a.B), block(kThreads);
    const int shift = shift_of(a.V);
    if (type == BPD_T_F32) hipLaunchKernelGGL(k_sample_row<BPD_T_F32>, grid, block, 0, s, a, shift);
    else if (type == BPD_T_F16) hipLaunchKernelGGL(k_sample_row<BPD_T_F16>, grid, block, 0, s, a, shift);
    else hipLaunchKernelGGL(k_sample_row<BPD_T_BF16>, grid, block, 0, s, a, shift);
}

}  // namespace bpdq
