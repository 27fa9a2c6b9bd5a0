// pages.hip — bpd_pages_extend_gpu and bpd_pages_release_gpu: pages handed to sequences that grow, and taken back.
//
// One workgroup decides for all sequences, 1024 at a time, a thread each: running sums of the pages and
// tokens that they ask for say who is served and from which place of the free stack.  Then a workgroup for each part of a
// sequence writes its table, its new tokens' slots and positions, or puts pages back onto the stack.
#include "bpdq_paged.h"

namespace bpdq {

namespace {

constexpr int N = 1024;

// The sum of v over the threads before this one, and over all.
struct Sums {
    int64_t before, all;
};
struct Scan {
    int64_t wave[N / 64];
    __device__ __forceinline__ Sums go(int64_t v) {
        const int lane = (int)threadIdx.x & 63, w = (int)threadIdx.x >> 6;
        int64_t x = v;
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t o = __shfl_up(x, d);
            if (lane >= d) x += o;
        }
        __syncthreads();
        if (lane == 63) wave[w] = x;
        __syncthreads();
        Sums r = {x - v, 0};
        for (int i = 0; i < N / 64; i++) {
            if (i < w) r.before += wave[i];
            r.all += wave[i];
        }
        return r;
    }
};

__device__ __forceinline__ int clamp(int v, int lo, int hi) { return max(lo, min(v, hi)); }
__device__ __forceinline__ int pages_of(const PoolArgs& g, int rows) {  // rows up to 2^31 - 1
    return rows == 0 ? 0 : fdiv(g.page, rows - 1) + 1;
}

// The row that sequence b names, or -1: none, or one that an earlier sequence names.
__device__ __forceinline__ int row_of(const PoolArgs& g, const int* claim, int b) {
    if (g.rows == nullptr) return b < g.n_rows ? b : -1;
    const int r = g.rows[b];
    return r >= 0 && r < g.n_rows && claim[r] == b ? r : -1;
}
__device__ __forceinline__ void claim_rows(const PoolArgs& g, int* claim) {
    if (g.rows == nullptr) return;
    for (int i = (int)threadIdx.x; i < g.n_rows; i += N) claim[i] = g.B;
    __syncthreads();
    for (int b = (int)threadIdx.x; b < g.B; b += N) {
        const int r = g.rows[b];
        if (r >= 0 && r < g.n_rows) atomicMin(&claim[r], b);
    }
    __syncthreads();
}

__global__ __launch_bounds__(N) void k_extend_plan(PoolArgs g) {
    extern __shared__ int claim[];
    __shared__ Scan s;
    const int most = g.W * (int)g.page.d;  // rows of a table
    const int n_free = clamp(g.n_free[0], 0, g.n_pages);
    claim_rows(g, claim);
    int64_t asked = 0, wanted = 0;  // pages by all before, tokens by those of them who can be paid
    int tokens = 0, pages = 0;      // granted to those before
    for (int b0 = 0; b0 < g.B; b0 += N) {
        const int b = b0 + (int)threadIdx.x;
        int row = -1, old = 0, add = 0, code = 1;
        if (b < g.B) {
            row = row_of(g, claim, b);
            add = g.add[b];
            if (row >= 0) old = clamp(g.lens[row], 0, most);
            if (row >= 0 && add >= 0) code = (int64_t)old + add <= most ? 0 : 2;
        }
        const int need = code == 0 ? pages_of(g, old + add) - pages_of(g, old) : 0;
        const Sums p = s.go(need);
        if (code == 0 && need > 0 && asked + p.before + need > n_free) code = 3;
        asked += p.all;
        const Sums t = s.go(code == 0 ? add : 0);
        if (code == 0 && wanted + t.before + add > g.T) code = 4;
        wanted += t.all;
        const bool ok = code == 0;
        const Sums q = s.go(ok ? add : 0), u = s.go(ok ? need : 0);
        if (b < g.B) {
            g.plan[b] = make_int4(row, old, ok ? add : 0, pages + (int)u.before);
            g.q_start[b] = tokens + (int)q.before;
            g.lens_out[b] = ok ? old + add : old;
            g.refused[b] = code;
            if (ok) g.lens[row] = old + add;
        }
        tokens += (int)q.all;
        pages += (int)u.all;
    }
    if (threadIdx.x == 0) {
        g.q_start[g.B] = tokens;
        g.plan[g.B] = make_int4(n_free, tokens, 0, 0);
        g.n_free[0] = n_free - pages;
    }
}

// Part blockIdx.x % parts of a sequence's table and new tokens; the workgroups of the last sequence take the tokens
// behind all too.
__global__ __launch_bounds__(256) void k_extend_fill(PoolArgs g) {
    const int b = (int)(blockIdx.x / (unsigned)g.parts), part = (int)blockIdx.x - b * g.parts;
    const int step = 256 * g.parts, first = part * 256 + (int)threadIdx.x;
    const int4 p = g.plan[b];
    const int n_free = g.plan[g.B].x, tokens = g.plan[g.B].y;
    const int row = p.x, old = p.y, add = p.z;
    const int had = pages_of(g, old), has = pages_of(g, old + add);
    int32_t* table = row >= 0 ? g.table + (int64_t)row * g.table_stride : nullptr;
    auto entry = [&](int i) { return i < had ? table[i] : g.free_pages[n_free - 1 - p.w - (i - had)]; };
    if (g.table_out != nullptr) {
        int32_t* out = g.table_out + (int64_t)b * g.table_out_stride;
        for (int i = first; i < g.W; i += step) out[i] = row >= 0 && i < has ? entry(i) : -1;
    }
    for (int i = had + first; i < has; i += step) table[i] = entry(i);
    const int t0 = g.q_start[b];
    for (int i = first; i < add; i += step) {
        const int index = old + i, pg = fdiv(g.page, index), in = index - pg * (int)g.page.d, page = entry(pg);
        g.slots[t0 + i] = page >= 0 && page < g.n_pages ? page * (int)g.page.d + in : -1;
        g.pos[t0 + i] = g.prefix_len + index;
    }
    if (b == g.B - 1)
        for (int i = tokens + first; i < g.T; i += step) g.slots[i] = g.pos[i] = -1;
}

// Of a sequence with `old` rows: those it keeps, and which pages it gives back.
struct Release {
    int old, keep;       // rows before and after
    int k0, k1;          // pages [k0, k1) slide out of the window; gone [g0, g1) before, [n0, n1) after
    int n0, n1;
    int used, kept;      // pages before and after
    int g0, g1;
};
__device__ __forceinline__ Release release_of(const PoolArgs& g, int b, int row) {
    Release r = {};
    if (row < 0) return r;
    const int most = g.W * (int)g.page.d;
    r.old = clamp(g.lens[row], 0, most);
    r.keep = g.keep != nullptr ? clamp(g.keep[b], 0, r.old) : r.old;
    r.used = pages_of(g, r.old);
    r.kept = pages_of(g, r.keep);
    if (g.gone != nullptr) {
        r.g0 = clamp(g.gone[2 * row], 0, r.used);
        r.g1 = clamp(g.gone[2 * row + 1], r.g0, r.used);
    }
    r.n0 = min(r.g0, r.kept);
    r.n1 = min(r.g1, r.kept);
    if (r.n0 == r.n1) r.n0 = r.n1 = 0;
    if (g.window > 0 && g.gone != nullptr) {
        // the next token stands at row `keep` and sees the rows from keep - window + 1 on
        const int low = r.keep - g.window + 1;
        const int k1 = low > 0 ? fdiv(g.page, low) : 0, k0 = pages_of(g, min(g.sinks, most));
        r.k0 = r.n1 > 0 ? r.n1 : k0;
        r.k1 = max(k1, r.k0);
        if (r.k1 > r.k0) {
            if (r.n1 == 0) r.n0 = r.k0;
            r.n1 = r.k1;
        }
    }
    return r;
}
__device__ __forceinline__ int given(const Release& r) {
    // behind the rows kept, but for what had gone before; then what slides out
    const int lo = max(r.kept, r.g0), hi = max(r.kept, r.g1);
    return r.used - r.kept - (hi - lo) + r.k1 - r.k0;
}

__global__ __launch_bounds__(N) void k_release_plan(PoolArgs g) {
    extern __shared__ int claim[];
    __shared__ Scan s;
    claim_rows(g, claim);
    int64_t pages = 0;
    for (int b0 = 0; b0 < g.B; b0 += N) {
        const int b = b0 + (int)threadIdx.x;
        const int row = b < g.B ? row_of(g, claim, b) : -1;
        const Sums p = s.go(given(release_of(g, b, row)));
        if (b < g.B) g.plan[b] = make_int4(row, (int)min(pages + p.before, (int64_t)INT32_MAX), 0, 0);
        pages += p.all;
    }
    if (threadIdx.x == 0) g.plan[g.B] = make_int4((int)min(pages, (int64_t)INT32_MAX), 0, 0, 0);
}

__global__ __launch_bounds__(256) void k_release_fill(PoolArgs g) {
    const int b = (int)(blockIdx.x / (unsigned)g.parts), part = (int)blockIdx.x - b * g.parts;
    const int step = 256 * g.parts, first = part * 256 + (int)threadIdx.x;
    const int4 p = g.plan[b];
    const int row = p.x;
    if (row < 0) return;
    const Release r = release_of(g, b, row);
    const int n_free = clamp(g.n_free[0], 0, g.n_pages), total = g.plan[g.B].x;
    int32_t* table = g.table + (int64_t)row * g.table_stride;
    auto give = [&](int i, int k) {  // page i of the table, the k-th that the sequence gives
        const int64_t at = (int64_t)n_free + total - 1 - p.y - k;
        if (at >= 0 && at < g.n_pages) g.free_pages[at] = table[i];
        table[i] = -1;
    };
    for (int i = r.k0 + first; i < r.k1; i += step) give(i, i - r.k0);
    const int before = r.k1 - r.k0, lo = max(r.kept, r.g0), hi = max(r.kept, r.g1);
    for (int i = r.kept + first; i < r.used; i += step)
        if (i < lo || i >= hi) give(i, before + i - r.kept - (i >= hi ? hi - lo : 0));
}

__global__ __launch_bounds__(N) void k_release_done(PoolArgs g) {
    for (int b = (int)threadIdx.x; b < g.B; b += N) {
        const int row = g.plan[b].x;
        if (row < 0) continue;
        const Release r = release_of(g, b, row);
        g.lens[row] = r.keep;
        if (g.gone != nullptr) {
            g.gone[2 * row] = r.n0;
            g.gone[2 * row + 1] = r.n1;
        }
    }
    if (threadIdx.x == 0)
        g.n_free[0] = (int)min((int64_t)clamp(g.n_free[0], 0, g.n_pages) + g.plan[g.B].x, (int64_t)g.n_pages);
}

int parts_of(int64_t work, int B) {
    int64_t p = work / (2048 * (int64_t)B);  // 8 of a workgroup's rounds
    return (int)(p < 1 ? 1 : p > 64 ? 64 : p);
}

}  // namespace

int64_t pages_ws(int B) { return ((int64_t)B + 1) * (int64_t)sizeof(int4); }

void launch_pages_extend(const PoolArgs& a, hipStream_t s) {
    PoolArgs g = a;
    g.parts = parts_of((int64_t)g.T + (g.table_out != nullptr ? (int64_t)g.B * g.W : 0), g.B);
    const size_t lds = g.rows != nullptr ? 4 * (size_t)g.n_rows : 0;
    hipLaunchKernelGGL(k_extend_plan, dim3(1), dim3(N), lds, s, g);
    hipLaunchKernelGGL(k_extend_fill, dim3((unsigned)g.B * (unsigned)g.parts), dim3(256), 0, s, g);
}

void launch_pages_release(const PoolArgs& a, hipStream_t s) {
    PoolArgs g = a;
    g.parts = parts_of((int64_t)g.B * g.W, g.B);
    const size_t lds = g.rows != nullptr ? 4 * (size_t)g.n_rows : 0;
    hipLaunchKernelGGL(k_release_plan, dim3(1), dim3(N), lds, s, g);
    hipLaunchKernelGGL(k_release_fill, dim3((unsigned)g.B * (unsigned)g.parts), dim3(256), 0, s, g);
    hipLaunchKernelGGL(k_release_done, dim3(1), dim3(N), 0, s, g);
}

}  // namespace bpdq
