// pages.hip — bpd_pages_extend_gpu and bpd_pages_release_gpu: pages handed to sequences that grow, and taken back.
//
// One launch each.  Every workgroup goes through all sequences, one round of a thread each up to 1,024: running sums of the pages
// and tokens that they ask for say who is served and from which place of the free stack.  That is a few kilobytes out of
// the L2, and spares a launch (or a grid-wide wait) between deciding and doing.  Of each round it then takes its parts: the
// sequences' tables, their new tokens' slots and positions, or the pages that they put back onto the stack.  The
// pool's lengths and counts, which all of them read, are written by the workgroup that is done last.
// Latency bounds both: the names, the lengths, the sums, the table or the stack, the count of workgroups, one after the
// other: 7.8 us for 256 sequences of up to 513 pages that grow by up to 4 rows each, 6.2 us back (a megabyte of tables, 0.2 us
// of memory); 64 prompts of up to 2,048 rows 8.0 and 5.3.  In two and three launches the two calls took 24 us, in one
// with a fence before the count 19, without 15.4, with 128 workgroups 13.6.
#include "bpdq_paged.h"

namespace bpdq {

namespace {

constexpr int kAhead = 4;  // places of a table under way

// A pair of numbers; its sums over the threads before this one, and over all.
struct Two {
    int64_t a, b;
};
struct Sums {
    Two before, all;
};
template <int N>  // threads
struct Scan {
    Two wave[2][N / 64];  // of this sum, and of the one before
    __device__ __forceinline__ Sums go(int64_t a, int64_t b, int& turn) {
        const int lane = (int)threadIdx.x & 63, w = (int)threadIdx.x >> 6;
        Two x = {a, b};
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t oa = __shfl_up(x.a, d), ob = __shfl_up(x.b, d);
            if (lane >= d) {
                x.a += oa;
                x.b += ob;
            }
        }
        if (lane == 63) wave[turn][w] = x;
        __syncthreads();
        Sums r = {{x.a - a, x.b - b}, {0, 0}};
#pragma unroll
        for (int i = 0; i < N / 64; i++) {
            const Two y = wave[turn][i];
            if (i < w) {
                r.before.a += y.a;
                r.before.b += y.b;
            }
            r.all.a += y.a;
            r.all.b += y.b;
        }
        turn ^= 1;  // a thread that is ahead writes the other one: the barrier of its next sum keeps it from this one
        return r;
    }
};

__device__ __forceinline__ int clamp(int v, int lo, int hi) { return max(lo, min(v, hi)); }
__device__ __forceinline__ int pages_of(const PoolArgs& g, int rows) {  // rows up to 2^31 - 1
    return rows == 0 ? 0 : fdiv(g.page, rows - 1) + 1;
}

// Which sequence is the first to name each row; then the row that sequence b names, or -1: none, or one that an earlier
// sequence names.
template <int N>
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
__device__ __forceinline__ int named_row(const PoolArgs& g, int b) {
    const int r = b >= g.B ? -1 : g.rows != nullptr ? g.rows[b] : b;
    return r >= 0 && r < g.n_rows ? r : -1;
}
__device__ __forceinline__ int row_of(const PoolArgs& g, const int* claim, int b) {
    const int r = named_row(g, b);
    return r < 0 || g.rows == nullptr || claim[r] == b ? r : -1;
}

// Whether this workgroup is the last that comes here.  The others' reads of the pool are over, as what they did with them
// stands before their count; nothing that they wrote is read, so no fence is needed.
__device__ __forceinline__ bool last_here(const PoolArgs& g) {
    __shared__ int is_last;
    __syncthreads();
    if (threadIdx.x == 0)
        is_last = __hip_atomic_fetch_add(&g.n_free[1], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
    __syncthreads();
    return is_last != 0;
}

// A sequence as its round has it: the row of the pool, rows before, rows granted, its first token and its first page's
// place among those handed out.
struct Grant {
    int row, old, add, t0, page0;
};

template <int N>
__global__ __launch_bounds__(N) void k_extend(PoolArgs g) {
    extern __shared__ int claim[];
    __shared__ Scan<N> s;
    __shared__ Grant grant[N];
    const int tid = (int)threadIdx.x, most = g.W * (int)g.page.d;  // rows of a table
    const int n_free = clamp(g.n_free[0], 0, g.n_pages);
    claim_rows<N>(g, claim);
    int turn = 0;
    int64_t asked = 0, wanted = 0;  // pages by all before, tokens by those of them who can be paid
    int tokens = 0, pages = 0;      // granted to those before
    // the grants of sequences b0 .. b0 + N - 1; the first workgroup writes what every sequence is told
    auto decide = [&](int b0, bool tell) {
        const int b = b0 + tid, row = row_of(g, claim, b);
        int old = 0, add = 0, code = 1;
        if (b < g.B) add = g.add[b];
        if (row >= 0) {
            old = clamp(g.lens[row], 0, most);
            if (add >= 0) code = (int64_t)old + add <= most ? 0 : 2;
        }
        int need = code == 0 ? pages_of(g, old + add) - pages_of(g, old) : 0;
        if (code != 0) add = 0;
        Sums p = s.go(need, add, turn);
        const bool all = asked + p.all.a <= n_free && wanted + p.all.b <= g.T;
        if (!all) {  // someone has to be refused
            if (code == 0 && need > 0 && asked + p.before.a + need > n_free) code = 3;
            asked += p.all.a;
            const Sums t = s.go(0, code == 0 ? add : 0, turn);
            if (code == 0 && wanted + t.before.b + add > g.T) code = 4;
            wanted += t.all.b;
            if (code != 0) need = add = 0;
            p = s.go(need, add, turn);
        } else {
            asked += p.all.a;
            wanted += p.all.b;
        }
        const int t0 = tokens + (int)p.before.b;
        grant[tid] = {row, old, add, t0, pages + (int)p.before.a};
        if (tell && b < g.B) {
            g.q_start[b] = t0;
            g.lens_out[b] = old + add;
            g.refused[b] = code;
        }
        tokens += (int)p.all.b;
        pages += (int)p.all.a;
        __syncthreads();
    };
    for (int b0 = 0; b0 < g.B; b0 += N) {
        if (b0 > 0) __syncthreads();  // the round before is read
        decide(b0, blockIdx.x == 0);
        const int items = min(N, g.B - b0) * g.parts;
        // items go to the workgroups in turn, from round to round
        const int first = (int)(((int64_t)blockIdx.x - (int64_t)b0 * g.parts % gridDim.x + gridDim.x) % gridDim.x);
        for (int item = first; item < items; item += (int)gridDim.x) {
            const int at = item / g.parts, part = item - at * g.parts, step = N * g.parts, i0 = part * N + tid;
            const Grant x = grant[at];
            const int had = pages_of(g, x.old), has = pages_of(g, x.old + x.add);
            int32_t* table = x.row >= 0 ? g.table + (int64_t)x.row * g.table_stride : nullptr;
            // the counters have 64 bits: a step past the end of the longest tables is beyond 2^31
            auto entry = [&](int i) { return i < had ? table[i] : g.free_pages[n_free - 1 - x.page0 - (i - had)]; };
            if (g.table_out != nullptr) {
                int32_t* out = g.table_out + (int64_t)(b0 + at) * g.table_out_stride;
                for (int64_t i = i0; i < g.W; i += kAhead * step) {
                    int page[kAhead];
#pragma unroll
                    for (int u = 0; u < kAhead; u++) {
                        const int64_t j = i + u * step;
                        page[u] = x.row >= 0 && j < has ? entry((int)j) : -1;
                    }
#pragma unroll
                    for (int u = 0; u < kAhead; u++) {
                        const int64_t j = i + u * step;
                        if (j < g.W) out[j] = page[u];
                        if (x.row >= 0 && j >= had && j < has) table[j] = page[u];
                    }
                }
            } else {
                for (int64_t i = (int64_t)had + i0; i < has; i += step) table[i] = entry((int)i);
            }
            for (int64_t i = i0; i < x.add; i += step) {
                const int index = x.old + (int)i, pg = fdiv(g.page, index), in = index - pg * (int)g.page.d, page = entry(pg);
                g.slots[x.t0 + i] = page >= 0 && page < g.n_pages ? page * (int)g.page.d + in : -1;
                g.pos[x.t0 + i] = g.prefix_len + index;
            }
        }
    }
    for (int64_t i = (int64_t)tokens + blockIdx.x * N + tid; i < g.T; i += gridDim.x * N) g.slots[i] = g.pos[i] = -1;
    const int taken = pages;
    if (blockIdx.x == 0 && tid == 0) g.q_start[g.B] = tokens;
    if (!last_here(g)) return;
    asked = wanted = tokens = pages = 0;
    for (int b0 = 0; b0 < g.B; b0 += N) {
        if (g.B > N) {  // one round's grants are still there
            __syncthreads();
            decide(b0, false);
        }
        const Grant x = grant[tid];
        if (x.row >= 0 && x.add > 0) g.lens[x.row] = x.old + x.add;
    }
    if (tid == 0) {
        g.n_free[0] = n_free - taken;
        g.n_free[1] = 0;
    }
}

// Of a sequence with `old` rows: those it keeps, and which pages it gives back.
struct Release {
    int keep;        // rows after
    int k0, k1;      // pages [k0, k1) slide out of the window
    int n0, n1;      // gone after
    int used, kept;  // pages before and after
    int lo, hi;      // of those behind the rows kept, [lo, hi) had gone before
    __device__ __forceinline__ int pages() const { return used - kept - (hi - lo) + k1 - k0; }
};
__device__ __forceinline__ Release release_of(const PoolArgs& g, int b, int row) {
    Release r = {};
    if (row < 0) return r;
    const int most = g.W * (int)g.page.d, old = clamp(g.lens[row], 0, most);
    r.keep = g.keep != nullptr ? clamp(g.keep[b], 0, old) : old;
    r.used = pages_of(g, old);
    r.kept = pages_of(g, r.keep);
    int g0 = 0, g1 = 0;
    if (g.gone != nullptr) {
        g0 = clamp(g.gone[2 * row], 0, r.used);
        g1 = clamp(g.gone[2 * row + 1], g0, r.used);
    }
    r.lo = max(r.kept, g0);
    r.hi = max(r.kept, g1);
    r.n0 = min(g0, r.kept);
    r.n1 = min(g1, r.kept);
    if (r.n0 == r.n1) r.n0 = r.n1 = 0;
    if (g.window > 0 && g.gone != nullptr) {
        // the next token stands at row `keep` and sees the rows from keep - window + 1 on
        const int low = r.keep - g.window + 1;
        r.k0 = r.n1 > 0 ? r.n1 : pages_of(g, min(g.sinks, most));
        r.k1 = max(low > 0 ? fdiv(g.page, low) : 0, r.k0);
        if (r.k1 > r.k0) {
            if (r.n1 == 0) r.n0 = r.k0;
            r.n1 = r.k1;
        }
    }
    return r;
}

template <int N>
__global__ __launch_bounds__(N) void k_release(PoolArgs g) {
    extern __shared__ int claim[];
    __shared__ Scan<N> s;
    __shared__ Release what[N];
    __shared__ int2 where[N];  // row, pages given before it
    const int tid = (int)threadIdx.x, n_free = clamp(g.n_free[0], 0, g.n_pages);
    claim_rows<N>(g, claim);
    int turn = 0;
    int64_t total = 0, pages = 0;  // given by all, and by those before
    if (g.B > N)                   // one round says both
        for (int b0 = 0; b0 < g.B; b0 += N) {
            const int b = b0 + tid;
            total += s.go(release_of(g, b, row_of(g, claim, b)).pages(), 0, turn).all.a;
        }
    auto decide = [&](int b0) {
        const int b = b0 + tid, row = row_of(g, claim, b);
        what[tid] = release_of(g, b, row);
        const Sums p = s.go(what[tid].pages(), 0, turn);
        where[tid] = make_int2(row, (int)min(pages + p.before.a, (int64_t)INT32_MAX));
        pages += p.all.a;
        if (g.B <= N) total = p.all.a;
        __syncthreads();
    };
    for (int b0 = 0; b0 < g.B; b0 += N) {
        if (b0 > 0) __syncthreads();
        decide(b0);
        const int items = min(N, g.B - b0) * g.parts;
        const int first = (int)(((int64_t)blockIdx.x - (int64_t)b0 * g.parts % gridDim.x + gridDim.x) % gridDim.x);
        for (int item = first; item < items; item += (int)gridDim.x) {
            const int at = item / g.parts, part = item - at * g.parts, step = N * g.parts, i0 = part * N + tid;
            const Release r = what[at];
            if (where[at].x < 0) continue;
            int32_t* table = g.table + (int64_t)where[at].x * g.table_stride;
            const int64_t top = (int64_t)n_free + total - 1 - where[at].y;
            auto give = [&](int64_t i, int64_t k) {  // page i of the table, the k-th that the sequence gives
                if (top - k >= 0 && top - k < g.n_pages) g.free_pages[top - k] = table[i];
                table[i] = -1;
            };
            for (int64_t i = (int64_t)r.k0 + i0; i < r.k1; i += step) give(i, i - r.k0);
            for (int64_t i = (int64_t)r.kept + i0; i < r.used; i += step)
                if (i < r.lo || i >= r.hi) give(i, r.k1 - r.k0 + i - r.kept - (i >= r.hi ? r.hi - r.lo : 0));
        }
    }
    if (!last_here(g)) return;
    for (int b0 = 0; b0 < g.B; b0 += N) {
        const int b = b0 + tid, row = row_of(g, claim, b);
        if (row < 0) continue;
        const Release r = release_of(g, b, row);
        g.lens[row] = r.keep;
        if (g.gone != nullptr) {
            g.gone[2 * row] = r.n0;
            g.gone[2 * row + 1] = r.n1;
        }
    }
    if (tid == 0) {
        g.n_free[0] = (int)min((int64_t)n_free + total, (int64_t)g.n_pages);
        g.n_free[1] = 0;
    }
}

// Threads: a round decides for as many sequences, and each more costs its sums again (300 and 512 sequences, the two calls:
// 18 and 23 us, in rounds of 256 23 and 29).
int threads_of(const PoolArgs& g) { return g.B <= 256 ? 256 : g.B <= 512 ? 512 : 1024; }

// Parts of a sequence's work, 8 of a workgroup's steps each on average, and the workgroups.  Each of them decides, and their
// counts at the end come one after the other: 128, or 256 where there is much to copy (256 / 512 sequences' tables of 513
// pages: 128 13.6 / 17.1 us, 256 15.6 / 18.0, 64 14.4 / 20.0; tables of 8,192: 30.4 / 33.0, 21.8 / 24.7, 50 / 53).
unsigned groups_of(PoolArgs& g, int threads, int64_t work) {
    const int64_t p = work / (8 * (int64_t)threads * g.B);
    const int64_t n = (int64_t)g.B * (g.parts = (int)(p < 1 ? 1 : p > 64 ? 64 : p)), most = work < 5 << 17 ? 128 : 256;
    return (unsigned)(n < most ? n : most);
}

}  // namespace

void launch_pages_extend(const PoolArgs& a, hipStream_t s) {
    PoolArgs g = a;
    const int threads = threads_of(g);
    const unsigned groups = groups_of(g, threads, (int64_t)g.T + (g.table_out != nullptr ? (int64_t)g.B * g.W : 0));
    const size_t lds = g.rows != nullptr ? 4 * (size_t)g.n_rows : 0;
    const auto k = threads == 256 ? k_extend<256> : threads == 512 ? k_extend<512> : k_extend<1024>;
    hipLaunchKernelGGL(k, dim3(groups), dim3(threads), lds, s, g);
}

void launch_pages_release(const PoolArgs& a, hipStream_t s) {
    PoolArgs g = a;
    const int threads = threads_of(g);
    const unsigned groups = groups_of(g, threads, (int64_t)g.B * g.W);
    const size_t lds = g.rows != nullptr ? 4 * (size_t)g.n_rows : 0;
    const auto k = threads == 256 ? k_release<256> : threads == 512 ? k_release<512> : k_release<1024>;
    hipLaunchKernelGGL(k, dim3(groups), dim3(threads), lds, s, g);
}

}  // namespace bpdq
