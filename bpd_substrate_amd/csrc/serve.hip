// serve.hip — the entry points of include/bpdq_serve.h: argument validation,
// workspaces and the launches.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdio>

#include "../../include/bpdq.h"
#include "../../include/bpdq_serve.h"
#include "bpdq_launch.h"
#include "bpdq_paged.h"

namespace {

// 2^31 rows this many elements of 4 bytes apart stay within 63 bits
constexpr int64_t kMaxStride = ((int64_t)1 << 30) - 1;

struct Args {
    const char* fn;
    bool ok = true;
    explicit Args(const char* f) : fn(f) {}
    Args& need(bool good, int code, const char* what) {
        if (ok && !good) {
            bpdq::abi_error(code, fn, what);
            ok = false;
        }
        return *this;
    }
    Args& shape(bool good, const char* what) { return need(good, BPDQ_ERR_SHAPE, what); }
    Args& ptr(const void* p, uintptr_t align, const char* name) {
        char buf[96];
        std::snprintf(buf, sizeof buf, "%s is NULL", name);
        need(p != nullptr, BPDQ_ERR_NULL, buf);
        std::snprintf(buf, sizeof buf, "%s is not %d-byte aligned", name, (int)align);
        return need((reinterpret_cast<uintptr_t>(p) & (align - 1)) == 0, BPDQ_ERR_ALIGN, buf);
    }
    Args& stride(int64_t s, int64_t row, int esize, const char* name) {
        char buf[96];
        std::snprintf(buf, sizeof buf, "%s is shorter than a token's row, or 2^30 or more", name);
        shape(s >= row && s <= kMaxStride, buf);
        std::snprintf(buf, sizeof buf, "%s is no multiple of 16 bytes", name);
        return need(s * esize % 16 == 0, BPDQ_ERR_ALIGN, buf);
    }
};

int esize(int type) { return type == BPD_T_F32 ? 4 : 2; }

// The host side of a cache and a batch.
void check_paged(Args& c, const bpd_paged_cache* kv, const bpd_paged_batch* b) {
    c.need(kv != nullptr, BPDQ_ERR_NULL, "cache is NULL").need(b != nullptr, BPDQ_ERR_NULL, "batch is NULL");
    if (!c.ok) return;
    c.shape(kv->type == BPD_T_F16 || kv->type == BPD_T_BF16, "the cache's type is neither f16 nor bf16");
    c.shape(kv->n_pages >= 0, "n_pages is negative").shape(kv->page_size >= 1, "page_size is below 1");
    c.shape(kv->n_kv_heads >= 1, "n_kv_heads is below 1");
    c.shape(kv->head_dim >= 8 && kv->head_dim <= 256 && kv->head_dim % 8 == 0,
            "head_dim is not a multiple of 8 in 8..256");
    const int64_t top = kMaxStride;
    c.shape(kv->page_stride >= 0 && kv->row_stride >= 0 && kv->head_stride >= 0 && kv->page_stride <= top &&
                kv->row_stride <= top && kv->head_stride <= top, "a cache stride is negative or too large");
    c.need(kv->page_stride % 8 == 0 && kv->row_stride % 8 == 0 && kv->head_stride % 8 == 0, BPDQ_ERR_ALIGN,
           "a cache stride is no multiple of 8 elements");
    if (c.ok && kv->n_pages > 0) c.ptr(kv->k, 16, "cache.k").ptr(kv->v, 16, "cache.v");
    c.shape(b->n_seqs >= 0, "n_seqs is negative").shape(b->n_tokens >= 0, "n_tokens is negative");
    c.shape(b->table_width >= 0, "table_width is negative").shape(b->prefix_len >= 0, "prefix_len is negative");
    c.shape(b->table_stride >= b->table_width, "table_stride is shorter than table_width");
    if (!c.ok) return;
    // the kernels round rows up to units of 64 and name those of units that they ask for ahead, in 32 bits
    c.shape((int64_t)b->table_width * kv->page_size + b->prefix_len + b->n_tokens <= INT_MAX - 1024,
            "prefix_len, the table's rows and n_tokens add up to 2^31 - 1024 or more");
    c.need(b->n_tokens <= 1 << 23, BPDQ_ERR_LIMIT, "n_tokens is above 2^23");  // a workgroup each
    c.need(b->n_seqs <= 1 << 30, BPDQ_ERR_LIMIT, "n_seqs is above 2^30");  // the search takes up to 63 more, in 32 bits
    c.shape(b->q_start != nullptr || b->n_tokens == b->n_seqs, "without q_start n_tokens has to be n_seqs");
    if (!c.ok || b->n_seqs == 0 || b->n_tokens == 0) return;
    if (b->table_width > 0) c.ptr(b->table, 4, "batch.table");
    c.ptr(b->lens, 4, "batch.lens");
    if (b->q_start != nullptr) c.ptr(b->q_start, 4, "batch.q_start");
    if (b->prefix_len > 0) c.ptr(b->prefix, 4, "batch.prefix");
}

bpdq::Paged paged(const bpd_paged_cache& kv, const bpd_paged_batch& b) {
    bpdq::Paged a;
    a.k = static_cast<uint8_t*>(kv.k);
    a.v = static_cast<uint8_t*>(kv.v);
    a.n_pages = kv.n_pages;
    a.hkv = kv.n_kv_heads;
    a.D = kv.head_dim;
    a.page = bpdq::fast_div(kv.page_size);
    a.page_stride = (int)kv.page_stride;
    a.row_stride = (int)kv.row_stride;
    a.head_stride = (int)kv.head_stride;
    a.table = b.table;
    a.table_stride = b.table_stride;
    a.W = b.table_width;
    a.lens = b.lens;
    a.q_start = b.q_start;
    a.B = b.n_seqs;
    a.T = b.n_tokens;
    a.prefix = b.prefix;
    a.P = b.prefix_len;
    return a;
}

// The caller's workspace or the library's; nullptr with the error recorded.
void* work_space(bpdq::WsLease& lease, void* ws, int64_t ws_bytes, int64_t need, hipStream_t stream, const char* fn) {
    if (ws == nullptr) {
        lease = bpdq::workspace((size_t)need, stream, fn);
        return lease.ptr;
    }
    Args c(fn);
    c.shape(ws_bytes >= need, "ws_bytes is below what the call needs").ptr(ws, 16, "ws");
    return c.ok ? ws : nullptr;
}

// Whether rows of `row` bytes, n of them `as` and `bs` bytes apart, share a byte.  Rows of one stride may lie
// between each other.
bool overlap(const void* a, int64_t as, int64_t arow, const void* b, int64_t bs, int64_t brow, int n) {
    const int64_t d = (int64_t)(reinterpret_cast<uintptr_t>(b) - reinterpret_cast<uintptr_t>(a));
    if (d >= (n - 1) * as + arow || -d >= (n - 1) * bs + brow) return false;
    if (as != bs) return true;
    const int64_t at = (d % as + as) % as;  // of b's rows behind a's
    return at < arow || at + brow > as;
}

// What the attention's kernels index with 32 bits: heads of a launch, rows of a kv head, units, results.
void check_attn(Args& c, const bpd_paged_cache& kv, const bpd_paged_batch& b, int n_heads) {
    c.shape(n_heads >= 1 && n_heads % kv.n_kv_heads == 0, "n_heads is no multiple of n_kv_heads above 0");
    c.need(n_heads <= 1 << 16, BPDQ_ERR_LIMIT, "n_heads is above 2^16");
    if (!c.ok) return;
    const int64_t rows = (int64_t)b.n_tokens * (n_heads / kv.n_kv_heads);
    c.need(rows <= 1 << 26, BPDQ_ERR_LIMIT, "n_tokens times the heads of a kv head is above 2^26");
    const int64_t items = 2 * (rows / 64 + 1) + b.n_seqs;  // of 64 rows at least, of 64 keys' units
    const int64_t units = ((int64_t)b.table_width * kv.page_size + b.prefix_len) / (b.q_start != nullptr ? 64 : 32) + 2;
    c.need(items <= INT_MAX / units && items <= INT_MAX / 2 / kv.n_kv_heads, BPDQ_ERR_LIMIT,
           "sequences, tokens and their lengths multiply to 2^31 or more");
}

void check_sample(Args& c, int n_rows, int vocab) {
    c.shape(n_rows >= 0, "n_rows is negative").shape(vocab >= 0, "vocab is negative");
    c.need(vocab <= 1 << 22, BPDQ_ERR_LIMIT, "vocab is above 2^22");
    // workgroups of a launch: a row's, or its slices' of 2048 logits at least, 16384 where they are many
    c.need(n_rows < 1 << 22 && (int64_t)n_rows * (vocab / 16384 + 1) < 1 << 22, BPDQ_ERR_LIMIT, "n_rows is too large");
}

}  // namespace

extern "C" {

void bpd_rope_append_paged_on_gpu(void* hip_stream, const bpd_paged_cache* kv, const bpd_paged_batch* b,
                                  const bpd_rope* rope, const int32_t* pos, const void* q, int64_t q_stride,
                                  const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* q_out,
                                  int64_t q_out_stride, int x_type, int n_heads) {
    const char* fn = "bpd_rope_append_paged_gpu";
    const hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    Args c(fn);
    check_paged(c, kv, b);
    c.shape(x_type == BPD_T_F32 || x_type == BPD_T_F16 || x_type == BPD_T_BF16, "x_type is unknown");
    c.shape(n_heads >= 0 && n_heads <= INT_MAX / 1024, "n_heads is negative or too large");
    c.shape((k == nullptr) == (v == nullptr), "one of k and v is NULL");
    if (!c.ok) return;
    c.shape(kv->n_kv_heads <= INT_MAX / 1024, "n_kv_heads is too large");
    if (rope != nullptr)
        c.shape(rope->rot_dim >= 0 && rope->rot_dim % 2 == 0 && rope->rot_dim <= kv->head_dim,
                "rot_dim is negative, odd or above head_dim").shape(rope->neox == 0 || rope->neox == 1,
                                                                     "neox is neither 0 nor 1");
    if (!c.ok || b->n_seqs == 0 || b->n_tokens == 0) return;
    const int es = esize(x_type);
    if (n_heads > 0)
        c.ptr(q, 16, "q").ptr(q_out, 16, "q_out").stride(q_stride, (int64_t)n_heads * kv->head_dim, es, "q_stride")
            .stride(q_out_stride, (int64_t)n_heads * kv->head_dim, es, "q_out_stride");
    if (k != nullptr)
        c.ptr(k, 16, "k").ptr(v, 16, "v").stride(k_stride, (int64_t)kv->n_kv_heads * kv->head_dim, es, "k_stride")
            .stride(v_stride, (int64_t)kv->n_kv_heads * kv->head_dim, es, "v_stride");
    const int rot = rope == nullptr ? 0 : rope->rot_dim;
    if (rot > 0) c.ptr(rope->turns, 8, "rope.turns");
    if (pos != nullptr) c.ptr(pos, 4, "pos");
    if (!c.ok || (n_heads == 0 && k == nullptr)) return;
    if (n_heads > 0) {
        const int64_t row = (int64_t)es * n_heads * kv->head_dim, kv_row = (int64_t)es * kv->n_kv_heads * kv->head_dim;
        c.shape((q == q_out && q_stride == q_out_stride) ||
                    !overlap(q, es * q_stride, row, q_out, es * q_out_stride, row, b->n_tokens),
                "q_out overlaps q and is not q");
        if (k != nullptr)
            c.shape(!overlap(q_out, es * q_out_stride, row, k, es * k_stride, kv_row, b->n_tokens) &&
                        !overlap(q_out, es * q_out_stride, row, v, es * v_stride, kv_row, b->n_tokens),
                    "q_out overlaps k or v");
        if (!c.ok) return;
    }
    bpdq::launch_rope_append(paged(*kv, *b), kv->type, rot > 0 ? rope->turns : nullptr, rot,
                             rot > 0 && rope->neox == 1, pos, q, q_stride, k, k_stride, v, v_stride, q_out,
                             q_out_stride, x_type, n_heads, stream);
    bpdq::abi_hip_ok(hipGetLastError(), fn);
}

void bpd_rope_append_paged_gpu(const bpd_paged_cache* kv, const bpd_paged_batch* b, const bpd_rope* rope,
                               const int32_t* pos, const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                               const void* v, int64_t v_stride, void* q_out, int64_t q_out_stride, int x_type,
                               int n_heads) {
    bpd_rope_append_paged_on_gpu(bpdq::abi_stream(), kv, b, rope, pos, q, q_stride, k, k_stride, v, v_stride, q_out,
                                 q_out_stride, x_type, n_heads);
}

int64_t bpd_attn_paged_workspace(const bpd_paged_cache* kv, const bpd_paged_batch* b, int n_heads) {
    Args c("bpd_attn_paged_workspace");
    check_paged(c, kv, b);
    if (!c.ok) return -1;
    check_attn(c, *kv, *b, n_heads);
    if (!c.ok) return -1;
    return bpdq::attn_paged_ws(b->q_start, b->n_seqs, b->n_tokens, n_heads, kv->n_kv_heads, kv->head_dim,
                               b->prefix_len);
}

void bpd_attn_paged_on_gpu(void* hip_stream, const bpd_paged_cache* kv, const bpd_paged_batch* b, const void* q,
                           int64_t q_stride, void* out, int64_t out_stride, float* lse, int q_type, int n_heads,
                           float scale, void* ws, int64_t ws_bytes) {
    const char* fn = "bpd_attn_paged_gpu";
    const hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    Args c(fn);
    check_paged(c, kv, b);
    if (!c.ok) return;
    c.shape(q_type == BPD_T_F32 || q_type == kv->type, "q_type is neither fp32 nor the cache's type");
    check_attn(c, *kv, *b, n_heads);
    if (!c.ok || b->n_seqs == 0 || b->n_tokens == 0) return;
    const int es = esize(q_type);
    const int64_t row = (int64_t)n_heads * kv->head_dim;
    c.ptr(q, 16, "q").stride(q_stride, row, es, "q_stride");
    c.ptr(out, 16, "out").stride(out_stride, row, es, "out_stride");
    if (lse != nullptr) c.ptr(lse, 4, "lse");
    if (!c.ok) return;
    // rows are written while others are still read
    c.shape(!overlap(q, es * q_stride, es * row, out, es * out_stride, es * row, b->n_tokens), "q and out overlap");
    if (!c.ok) return;
    bpdq::WsLease lease;
    const int64_t need = bpdq::attn_paged_ws(b->q_start, b->n_seqs, b->n_tokens, n_heads, kv->n_kv_heads, kv->head_dim,
                                             b->prefix_len);
    void* w = work_space(lease, ws, ws_bytes, need, stream, fn);
    if (w == nullptr) return;
    bpdq::launch_attn_paged(paged(*kv, *b), kv->type, q, q_stride, out, out_stride, lse, q_type, n_heads, scale, w,
                            stream);
    bpdq::abi_hip_ok(hipGetLastError(), fn);
}

void bpd_attn_paged_gpu(const bpd_paged_cache* kv, const bpd_paged_batch* b, const void* q, int64_t q_stride,
                        void* out, int64_t out_stride, float* lse, int q_type, int n_heads, float scale, void* ws,
                        int64_t ws_bytes) {
    bpd_attn_paged_on_gpu(bpdq::abi_stream(), kv, b, q, q_stride, out, out_stride, lse, q_type, n_heads, scale, ws,
                          ws_bytes);
}

int64_t bpd_sample_workspace(int n_rows, int vocab) {
    Args c("bpd_sample_workspace");
    check_sample(c, n_rows, vocab);
    return c.ok ? bpdq::sample_ws(n_rows, vocab) : -1;
}

void bpd_sample_on_gpu(void* hip_stream, const void* logits, int type, int64_t row_stride, int n_rows, int vocab,
                       const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                       const float* u, int32_t* token, float* logprob, int32_t* n_kept, void* ws, int64_t ws_bytes) {
    const char* fn = "bpd_sample_gpu";
    const hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    Args c(fn);
    c.shape(type == BPD_T_F32 || type == BPD_T_F16 || type == BPD_T_BF16, "type is unknown");
    check_sample(c, n_rows, vocab);
    c.shape(row_stride >= vocab && row_stride <= kMaxStride, "row_stride is shorter than a row, or 2^30 or more");
    if (!c.ok || n_rows == 0) return;
    if (vocab > 0) c.ptr(logits, (uintptr_t)esize(type), "logits");
    c.ptr(u, 4, "u").ptr(token, 4, "token");
    if (temperature != nullptr) c.ptr(temperature, 4, "temperature");
    if (top_k != nullptr) c.ptr(top_k, 4, "top_k");
    if (top_p != nullptr) c.ptr(top_p, 4, "top_p");
    if (min_p != nullptr) c.ptr(min_p, 4, "min_p");
    if (logprob != nullptr) c.ptr(logprob, 4, "logprob");
    if (n_kept != nullptr) c.ptr(n_kept, 4, "n_kept");
    if (!c.ok) return;
    bpdq::WsLease lease;
    void* w = work_space(lease, ws, ws_bytes, bpdq::sample_ws(n_rows, vocab), stream, fn);
    if (w == nullptr) return;
    bpdq::launch_sample({logits, row_stride, n_rows, vocab, temperature, top_k, top_p, min_p, u, token, logprob,
                         n_kept}, type, w, stream);
    bpdq::abi_hip_ok(hipGetLastError(), fn);
}

void bpd_sample_gpu(const void* logits, int type, int64_t row_stride, int n_rows, int vocab, const float* temperature,
                    const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* token,
                    float* logprob, int32_t* n_kept, void* ws, int64_t ws_bytes) {
    bpd_sample_on_gpu(bpdq::abi_stream(), logits, type, row_stride, n_rows, vocab, temperature, top_k, top_p, min_p, u,
                      token, logprob, n_kept, ws, ws_bytes);
}

}  // extern "C"
