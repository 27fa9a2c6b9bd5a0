/* bpdq_serve.h — operators that serve many sequences at once, part of
 * libbpdq_hip.so (gfx950 / MI355X).  No counterpart in the reference, whose
 * decode step runs one sequence over one contiguous cache and takes the argmax
 * (include/bpdq_llama.h); the conventions are those of include/bpdq.h.
 *
 *   bpd_rope_append_paged_gpu  the new tokens' queries and keys rotated, keys and
 *                              values written into the pages of a shared cache
 *   bpd_attn_paged_gpu         attention over those pages for a batch whose
 *                              sequences may share a prefix
 *   bpd_sample_gpu             one token per row of logits: temperature, top-k,
 *                              top-p, min-p, from given random numbers
 *
 * The structs are host memory, read during the call; the pointers in them and
 * every other tensor argument are device memory.  Sizes that live on the device
 * (lens, q_start, table, prefix) are read by the kernels, so a captured graph
 * follows their contents from replay to replay.  Whatever they hold, no access
 * leaves the tensors that the structs describe: a length is clamped to the
 * table, a value of q_start to [0, n_tokens], and a page index outside [0, n_pages)
 * makes its rows absent (not written by the append, not seen by the attention).
 */
#ifndef BPDQ_SERVE_H
#define BPDQ_SERVE_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
#define BPD_T_F32 0
#define BPD_T_F16 1
#define BPD_T_BF16 2

/* A paged K/V cache: row r of head h of page p starts at element
 * p * page_stride + r * row_stride + h * head_stride of k and of v and holds
 * head_dim contiguous elements.  Any layout with 16-byte aligned rows will do: pages
 * of [heads][rows] or of [rows][heads], or the contiguous [max_seq][n_head_kv *
 * head_dim] binary16 cache of the decode step as one page per sequence or per
 * max_seq / page_size rows. */
typedef struct {
    void* k;
    void* v;
    int type; /* BPD_T_F16 or BPD_T_BF16 */
    int n_pages, page_size, n_kv_heads, head_dim; /* head_dim a multiple of 8, 8..256 */
    int64_t page_stride, row_stride, head_stride; /* elements, multiples of 8 */
} bpd_paged_cache;

/* A batch of n_seqs sequences and its n_tokens new tokens.  Row i of sequence
 * b's own part is row i % page_size of page table[b * table_stride + i / page_size]; it
 * holds lens[b] rows, the new tokens' among them, which are the last
 * n_b = q_start[b + 1] - q_start[b].  New token t of sequence b
 * (q_start[b] <= t < q_start[b + 1], q_start not decreasing) has index
 * lens[b] - n_b + t - q_start[b] there and position prefix_len + index.  Tokens
 * outside [q_start[0], q_start[n_seqs]) belong to no sequence: nothing is written
 * for them.  With q_start NULL every sequence has one new token
 * (n_tokens == n_seqs).  The prefix comes before every sequence's own part: row i is
 * row i % page_size of page prefix[i / page_size].  table_width * page_size, prefix_len
 * and n_tokens add up to less than 2^31 - 1024; n_seqs up to 2^30 (BPDQ_ERR_LIMIT). */
typedef struct {
    const int32_t* table;
    int64_t table_stride;
    int table_width;
    const int32_t* lens;
    const int32_t* q_start;
    int n_seqs, n_tokens;
    const int32_t* prefix;
    int prefix_len;
} bpd_paged_batch;

/* The rotation: the first rot_dim (even) elements of each head turn in pairs,
 * elements (2j, 2j + 1), or with neox 1 (j, j + rot_dim / 2).  turns[j], device
 * binary64: revolutions of pair j per position (frequency / 2 pi). */
typedef struct {
    const double* turns;
    int rot_dim;
    int neox;
} bpd_rope;

/* For every new token: q_out = rotated q, and the token's row of the cache =
 * rotated k and v, rounded once to the cache's type.  The angle is taken in
 * binary64 and the rotation in binary32.  rope NULL: no rotation.  pos (int32
 * [n_tokens]) or NULL: positions other than prefix_len + index.  q [n_tokens]
 * [n_heads][head_dim] and k, v [n_tokens][n_kv_heads][head_dim] of x_type, tokens
 * q_stride, k_stride and v_stride elements apart (the parts of one projection's
 * row, for instance); q_out of x_type, may be q itself and overlaps it or k and v in no
 * other way; q may be NULL with n_heads 0, k and v NULL together (nothing is appended).  Tensors and token
 * strides 16-byte aligned.  A row that two tokens write (one page in two
 * sequences' tables) holds elements of either. */
void bpd_rope_append_paged_gpu(const bpd_paged_cache* cache, const bpd_paged_batch* batch, const bpd_rope* rope,
                               const int32_t* pos, const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                               const void* v, int64_t v_stride, void* q_out, int64_t q_out_stride, int x_type,
                               int n_heads);

/* out[t][h] = sum_i softmax_i(scale * q[t][h] . k_i) v_i over the prefix's rows and
 * rows 0..index of the token's sequence, of kv head h / (n_heads / n_kv_heads);
 * lse[t][h] (fp32, may be NULL) = log sum_i exp(scale * q . k_i).  A token
 * that sees no row gets zeros, and an lse of -infinity.  What stands in rows that a
 * token does not see (infinities and NaN too) does not reach its output.  q and out
 * [n_tokens][n_heads][head_dim] of q_type: the cache's type, or fp32; rows of out and q do
 * not overlap.  Scores, statistics and sums are fp32 for either.  With q of the cache's type
 * the softmax's weights are rounded to that type once before they meet v (half a step of each,
 * 2^-11 or 2^-8; the denominator sums them unrounded); with fp32 q they keep 22 bits (f16 pages)
 * or 24 (bf16), as the queries do.  Tensors and token strides
 * 16-byte aligned (lse 4).  n_heads a multiple of n_kv_heads, up to 2^16; n_tokens up to
 * 2^23, times n_heads / n_kv_heads 2^26; beyond, and where the tokens' tiles times
 * the table's rows pass 2^31 units, BPDQ_ERR_LIMIT.
 * ws: at least bpd_attn_paged_workspace() bytes, 16-byte aligned, for this call
 * alone until it has run, or NULL: the library's workspace of (device, stream). */
void bpd_attn_paged_gpu(const bpd_paged_cache* cache, const bpd_paged_batch* batch, const void* q, int64_t q_stride,
                        void* out, int64_t out_stride, float* lse, int q_type, int n_heads, float scale, void* ws,
                        int64_t ws_bytes);
int64_t bpd_attn_paged_workspace(const bpd_paged_cache* cache, const bpd_paged_batch* batch, int n_heads);

/* One token per row of logits [n_rows][vocab] (type, rows row_stride elements
 * apart, aligned to an element; vocab up to 2^22, n_rows and n_rows * vocab / 16384
 * below 2^22, more is BPDQ_ERR_LIMIT).  In order, each over what the one before left,
 * equal logits ranked by index:
 *   temperature  weights w_i = exp((l_i - max l) / temperature); not above 0: the
 *                largest logit alone
 *   top_k        the top_k largest; below 1: all
 *   top_p        the fewest largest ones whose weights reach top_p of the sum, at
 *                least one; 1 or more: all
 *   min_p        those with w_i >= min_p (times the largest weight, which is 1), at
 *                least the first of the largest, which above 1 is left alone
 * then token = the first index, in the vocabulary's order, at which the sum of the
 * weights left exceeds u times their total.  One value of each per row; a NULL array:
 * temperature 1, no filter.  u in [0, 1).  NaN and -infinity logits are never
 * chosen; with +infinity ones among them, only these are, alike.  logprob (may
 * be NULL): the log of token's share of the weights left; n_kept (may be NULL): how
 * many are left.  A row with nothing to choose gives -1, NaN and 0.  Weights are taken
 * in binary64 and summed exactly as multiples of 2^-44 (vocab up to 2^18; twice
 * that for every doubling beyond), so no result depends on the order of a sum.
 * ws: as above, at least bpd_sample_workspace() bytes. */
void bpd_sample_gpu(const void* logits, int type, int64_t row_stride, int n_rows, int vocab, const float* temperature,
                    const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* token,
                    float* logprob, int32_t* n_kept, void* ws, int64_t ws_bytes);
int64_t bpd_sample_workspace(int n_rows, int vocab);

/* The same three on a stream of the current device given with the call (a hipStream_t; NULL = the null
 * stream).  bpd_gpu_set_stream()'s stream is one for the process, and a call that takes it has to be kept apart from
 * other threads' choices; these neither read nor change it. */
void bpd_rope_append_paged_on_gpu(void* hip_stream, const bpd_paged_cache* cache, const bpd_paged_batch* batch,
                                  const bpd_rope* rope, const int32_t* pos, const void* q, int64_t q_stride,
                                  const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* q_out,
                                  int64_t q_out_stride, int x_type, int n_heads);
void bpd_attn_paged_on_gpu(void* hip_stream, const bpd_paged_cache* cache, const bpd_paged_batch* batch, const void* q,
                           int64_t q_stride, void* out, int64_t out_stride, float* lse, int q_type, int n_heads,
                           float scale, void* ws, int64_t ws_bytes);
void bpd_sample_on_gpu(void* hip_stream, const void* logits, int type, int64_t row_stride, int n_rows, int vocab,
                       const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                       const float* u, int32_t* token, float* logprob, int32_t* n_kept, void* ws, int64_t ws_bytes);

#ifdef __cplusplus
}
#endif
#endif
