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
 *   bpd_pages_extend_gpu       pages from a pool for sequences that grow, with their
 *                              tables, and every new token's slot and position
 *   bpd_pages_release_gpu      pages back to the pool
 *   bpd_norm_rope_append_paged_gpu  the append, every head of q and k normed first
 *   bpd_attn_window_paged_gpu  the attention over a sliding window and the first rows
 *   bpd_adjust_logits_gpu      penalties, biases and masks on logits
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

/* A pool of n_pages pages of page_size rows, and the sequences that hold them, a row of table each.
 * Entries [0, ceil(lens[r] / page_size)) of row r are its pages, in order; -1 one that it gave
 * back.  free_pages[0 .. n_free[0]) are the pages that no sequence holds.  gone (may be NULL, without windows):
 * pages [gone[2 r], gone[2 r + 1]) of row r have slid out of its window and were given back.  All of it is
 * device memory that the caller fills once (tables -1, lens, gone and n_free[1] 0) and the two calls below keep.
 * Calls on one pool follow each other, on one stream or by events.  Their rows, n_new and keep lie in none of its
 * arrays; with rows NULL n_new and keep may be lens.
 * Pages that are no part of the pool (a shared prefix's) are left out of free_pages.  n_pages and table_width times
 * page_size stay below 2^31; n_rows up to 16384 (BPDQ_ERR_LIMIT). */
typedef struct {
    int32_t* table;
    int64_t table_stride;
    int table_width;
    int32_t* lens;
    int32_t* gone;
    int32_t* free_pages;
    int32_t* n_free; /* [2]: how many, and a counter of the calls' own */
    int n_rows, n_pages, page_size;
} bpd_page_pool;

/* Sequence b = 0 .. n_seqs - 1 (n_seqs up to n_rows), row rows[b] of the pool (rows NULL: row b), grows by
 * n_new[b] rows, 0 or more.  In that order each is granted what it asks for, or nothing; refused[b] says
 * which: 0 granted; 1 no row of the pool, one that an earlier sequence names, or n_new below 0; 2 more rows than
 * its table holds; 3 the pages asked for by it and all before it are more than the pool has (a sequence that needs no
 * page is not refused for that); 4 with the tokens of it and of those before it that pages were there for they would be
 * more than n_tokens.  Pages come from the end of free_pages.  lens and table of the pool follow.
 * Outputs, device memory that overlaps nothing else of the call (with n_seqs 0 nothing is written): lens_out[b] the sequence's rows (0 without a row of the pool), q_start[n_seqs + 1] the running sum of tokens granted,
 * slots[t] and pos[t] of every new token its row of the cache, page * page_size + row in it (-1 where its
 * page is outside the pool), and its position, prefix_len + index; -1 of tokens behind the last.  table_out
 * (may be NULL) [n_seqs][table_width]: the sequences' tables, -1 behind their pages.  With these a bpd_paged_batch
 * describes the step.  n_tokens up to 2^23, with prefix_len and a table's rows below 2^31 - 1024. */
void bpd_pages_extend_gpu(const bpd_page_pool* pool, const int32_t* rows, const int32_t* n_new, int n_seqs, int n_tokens,
                          int prefix_len, int32_t* table_out, int64_t table_out_stride, int32_t* lens_out,
                          int32_t* q_start, int32_t* slots, int32_t* pos, int32_t* refused);

/* Sequence b keeps its first keep[b] rows (NULL, or more than it has: all), and of those, with a window above 0
 * (gone not NULL), the pages that hold one of the first `sinks` rows or a row that a token at index keep[b] or
 * later sees through the window: those from keep[b] - window + 1 on.  sinks counts rows of the sequence's own part and
 * is the same from call to call.  A page that slid out stays out, also where its sequence is cut back behind it later.
 * The other pages go to the end of free_pages, the first sequence's first page last, so that an extension which is
 * taken back leaves the pool as it was; their entries become -1.  Rows that are not the pool's, and all
 * but the first sequence that names a row, are passed over. */
void bpd_pages_release_gpu(const bpd_page_pool* pool, const int32_t* rows, const int32_t* keep, int n_seqs, int window,
                           int sinks);

/* bpd_rope_append_paged_gpu with every head of q and k normed before it turns:
 *   y_i = x_i / sqrt(mean over the head of x^2 + eps) * w_i
 * q_norm and k_norm: [head_dim] weights of all heads (stride 0), or of each, a head's stride elements
 * behind the one before (multiples of 8, head_dim at least); of w_type, fp32 or x_type, 16-byte aligned.  NULL: not
 * normed.  eps is not below 0.  The sum of squares, the scale and the rotation are binary32 (a head whose squares add up beyond it
 * becomes 0), and the result is rounded once. */
void bpd_norm_rope_append_paged_gpu(const bpd_paged_cache* cache, const bpd_paged_batch* batch, const void* q_norm,
                                    int64_t q_norm_stride, const void* k_norm, int64_t k_norm_stride, int w_type,
                                    float eps, const bpd_rope* rope, const int32_t* pos, const void* q, int64_t q_stride,
                                    const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* q_out,
                                    int64_t q_out_stride, int x_type, int n_heads);

/* bpd_attn_paged_gpu over a window: of the rows that it lets a token at position p (prefix_len + index) see, those at
 * positions j > p - window or j < sinks, the prefix's rows being the first.  window at least 1, sinks 0 or more.
 * Pages without a row that a new token sees are not read: their entries of the table may be -1.  The same rules and
 * limits otherwise; ws: at least bpd_attn_window_paged_workspace() bytes, which may be 0 (then ws is not looked at). */
void bpd_attn_window_paged_gpu(const bpd_paged_cache* cache, const bpd_paged_batch* batch, const void* q,
                               int64_t q_stride, void* out, int64_t out_stride, float* lse, int q_type, int n_heads,
                               float scale, int window, int sinks, void* ws, int64_t ws_bytes);
int64_t bpd_attn_window_paged_workspace(const bpd_paged_cache* cache, const bpd_paged_batch* batch, int q_type,
                                        int n_heads, int window, int sinks);

/* What happens to a row of logits before it is sampled, in this order, in binary32:
 *   history    tokens[row][0 .. lens[row]) (lens NULL: width), the first prompt[row] of them the prompt's (NULL:
 *              none).  A token that stands there has l = l > 0 ? l / repetition : l * repetition; one that stands
 *              behind the prompt, n times, then l - n * frequency - presence
 *   bias       entries bias_start[row] .. bias_start[row + 1] of a list: l + bias_value of its bias_token; of a token with
 *              several entries the last one counts
 *   mask       bit t % 32 of word t / 32 of mask row mask_row[row] (NULL: row `row`): where it is 0, l =
 *              -infinity whatever it was.  A row outside [0, n_masks): none
 * One repetition, frequency and presence per row; NULL: 1, 0, 0.  Lengths are clamped to the arrays
 * (bias_start to [0, n_bias]), and tokens outside [0, vocab) passed over, so rows may be padded with them. */
typedef struct {
    const int32_t* tokens; /* NULL: no history */
    int64_t token_stride;
    int token_width;
    const int32_t *lens, *prompt;
    const float *repetition, *frequency, *presence;
    const int32_t* bias_start; /* NULL: no biases */
    const int32_t* bias_token;
    const float* bias_value;
    int n_bias;
    const int32_t* mask; /* NULL: no masks */
    int64_t mask_stride; /* words, ceil(vocab / 32) at least */
    int n_masks;
    const int32_t* mask_row;
} bpd_logit_rules;

/* out [n_rows][vocab] (out_type: that of the logits, or fp32) = the logits under the rules, rounded once; rows
 * row_stride and out_stride elements apart, aligned to an element.  out may be the logits themselves, and overlaps them in
 * no other way.  vocab as in bpd_sample_gpu, n_rows * (vocab / 8192 + 1) below 2^22 (BPDQ_ERR_LIMIT). */
void bpd_adjust_logits_gpu(const void* logits, int type, int64_t row_stride, void* out, int out_type, int64_t out_stride,
                           int n_rows, int vocab, const bpd_logit_rules* rules);

/* The same on a stream of the current device given with the call (a hipStream_t; NULL = the null
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
void bpd_pages_extend_on_gpu(void* hip_stream, const bpd_page_pool* pool, const int32_t* rows, const int32_t* n_new,
                             int n_seqs, int n_tokens, int prefix_len, int32_t* table_out, int64_t table_out_stride,
                             int32_t* lens_out, int32_t* q_start, int32_t* slots, int32_t* pos, int32_t* refused);
void bpd_pages_release_on_gpu(void* hip_stream, const bpd_page_pool* pool, const int32_t* rows, const int32_t* keep,
                              int n_seqs, int window, int sinks);
void bpd_norm_rope_append_paged_on_gpu(void* hip_stream, const bpd_paged_cache* cache, const bpd_paged_batch* batch,
                                       const void* q_norm, int64_t q_norm_stride, const void* k_norm,
                                       int64_t k_norm_stride, int w_type, float eps, const bpd_rope* rope,
                                       const int32_t* pos, const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                                       const void* v, int64_t v_stride, void* q_out, int64_t q_out_stride, int x_type,
                                       int n_heads);
void bpd_attn_window_paged_on_gpu(void* hip_stream, const bpd_paged_cache* cache, const bpd_paged_batch* batch,
                                  const void* q, int64_t q_stride, void* out, int64_t out_stride, float* lse, int q_type,
                                  int n_heads, float scale, int window, int sinks, void* ws, int64_t ws_bytes);
void bpd_adjust_logits_on_gpu(void* hip_stream, const void* logits, int type, int64_t row_stride, void* out, int out_type,
                              int64_t out_stride, int n_rows, int vocab, const bpd_logit_rules* rules);

#ifdef __cplusplus
}
#endif
#endif
