/* artread.h — C ABI of libartread.so: the operators that READ the passages a search found.
 *
 * libartmips finds passages, libarttok fetches their tokens into padded rows with lengths; these
 * operators take those rows on: the embedding lookup of the gathered tokens with its gradient, and
 * the attention of a question to the states of its passages with its gradient.
 *
 * Conventions as in artmips.h and arttok.h: 0 on success, a negative code on failure,
 * artread_last_error() for the message of the calling thread; plain device pointers and sizes, no
 * torch types, no exceptions; `stream` is a hipStream_t as void*.  Every call only enqueues work on
 * `stream` of `device` (no allocation, no synchronisation, no state kept between calls), so calls
 * may be captured into a HIP graph and any number of threads may call at once.  Workspaces belong
 * to the caller: calls that may overlap need one each.  Arguments are checked before anything is
 * launched; lengths, tokens and the other contents of device memory are bounded by the kernels.
 *
 * Outputs and workspaces overlap neither each other nor any input.
 *
 * `lengths` is what arttok_gather writes: the number of valid entries of a padded row, negative for
 * a passage that is not there (read as 0); a value above the padded length is read as that length.
 */
#ifndef ARTREAD_H
#define ARTREAD_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types, numbered as in artmips.h */
enum { ARTREAD_F16 = 0, ARTREAD_BF16 = 1, ARTREAD_F32 = 2 };

enum {
    ARTREAD_OK = 0,
    ARTREAD_ERR_ARG = -1,
    ARTREAD_ERR_HIP = -2,
    ARTREAD_ERR_UNSUPPORTED = -4
};

/* out[i, t, :] = scale * table[tokens[i, t] - vocab_base, :]   for t < lengths[i],
 * zeros at the other positions and for a token outside [vocab_base, vocab_base + vocab): the rows of
 * a vocabulary split over ranks add up (megatron/mpu/layers.py, VocabParallelEmbedding).
 *   table    [vocab, dim], rows table_stride elements apart
 *   tokens   [n, len] contiguous, int32 or int64 (token_bytes 4 or 8); lengths [n] or NULL (all of len)
 *   out      [n, len, dim] contiguous, of out_dtype: the table's type, or f16 / bf16 of an f32 table.
 * The product is formed in f32 and rounded once.  n * len and vocab are below 2^31. */
int artread_embed(int device, const void* table, int table_dtype, int64_t vocab, int64_t dim,
                  int64_t table_stride, const void* tokens, int token_bytes, const int32_t* lengths, int64_t n,
                  int64_t len, int64_t vocab_base, float scale, void* out, int out_dtype, void* stream);

/* grad_table[v, :] = scale * (sum of grad_out[i, t, :] over the valid positions whose token is
 * v + vocab_base): every row of grad_table [vocab, dim] (contiguous) is written, unused ones with
 * zeros.  Sums are f32, in an order fixed by the tokens and sizes alone: equal inputs give equal bits.
 * grad_out is contiguous [n, len, dim] of f16, bf16 or f32; grad_table has its type, or f32.
 * `workspace` (16-byte aligned device memory) holds at least artread_embed_grad_workspace bytes. */
int64_t artread_embed_grad_workspace(int64_t vocab, int64_t dim, int64_t n, int64_t len);
int artread_embed_grad(int device, const void* grad_out, int grad_dtype, const void* tokens, int token_bytes,
                       const int32_t* lengths, int64_t n, int64_t len, int64_t vocab, int64_t dim,
                       int64_t vocab_base, float scale, void* grad_table, int table_dtype, void* workspace,
                       int64_t workspace_bytes, void* stream);

/* Attention of `rows` query rows per batch entry to the states of `passages` passages of `len` padded
 * entries each; entry j of passage p of batch entry b is a key iff j < lengths[b, p].  One softmax runs
 * over all keys of a batch entry; a row without any key gives zeros and lse = -inf.  What lies behind a
 * passage's length is never used, whatever its value.
 *   q, out   [batch, rows, heads, dim];  k, v [batch, passages, len, kv_heads, dim];
 *   lse      [batch, heads, rows] f32: log of the sum of exp(scale * q.k), or NULL
 *   rest     [batch, rows, heads, dim] contiguous, or NULL: what rounding took from out, rounded to its type.
 *            out + rest carries about twice out's bits, which the gradient's row sums need
 *   heads is a multiple of kv_heads: query head h reads key head h / (heads / kv_heads)
 * f16 or bf16, dim a multiple of 8 up to 128.  Strides count elements; the innermost one is 1, the
 * others are >= 0 and multiples of 8, those of rows below 2^24, the query heads that share a key head
 * within 2^29 elements, the rest below 2^40.  Pointers are 16-byte aligned; out is contiguous.
 * Scores, softmax statistics and sums are f32; weights are rounded once to the states' type before they meet v.
 * Passages that lie one behind the other in memory may share tiles, those with gaps between them do not: equal
 * inputs with equal strides give equal bits, with other strides the last ones may differ. */
typedef struct {
    const void* q;
    const void* k;
    const void* v;
    const int32_t* lengths; /* [batch, passages] contiguous, or NULL: all of len */
    void* out;
    float* lse;
    void* rest;
    int64_t batch, rows, passages, len, heads, kv_heads, dim;
    int64_t q_batch, q_row, q_head;
    int64_t k_batch, k_passage, k_row, k_head;
    int64_t v_batch, v_passage, v_row, v_head;
    int32_t dtype;
    float scale;
} artread_attend_t;

int64_t artread_attend_workspace(const artread_attend_t* a);
int artread_attend(int device, const artread_attend_t* a, void* workspace, int64_t workspace_bytes, void* stream);

/* Gradients of artread_attend.  `a` describes the forward call, with its out, lse and rest as inputs here
 * (rest may be NULL: the row sums of grad_out * out then take out as it was rounded).
 * grad_out is [batch, rows, heads, dim] with the given strides; grad_q, grad_k and grad_v are contiguous
 * of q's, k's and v's shapes and written whole, zeros behind each passage's length.  No atomics: equal
 * inputs with equal strides give equal bits.  Weights and their gradients are rounded to the states' type
 * before the products that make grad_q, grad_k and grad_v, which add in f32. */
typedef struct {
    const void* grad_out;
    int64_t g_batch, g_row, g_head;
    void* grad_q;
    void* grad_k;
    void* grad_v;
} artread_attend_grads_t;

int64_t artread_attend_grad_workspace(const artread_attend_t* a);
int artread_attend_grad(int device, const artread_attend_t* a, const artread_attend_grads_t* g, void* workspace,
                        int64_t workspace_bytes, void* stream);

const char* artread_last_error(void);

#ifdef __cplusplus
}
#endif
#endif /* ARTREAD_H */
