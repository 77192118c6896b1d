/*
 * C ABI of the decode operators of libSpMM_API.so for gfx950 (MI355X): a paged key/value cache held in 4 bits with the
 * attention that reads it, and linears with 4-bit weights.  They stand beside the bitmap SpMM of spmm_api.h: what a
 * decode step needs between and next to the pruned linears.  None has a counterpart in the reference's library, whose
 * attention and dense linears are its FasterTransformer host's (third_party/ft_spinfer.patch:3722-3753 is the call that
 * the SpMM replaces there).
 *
 * All pointers are device memory unless stated; calls are asynchronous on `stream`, allocate nothing and never
 * synchronise the host, so they can be recorded into a HIP graph.  They return a hipError_t value as int: 0 on success,
 * 1 (hipErrorInvalidValue, with a message on stdout) for arguments that they refuse on the host before anything is
 * launched, otherwise the launch status.  An empty batch (no tokens, N = 0) is a success that launches nothing.
 *
 * The 4-bit cache.  A page holds `page_size` tokens of every key/value head:
 *   codes   uint8 [num_pages][kv_heads][page_size][head_dim/2]   element 2b in the low, 2b+1 in the high half of byte b
 *   words   int32 [num_pages][kv_heads][page_size]               bits of a float32 scale whose four lowest mantissa bits
 *                                                                are the zero point z of the token's vector
 *   value = float(word) * (code - z)
 * one pair of arrays for the keys, one for the values.  A vector x is encoded as
 *   hi = max(x, 0), lo = min(x, 0) over its elements, s = hi/15 - lo/15, rounded to 20 significant bits (s below 2^-100
 *   becomes 1), z = rint(-lo/s) in 0..15, put into the four lowest bits of s, code = clamp(rint(x/s) + z, 0, 15),
 * in float32 with quotients taken as products with the reciprocal; a vector with an infinite or NaN element is held as
 * NaN throughout, so that it shows in every row that sees it and in no other.
 * Words that a caller writes: a scale is 0, a positive normal number below 2^127, or NaN.  0, which a cleared cache holds, is a
 * vector of zeros; attention reads a value scale below 2^-126 as 0.  A row that sees a negative or an infinite scale has no
 * defined result.  Words of places that no row sees may be anything.
 *
 * A batch.  Sequence b has seq_lens[b] tokens in the cache, its tokens to be processed in this step (n_b of them, the
 * last ones) included; token p of it lies in page block_table[b*table_stride + p/page_size], slot p%page_size.  The
 * rows of q, k, v and of the outputs are the processed tokens of sequence 0, then of sequence 1 and so on:
 * cu_tokens[b] .. cu_tokens[b+1]-1 are sequence b's.  cu_tokens NULL: one token of every sequence.  The kernels check
 * every table entry and length against the arrays' sizes: a token of no sequence (past cu_tokens[batch]), one before a
 * sequence's start (n_b above seq_lens[b], as in padding with seq_lens[b] = 0), past the table's width or in a page
 * outside 0..num_pages-1 is neither written nor seen, and its row of an output is 0 (a query whose own page is outside
 * still attends to the keys that are there).
 */
#ifndef DECODE_API_H
#define DECODE_API_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#ifndef HIP_INCLUDE_HIP_HIP_RUNTIME_API_H
typedef struct ihipStream_t* hipStream_t;
#endif

/* Element types of activations, outputs and weight scales. */
#define DECODE_FP16 0
#define DECODE_BF16 1

/* A 4-bit cache: device arrays as above.  head_dim 64, 96, 128 or 256; page_size a power of two from 16 to 1024; codes
 * 16-byte aligned, words 16-byte aligned.  The struct itself is host memory and is read during the call only. */
typedef struct KV4_Cache {
    void*    k_codes;
    int32_t* k_words;
    void*    v_codes;
    int32_t* v_words;
    int32_t  num_pages;
    int32_t  page_size;
    int32_t  kv_heads;
    int32_t  head_dim;
} KV4_Cache;

/* A batch: device arrays as above, sizes on the host.  total_tokens is the number of rows of q, k, v and the outputs
 * (with cu_tokens NULL it equals batch).  Host memory, read during the call only. */
typedef struct KV4_Batch {
    const int32_t* block_table;
    const int32_t* seq_lens;
    const int32_t* cu_tokens;
    int32_t        batch;
    int32_t        table_width;
    int32_t        table_stride;
    int32_t        total_tokens;
} KV4_Batch;

/* Rows of heads: element (token, head, d) at data[token*token_stride + head*head_stride + d], strides in elements. */
typedef struct KV4_Rows {
    const void* data;
    int64_t     token_stride;
    int64_t     head_stride;
} KV4_Rows;

/* Rotary positions: for the first `dims` elements of a head (even, at most head_dim; 0 rotates nothing) the pair (a, b)
 * becomes (a*cos - b*sin, b*cos + a*sin), pairs (i, i + dims/2), or (2i, 2i+1) with `interleaved`; products and sums are
 * rounded to float32 one by one.  `table` is float32 [table_rows][dims], cosines in the first half of a row, sines in the
 * second.  A token's row is `positions`[token] (int32, may be NULL), otherwise its place in its sequence; a row outside
 * the table gives NaN, a token with no place and no entry in `positions` stays unrotated. */
typedef struct KV4_Rotary {
    const float*   table;
    const int32_t* positions;
    int32_t        table_rows;
    int32_t        dims;
    int32_t        interleaved;
} KV4_Rotary;

/* Encodes the keys (rotated) and values of the batch's tokens into the cache, and writes the rotated queries, rounded
 * once to `dtype`, to q_out [total_tokens][q_heads][head_dim].  q.data NULL: no queries (q_heads and q_out are not
 * read).  rotary NULL: nothing is rotated; then q must be NULL too.  q_out may be q.data itself where q is contiguous.
 * q, k, v may be any strided rows aligned to their element type; rows aligned to 16 bytes are read 16 bytes at a time. */
int KV4_Append(hipStream_t stream, const KV4_Cache* cache, const KV4_Batch* batch, KV4_Rows k, KV4_Rows v, KV4_Rows q,
               int q_heads, void* q_out, const KV4_Rotary* rotary, int dtype);

/* Reads the batch's tokens back: k and v [total_tokens][kv_heads][head_dim], the values of the cache rounded to `dtype`.
 * With cu_tokens spanning whole sequences it reads the whole cache of them.  k or v may be NULL. */
int KV4_Gather(hipStream_t stream, const KV4_Cache* cache, const KV4_Batch* batch, void* k, void* v, int dtype);

/* Attention of the batch's tokens over the cache: out[t][h] = sum_j p_j v_j, p = softmax over the visible keys of
 * scale * q[t][h] . k_j; query head h reads key/value head h / (q_heads / kv_heads).  Token at place p of its sequence
 * sees the keys 0 .. p, with `window` > 0 only the last `window` of them (its own included).  out is
 * [total_tokens][q_heads][head_dim] contiguous in `dtype`; lse, float32 [total_tokens][q_heads] or NULL, receives the
 * natural logarithm of each row's sum of exponentials.  A row that sees no key is 0, its lse -infinity.
 * max_len: an upper bound of seq_lens where the caller knows one, 0 otherwise; it decides how the work is split and
 * nothing else.  `workspace` must hold KV4_AttentionWorkspaceBytes of the same arguments (may be NULL when that is 0),
 * 16-byte aligned; contents irrelevant.  q: rows aligned to 16 bytes (strides multiples of 8 elements, where they are used).
 * Roundings.  Scores, their maxima and the sums are float32; a score is within 2^-21 of sum_d |q_d| w (code + z) (as measured,
 * with few rows to a sequence; 2^-24 with many).  A probability is rounded to fp16 (11 bits, of either sign) before it is
 * multiplied by the values; the sum of probabilities is not.  With its value's scale (1 for a vector of zeros) it keeps those bits
 * down to 2^-21 of the row's largest such product, and counts as 0 below 2^-31 of it.  out is rounded once. */
int    KV4_Attention(hipStream_t stream, const KV4_Cache* cache, const KV4_Batch* batch, KV4_Rows q, int q_heads,
                     void* out, float* lse, float scale, int window, int max_len, void* workspace,
                     size_t workspace_bytes, int dtype);
size_t KV4_AttentionWorkspaceBytes(const KV4_Cache* cache, const KV4_Batch* batch, int q_heads, int window, int max_len);

/*
 * Linear with 4-bit weights:  Y[n][m] = act( sum_k X[n][k] * scale[m][k/group] * (code[m][k] - zero[m][k/group]) + bias[m] )
 * sums in float32, one rounding to `dtype` at the end; infinities and NaN in X give what the formula gives, in their own rows of Y
 * alone.  W4_Pack lays the weights out for the kernels, once: from
 * codes uint8 [M][K] (values 0..15; higher bits are ignored), scales [M][K/group] in `dtype`, zeros uint8 [M][K/group]
 * (0..15) into `packed`, W4_PackedBytes(M, K, group) bytes, 16-byte aligned.  M is any positive number, group 32, 64 or
 * 128, K a multiple of it, at most 2^30.  `dtype` of X, Y and bias is that of the scales.  W4_PackedBytes is 0 for sizes that are
 * refused.
 * X: rows of K elements, x_stride elements apart (a multiple of 8, at least K), 16-byte aligned; Y contiguous [N][M].
 * `activation`: 0 none, 1 ReLU, 2 GELU (tanh form), as in spmm_api.h.  N from 0 to 16 * 65535.  `workspace` must hold
 * W4_WorkspaceBytes(M, N, K, group) bytes (NULL where that is 0), 16-byte aligned; contents irrelevant.
 */
size_t W4_PackedBytes(int M, int K, int group);
int    W4_Pack(hipStream_t stream, const uint8_t* codes, const void* scales, const uint8_t* zeros, int M, int K,
               int group, int dtype, void* packed);
size_t W4_WorkspaceBytes(int M, int N, int K, int group);
int    W4_Linear(hipStream_t stream, const void* packed, const void* X, int64_t x_stride, void* Y, int M, int N, int K,
                 int group, const void* bias, int activation, void* workspace, size_t workspace_bytes, int dtype);

#ifdef __cplusplus
}
#endif

#endif /* DECODE_API_H */
