/*
 * dsa_mi355x_cache.h -- C ABI of the operators around a paged MLA cache: block
 * tables and slot maps, rotary positions, cache row writes, and dense attention
 * of a batch that shares a prefix or ends with trees of drafted tokens.  Part of the same library as dsa_mi355x.h
 * and of the same conventions: device pointers, a stream, nothing allocated,
 * no synchronisation, 0 / < 0 (invalid argument, nothing enqueued) / > 0 (a
 * hipError_t) with dsa_last_error().  No reference counterpart: the reference
 * takes its cache, rotated and contiguous, as given (README.md:19-21,
 * dsa/api.py:30-33).
 */
#ifndef DSA_MI355X_CACHE_H
#define DSA_MI355X_CACHE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * One step of a paged cache: sequence b holds lengths[b] tokens and gets
 * new_tokens[b] more (negative counts as 0).  It takes
 *   need_b = ceil((lengths[b] + new_tokens[b]) / block_size) - ceil(lengths[b] / block_size)
 * blocks (as many of them as its table row has room for), in the order of the
 * sequences, from the front of free_blocks: entry ceil(lengths[b] / block_size)
 * + j of its row becomes free_blocks[need_0 + .. + need_{b-1} + j], or -1 past
 * the list's end.  No other entry is written.
 *
 *   block_table [B, max_blocks] int32, updated in place
 *   lengths, new_tokens [B] int32;  free_blocks [num_free] int32
 *   slots, positions [max_tokens] int32: of the new tokens, sequence after
 *           sequence: the token's position in its sequence and its cache row
 *           block_table[b, position / block_size] * block_size + position %
 *           block_size, or -1 where there is no such entry or it is negative.
 *           Entries behind the last token: slot -1, position 0; tokens past
 *           max_tokens are left out.
 *   starts  [B + 1] int32: first token of each sequence, and their number
 *   totals  [B] int32: lengths + new_tokens
 *   used    [1] int32: need_0 + .. + need_{B-1}; above num_free the list was short
 * B <= DSA_TABLE_MAX_SEQUENCES.  Sums are held at 2^31 - 1.
 */
#define DSA_TABLE_MAX_SEQUENCES 4096
int dsa_extend_block_table(int32_t* block_table, const int32_t* lengths, const int32_t* new_tokens,
                           const int32_t* free_blocks, int32_t* slots, int32_t* positions, int32_t* starts,
                           int32_t* totals, int32_t* used, int B, int max_blocks, int block_size, int num_free,
                           int max_tokens, void* stream);

/*
 * Rotary positions.  For every token (a, t) and head h the pairs i < dim / 2 of
 * x[a, t, h, start .. start + dim) turn by the angle positions[a, t] *
 * frequencies[i]:
 *   y0 = magnitude * (x0 cos - x1 sin),  y1 = magnitude * (x0 sin + x1 cos)
 * where pair i is elements (2 i, 2 i + 1) (interleaved) or (i, i + dim / 2) of
 * the rotated part.  transposed: by the opposite angle, the gradient for x.
 * The angle is formed in 64 bits and reduced to a turn before the 32-bit sine
 * and cosine; the products are 32-bit, rounded once to x's type.  The rest of
 * each head is copied (out == x, with the same strides: left as it is).
 * heads * width <= 2^31.
 */
#define DSA_BF16 0
#define DSA_F16 1
#define DSA_F32 2
#define DSA_ROTARY_MAX_DIM 512
typedef struct dsa_rotary_args {
    const void* x;              /* [groups, tokens, heads, width], last stride 1 */
    void* out;                  /* the same shape; x itself, or no overlap with it */
    const void* positions;      /* [groups, tokens] int32, or int64 */
    const double* frequencies;  /* [dim / 2], radians a position */
    int64_t groups, tokens;
    int64_t x_stride[3], out_stride[3]; /* elements: group, token, head */
    int32_t heads, width, start, dim;
    int32_t dtype;              /* DSA_BF16, DSA_F16, DSA_F32 */
    int32_t positions_64, interleaved, transposed;
    float magnitude;
    int32_t reserved;           /* zero */
} dsa_rotary_args;
int dsa_rotary(const dsa_rotary_args* args, void* stream);

/*
 * New rows into a cache: row slots[i] of the cache becomes token i's kv and
 * (rotated, where frequencies is given: as dsa_rotary over dim 64) k_rope.  A
 * token whose slot lies outside [0, cache_rows) is left out.  No row may be named
 * twice: nothing orders the two tokens' writes, and the row holds parts of
 * either.  kv and k_rope must not lie in rows that the call writes.
 *
 *   kv [tokens, 512] bf16, kv_stride elements apart (a multiple of 8, 16-byte
 *   aligned); k_rope [tokens, 64] bf16, rope_stride apart (a multiple of 2,
 *   4-byte aligned)
 *   DSA_KV_BF16: cache [cache_rows, 512], rope_cache [cache_rows, 64] bf16
 *   DSA_KV_FP8:  cache [cache_rows] 656-byte rows (dsa_fwd_options.kv_format),
 *   rope_cache NULL; pow2_scales: each 128-wide block's scale is the least power
 *   of two >= amax / 448, else amax / 448
 */
typedef struct dsa_write_args {
    const uint16_t* kv;
    const uint16_t* k_rope;
    const int32_t* slots;
    const void* positions;      /* [tokens] int32 or int64; unused without frequencies */
    const double* frequencies;  /* [32], or NULL: k_rope is written as it is */
    void* cache;
    uint16_t* rope_cache;
    int64_t tokens, cache_rows, kv_stride, rope_stride;
    int32_t kv_format, pow2_scales, positions_64, interleaved;
    float magnitude;
    int32_t reserved;           /* zero */
} dsa_write_args;
int dsa_write_kv_rows(const dsa_write_args* args, void* stream);

/*
 * Dense attention of a batch whose sequences share their first `prefix` rows.
 * With the rows as dsa_fwd's kv and k_rope (contiguous, paged or fp8, as in
 * dsa_fwd_options), for query t of sequence b and head h:
 *
 *   score_j = (q[b,t,h,:] . kv_j + q_rope[b,t,h,:] . k_rope_j) * scale     j < lengths[b,t]
 *   max = max_j score_j;  sum = sum_j exp(score_j - max);  out = sum_j exp(score_j - max) kv_j / sum
 *
 * where row j is row j of sequence 0 for j < prefix, and of sequence b from
 * there on: the prefix is read, and its products formed, for the whole batch
 * at once.  A row whose block entry lies outside [0, num_blocks) is masked.  A
 * query with no row left gives out 0, max -inf, sum 0.  Any other takes
 * infinities and NaN as the formulas do: a score of +inf or NaN, or none above
 * -inf, makes its sum and out NaN (max: NaN where a score is and none is +inf); a
 * score of -inf beside finite ones is a weight of 0, whose product with an
 * infinite element of kv_j makes that column of out NaN.  Rows a query does not
 * see, whatever their bits, do not touch its result.
 *
 *   q [B, SQ, H, 512], q_rope [B, SQ, H, 64] bf16, H a multiple of 16
 *   lengths [B, SQ] int32: rows each query sees, clamped to [0, L]
 *   out [B, SQ, H, 512] bf16, out_max / out_sum [B, 1, SQ, H] fp32
 *   workspace: at least dsa_fwd_shared_ws_bytes bytes, 256-byte aligned, any
 *   contents; calls that can overlap need one each
 * Probabilities are rounded to bf16 before the second product, sums and
 * statistics are fp32; the output is finite for max|kv| < 2^38.  L and
 * num_blocks * block_size below 2^25, B * SQ * H at most 2^30.
 */
typedef struct dsa_shared_args {
    const uint16_t* q;
    const void* kv;             /* [B, L, 512] bf16 or [B, L] fp8 rows; a pool when paged */
    const uint16_t* q_rope;
    const uint16_t* k_rope;     /* [B, L, 64] bf16 or a pool; unused with fp8 rows */
    const int32_t* lengths;
    const int32_t* block_table; /* [B, max_blocks], or NULL */
    uint16_t* out;
    float* out_max;
    float* out_sum;
    void* workspace;
    int64_t workspace_bytes;
    int32_t B, SQ, H, L, prefix;
    int32_t block_size, max_blocks, num_blocks; /* paged: L = max_blocks * block_size */
    int32_t kv_format;          /* DSA_KV_BF16, DSA_KV_FP8 */
    int32_t num_cus;            /* compute units to plan for, at most 4096; 0: the device's */
    float scale;                /* 0: 1/24 */
    int32_t reserved;           /* zero */
} dsa_shared_args;
/* < 0: the sizes are refused (dsa_last_error).  Reads no pointer of args. */
int64_t dsa_fwd_shared_ws_bytes(const dsa_shared_args* args);
int dsa_fwd_shared(const dsa_shared_args* args, void* stream);

/*
 * Drafted tokens behind B sequences, SQ each: token t follows token
 * parents[b, t] < t, or the sequence's last row (-1).  Any other value, or an
 * ancestor with one, makes it no token (padding).
 *
 *   parents [B, SQ], lengths [B] int32
 *   tree    [B, SQ, ceil(SQ / 32)] int32: bit j % 32 of word j / 32 is set where
 *           drafted token j is t itself or an ancestor of it; none for padding
 *   positions [B, SQ] int32: lengths[b] (negative counts as 0) + the number of t's
 *           ancestors, at most 2^31 - 1; 0 for padding
 * B <= 2^20, SQ <= 32 * DSA_TREE_MAX_WORDS.
 */
#define DSA_TREE_MAX_WORDS 64
int dsa_draft_tree(const int32_t* parents, const int32_t* lengths, int32_t* tree, int32_t* positions, int B, int SQ,
                   void* stream);

/*
 * dsa_fwd_shared where the rows a query sees end with a tree: query t of sequence
 * b sees rows [0, shared.lengths[b]) and rows shared.lengths[b] + j below L for
 * every bit j of its `words` words that is set (word j / 32, bit j % 32).
 * shared.lengths is [B] here; all else is as there (rows below the prefix are
 * sequence 0's).  dsa_fwd_tree_ws_bytes reads shared's sizes only.
 */
typedef struct dsa_tree_args {
    dsa_shared_args shared;
    const int32_t* tree;        /* [B, SQ, words] */
    int32_t words;              /* at most DSA_TREE_MAX_WORDS */
    int32_t reserved;           /* zero */
} dsa_tree_args;
int64_t dsa_fwd_tree_ws_bytes(const dsa_tree_args* args);
int dsa_fwd_tree(const dsa_tree_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DSA_MI355X_CACHE_H */
