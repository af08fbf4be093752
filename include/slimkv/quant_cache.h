/*
 * quant_cache.h -- C ABI of a K/V cache held in 4 bits and of the step around
 * it: head norms with rotation, rows written into the cache and read back,
 * attention of new tokens over it.
 *
 * The entry points live in libslimkv_hip.so beside those of slimkv_hip.h and
 * follow its conventions (caller's stream, no allocation, no host
 * synchronisation, 0 or a negative SLIMKV_E* code with slimkv_last_error(),
 * strides in elements, last dimension contiguous).  They have an interface
 * number of their own.
 *
 * Element type `dtype`: SLIMKV_DTYPE_BF16 or SLIMKV_DTYPE_F16, one for all
 * tensors of a call; head_dim 64 or 128.  Rows start on 16-byte boundaries:
 * addresses aligned, strides multiples of 8 elements (strides of dimensions of
 * one element are not read).  Sizes: batch up to 65535, heads and kv_heads up to
 * 4096.
 */
#ifndef SLIMKV_QUANT_CACHE_H
#define SLIMKV_QUANT_CACHE_H

#include "../slimkv_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Interface number of this header. */
int slimkv_quant_abi_version(void);

/* ------------------------------------------------------------------------
 * The cache.  A row of one KV head is cut into blocks of 32 elements; a block
 * shares a power of two 2^e, stored as the byte e + 127 (255: the block held an
 * infinity or NaN and reads as NaN), and holds each element as a 4-bit float
 * times 2^e: code c in 0 .. 7 stands for 0, 0.5, 1, 1.5, 2, 3, 4, 6, code 8 + c
 * for -c.  Written, e + 2 is the exponent of the block's largest magnitude, one
 * more where its mantissa is 1.75 or above (then 4 2^(e + 1) is as near as 6 2^e
 * or nearer), e within [-127, the largest exponent of the element type - 2];
 * elements go to the nearest number, ties to the even code.
 *
 * pages: a pool of num_pages pages, page p of KV head h at pages + p * p_sb + h
 * * p_sh (bytes; 16-byte aligned, strides multiples of 16).  The block_size rows
 * (a multiple of 16) of one page and head are block_size (head_dim + head_dim /
 * 16) bytes:
 *   K codes   row r at r head_dim / 2: element 2 i in the low and 2 i + 1 in the
 *             high half of byte i
 *   V codes   16 rows at a time: of row 4 g + j the elements 32 p + m (low) and
 *             32 p + 16 + m (high) in byte ((16 g + m) 4 + j) head_dim / 32 + p,
 *             m < 16: the order in which the matrix cores take V, with the keys
 *             side by side
 *   K scales, then V scales   row r at r head_dim / 32, a byte a block
 * table NULL: sequence b is page b (num_pages >= batch), rows 0 .. block_size - 1.
 * table given: row n of sequence b is row n % block_size of page table[b * t_sb
 *   + n / block_size], n < t_cols * block_size and 2^30.  Entries follow torch's
 *   indexing rules; for one outside the pool that a row needs SLIMKV_STATUS_BAD_PAGE is
 *   stored in *status (optional): that row is not written, reads as zeros, and
 *   makes an attention's results undefined.
 * ---------------------------------------------------------------------- */
typedef struct slimkv_quant_pages {
    uint8_t* pages;  int64_t p_sb, p_sh;
    const int64_t* table;
    int64_t t_sb, t_cols, num_pages, block_size;
    int32_t* status;
} slimkv_quant_pages;

/* Rows i < counts[b] (NULL: rows; clamped to [0, rows]) of k and v [B, rows,
 * Hkv, D] become rows starts[b] + i (NULL: 0 + i) of the cache.  A row outside
 * the cache is not written and stores SLIMKV_STATUS_BAD_SLOT.  Nothing else of
 * the pool changes.  Two rows of one call must not name the same place. */
typedef struct slimkv_quantize_rows_args {
    slimkv_quant_pages cache;
    const void* k;  int64_t k_sb, k_sn, k_sh;
    const void* v;  int64_t v_sb, v_sn, v_sh;
    const int32_t* starts;
    const int32_t* counts;
    int64_t batch, rows, kv_heads, head_dim;
    int32_t dtype;
} slimkv_quantize_rows_args;

int slimkv_quantize_rows(const slimkv_quantize_rows_args* a, void* stream);

/* The reverse: row i of k and v [B, rows, Hkv, D] is cache row starts[b] + i for
 * i < counts[b], zero from counts[b] on.  A row outside the cache is zero and
 * stores SLIMKV_STATUS_BAD_SLOT.  What slimkv_quantize_rows wrote from bf16 or
 * fp16 is exact in bf16; fp16 rounds numbers below 2^-22 and turns those past
 * 65504 into infinities. */
typedef struct slimkv_dequantize_rows_args {
    slimkv_quant_pages cache;
    void* k;  int64_t k_sb, k_sn, k_sh;
    void* v;  int64_t v_sb, v_sn, v_sh;
    const int32_t* starts;
    const int32_t* counts;
    int64_t batch, rows, kv_heads, head_dim;
    int32_t dtype;
} slimkv_dequantize_rows_args;

int slimkv_dequantize_rows(const slimkv_dequantize_rows_args* a, void* stream);

/* ------------------------------------------------------------------------
 * Attention of new tokens over the cache and over each other: row (b, t) attends
 * to rows 0 .. lengths[b] - 1 of sequence b (NULL: keys; clamped to [0, keys])
 * and to the drafted rows j with mask[b, t, j] != 0 (m_sb 0: one mask for all;
 * NULL: j <= t); draft_k and draft_v NULL: to the cache alone (no mask then).
 *   out = sum_j softmax_j(scale q.k_j) v_j,  lse = log sum_j exp(scale q.k_j)
 * q [B, T, Hq, D], draft_k / draft_v [B, T, Hkv, D] in the element type, out
 * [B, T, Hq, D], lse [B, Hq, T] fp32 contiguous; query head j reads KV head j /
 * (heads / kv_heads).  A row that sees nothing gives 0 and -inf; what lies behind
 * a sequence's length, or in drafted rows that a query does not see, has no
 * influence.  Cached rows enter as slimkv_dequantize_rows gives them in this
 * element type.  Softmax weights are rounded to the element type for the product
 * with V (fp16: held 2^15 times as large); sums and LSE are fp32.
 * Up to 1024 tokens, 256 query heads a KV head, 2^30 keys; scale in [1e-18,
 * 1e18]; drafted rows lie [head_dim, 2^23) elements apart.
 * ---------------------------------------------------------------------- */
typedef struct slimkv_quantized_attention_args {
    slimkv_quant_pages cache;
    const int32_t* lengths;
    int64_t keys;
    const void* q;        int64_t q_sb, q_sl, q_sh;
    const void* draft_k;  int64_t dk_sb, dk_sn, dk_sh;
    const void* draft_v;  int64_t dv_sb, dv_sn, dv_sh;
    const uint8_t* mask;  int64_t m_sb, m_sl;
    void* out;            int64_t o_sb, o_sl, o_sh;
    float* lse;
    int64_t batch, tokens, heads, kv_heads, head_dim;
    double scale;
    int32_t dtype;
} slimkv_quantized_attention_args;

/* By the sizes of the call, `keys` among them. */
size_t slimkv_quantized_attention_workspace(const slimkv_quantized_attention_args* a);
int slimkv_quantized_attention(const slimkv_quantized_attention_args* a, void* workspace, size_t workspace_bytes,
                               void* stream);

/* ------------------------------------------------------------------------
 * Queries and keys of a step or window, each head normalised and rotated:
 *   y = x / sqrt(mean(x^2) + eps) * weight    (weight NULL: y = x)
 *   out = y * cos[pos] + rotate_half(y) * sin[pos],  pos = positions[b, l]
 * rotate_half(y) = (-y[D/2:], y[:D/2]).  fp32 throughout, one rounding; a
 * normalised head's sum of squares has to lie within fp32.
 * q [B, L, Hq, D], k [B, L, Hkv, D] (kv_heads 0: queries alone), q_weight /
 * k_weight [D] in the element type or (weight_f32) fp32, cos / sin [table_rows,
 * D] fp32, positions int64 (strides pos_sb, pos_sl).  A position outside the
 * table stores SLIMKV_STATUS_BAD_SLOT in *status (optional) and its token's rows
 * are not written.  out_q may be q itself (same strides), out_k k.
 * ---------------------------------------------------------------------- */
typedef struct slimkv_norm_rope_args {
    const void* q;      int64_t q_sb, q_sl, q_sh;
    const void* k;      int64_t k_sb, k_sl, k_sh;
    const void* q_weight;
    const void* k_weight;
    const float* cos;
    const float* sin;
    int64_t table_rows;
    const int64_t* positions;  int64_t pos_sb, pos_sl;
    void* out_q;        int64_t oq_sb, oq_sl, oq_sh;
    void* out_k;        int64_t ok_sb, ok_sl, ok_sh;
    int32_t* status;
    int64_t batch, length, heads, kv_heads, head_dim;
    double eps;
    int32_t weight_f32;
    int32_t dtype;
} slimkv_norm_rope_args;

int slimkv_norm_rope(const slimkv_norm_rope_args* a, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SLIMKV_QUANT_CACHE_H */
