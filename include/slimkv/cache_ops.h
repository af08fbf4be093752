/*
 * cache_ops.h -- C ABI of the cache operators: attention of drafted tokens over
 * a K/V cache, the attention weight its rows gather, and eviction by it.
 *
 * The entry points live in libslimkv_hip.so beside those of slimkv_hip.h and
 * follow its conventions (caller's stream, no allocation, no host
 * synchronisation, 0 or a negative SLIMKV_E* code with slimkv_last_error(),
 * strides in elements, last dimension contiguous).  They have an interface
 * number of their own: a binary built against slimkv_hip.h alone is not
 * concerned by a change here.
 *
 * Element type `dtype`: SLIMKV_DTYPE_BF16 or SLIMKV_DTYPE_F16, one for q, K, V
 * and the outputs; head_dim 64 or 128; heads a multiple of kv_heads (query
 * head j reads KV head j / (heads / kv_heads)).  Rows start on 16-byte
 * boundaries: addresses aligned, strides multiples of 8 elements (strides of
 * dimensions of one element are not read); rows of K, V and drafted tokens lie
 * [head_dim, 2^23) elements apart.
 *
 * Sizes: batch up to 65535, heads up to 4096, heads / kv_heads up to 256, drafted
 * up to 1024, keys up to 2^30.  `scale` lies in [1e-18, 1e18]: zero, negative,
 * infinite and NaN scales are SLIMKV_EINVAL, as is a call whose launches would
 * hold 2^32 threads or more.
 */
#ifndef SLIMKV_CACHE_OPS_H
#define SLIMKV_CACHE_OPS_H

#include "../slimkv_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Interface number of this header. */
int slimkv_cache_abi_version(void);

/* The rows of a cache: sequence b has rows 0 .. length_b - 1, length_b =
 * lengths[b] clamped to [0, keys] (lengths NULL: keys).
 *  table NULL:  row (b, n, h) of K at k + b * k_sb + n * k_sn + h * k_sh.
 *  table given: pages; row n of sequence b is token n % block_size of block
 *    table[b * t_sb + n / block_size], at k + block * k_sb + token * k_sn +
 *    h * k_sh (k and v point at the pool's K and V halves).  Entries follow
 *    torch's indexing rules; for one outside the pool that a row needs
 *    SLIMKV_STATUS_BAD_PAGE is stored in *status (optional) and the row's data
 *    are undefined.  keys <= t_cols * block_size. */
typedef struct slimkv_cache_rows {
    const void* k;  int64_t k_sb, k_sn, k_sh;
    const void* v;  int64_t v_sb, v_sn, v_sh;
    const int64_t* table;
    int64_t t_sb, t_cols, num_blocks, block_size;
    const int32_t* lengths;
    int64_t keys;
    int32_t* status;
} slimkv_cache_rows;

/* ------------------------------------------------------------------------
 * Attention of a tree of drafted tokens: row (b, t) attends to every row of
 * sequence b's cache and to the drafted tokens j with mask[b, t, j] != 0.
 *   out = sum_j softmax_j(scale q.k_j) v_j,  lse = log sum_j exp(scale q.k_j)
 * q [B, T, Hq, D], draft_k / draft_v [B, T, Hkv, D], mask [B, T, T] bytes (m_sb
 * 0: one for all; NULL: j <= t), out [B, T, Hq, D], lse [B, Hq, T] fp32
 * contiguous.  A row that sees nothing gives output 0 and LSE -inf; what lies
 * in rows a query does not see (infinities and NaN included) has no influence.
 * T = 1 without a mask is the decode of a single token.  Softmax weights are
 * rounded to the element type for the product with V (fp16: held 2^15 times as
 * large, so that 2^-39 of a row's largest is not lost); sums and LSE are fp32.
 * ---------------------------------------------------------------------- */
typedef struct slimkv_tree_attention_args {
    slimkv_cache_rows cache;
    const void* q;        int64_t q_sb, q_sl, q_sh;
    const void* draft_k;  int64_t dk_sb, dk_sn, dk_sh;
    const void* draft_v;  int64_t dv_sb, dv_sn, dv_sh;
    const uint8_t* mask;  int64_t m_sb, m_sl;
    void* out;            int64_t o_sb, o_sl, o_sh;
    float* lse;
    int64_t batch, drafted, heads, kv_heads, head_dim;
    double scale;
    int32_t dtype;
} slimkv_tree_attention_args;

size_t slimkv_tree_attention_workspace(const slimkv_tree_attention_args* a);
int slimkv_tree_attention(const slimkv_tree_attention_args* a, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Attention weight of cache rows, summed over queries and the query heads of
 * each KV head:
 *   out[b, h, j] = previous[b, h, j] + sum_{l, g} exp(scale q[b, l, hG + g] . k[b, j, h] - lse[b, hG + g, l])
 * for j < length_b over the query rows l that see row j: all of them, or with
 * `causal` those with j <= length_b - queries + l (the last query at the last
 * row).  A query row with LSE -inf counts nothing.  Entries from length_b on
 * take previous (0 without one).  out may be previous itself.  V is not read.
 * q [B, L, Hq, D], lse [B, Hq, L] fp32 (any strides), previous / out
 * [B, Hkv, keys] fp32.
 * ---------------------------------------------------------------------- */
typedef struct slimkv_attention_weights_args {
    slimkv_cache_rows cache;
    const void* q;          int64_t q_sb, q_sl, q_sh;
    const float* lse;       int64_t l_sb, l_sh, l_sl;
    const float* previous;  int64_t p_sb, p_sh;
    float* out;             int64_t w_sb, w_sh;
    int64_t batch, queries, heads, kv_heads, head_dim;
    double scale;
    int32_t causal;
    int32_t dtype;
} slimkv_attention_weights_args;

size_t slimkv_attention_weights_workspace(const slimkv_attention_weights_args* a);
int slimkv_attention_weights(const slimkv_attention_weights_args* a, void* workspace, size_t workspace_bytes,
                             void* stream);

/* ------------------------------------------------------------------------
 * The rows a cache keeps: of sequence b's n rows (lengths as above) the first
 * `sink`, the last `recent` and, of those between, the heaviest by weight
 * until `keep` rows are held (all n of them when n <= keep).  Equal weights:
 * the lower index first; NaN ranks below every number.  rows [B, H, keep]
 * int32 contiguous, ascending, -1 past the count; counts [B] = min(n, keep).
 * weights [B, H, keys] fp32.  sink + recent <= keep.
 * ---------------------------------------------------------------------- */
typedef struct slimkv_select_rows_args {
    const float* weights;  int64_t w_sb, w_sh;
    const int32_t* lengths;
    int32_t* rows;
    int32_t* counts;
    int64_t batch, heads, keys, keep, sink, recent;
} slimkv_select_rows_args;

size_t slimkv_select_rows_workspace(const slimkv_select_rows_args* a);
int slimkv_select_rows(const slimkv_select_rows_args* a, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * Moves chosen rows of a cache to its front.  Row i < counts[b] (clamped to
 * [0, keep]) of sequence b and KV head h comes from row rows[b, h, i] (r_sh 0:
 * one choice for all heads).  cache.lengths is not read.
 *  in_place 0: into out_k / out_v [B, keep, Hkv, D]; rows from counts[b] on are
 *    zero.  Rows may repeat and come in any order.
 *  in_place 1: within the cache (dense or pages, out_k / out_v unused); each
 *    choice strictly ascending, rows from counts[b] on stay as they are.  K and
 *    V of every sequence and head, and the weights, lie apart; no two sequences
 *    share a page that one of them writes.  Strides of 0 over sequences or heads
 *    (t_sb among them), and k = v, are refused.
 * weights (optional) [B, weight_heads, weight_keys] fp32 move along into
 * out_weights [B, weight_heads, keep], zero from counts[b] on; in place within
 * weights, whose entries from counts[b] on become zero.  weight_heads is the
 * head count of `rows` (1 or kv_heads), or 0 without weights.
 * A row outside [0, keys) (in place: or not above the one before) moves
 * nothing, gives a zero row out of place, and stores SLIMKV_STATUS_BAD_SLOT;
 * a bad page entry likewise with SLIMKV_STATUS_BAD_PAGE.
 * ---------------------------------------------------------------------- */
typedef struct slimkv_compact_rows_args {
    slimkv_cache_rows cache;
    const int32_t* rows;  int64_t r_sb, r_sh;
    const int32_t* counts;
    void* out_k;          int64_t ok_sb, ok_sn, ok_sh;
    void* out_v;          int64_t ov_sb, ov_sn, ov_sh;
    float* weights;       int64_t w_sb, w_sh;
    float* out_weights;   int64_t ow_sb, ow_sh;
    int64_t weight_heads, weight_keys;
    int64_t batch, kv_heads, head_dim, keep;
    int32_t in_place;
    int32_t dtype;
} slimkv_compact_rows_args;

int slimkv_compact_rows(const slimkv_compact_rows_args* a, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SLIMKV_CACHE_OPS_H */
