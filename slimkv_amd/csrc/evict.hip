// Eviction from a cache: the rows to keep by weight, and their move.
//
// select: a radix selection.  fp32 weights map to unsigned integers in their
// order (NaN to 0), the rows between the first `sink` and the last `recent`
// are ranked by them, and four passes over 8 bits each find the weight of the
// last row kept and how many rows of exactly that weight fit.  Two more passes
// count and write the kept rows in ascending order.  All counts are integers,
// so the result does not depend on the order of the LDS atomics.
//
// compact: bytes moved.  Out of place a lane moves 16 bytes of K and V of one
// row; in place a workgroup takes a 64-byte column of one head's K or V and
// walks the kept rows in order, reading a run of them before it writes them:
// row i comes from a row not below i, and later rows come from above.

#include "cache.hpp"

namespace slimkv {

namespace {

constexpr int kSelectThreads = 1024;

struct SelectParams {
    const float* weights; int64_t w_sb, w_sh;
    const int32_t* lengths;
    int32_t* rows;
    int32_t* counts;
    int H, keys, keep, sink, recent;
};

// Order-preserving image of a weight: -0 as +0, NaN below everything.
__device__ __forceinline__ uint32_t rank_of(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int lanes_below(uint64_t mask, int lane) {
    return __popcll(mask & (((uint64_t)1 << lane) - 1));
}

__global__ void __launch_bounds__(kSelectThreads) select_kernel(SelectParams p) {
    constexpr int kWaves = kSelectThreads / 64;
    __shared__ uint32_t hist[256];
    __shared__ uint32_t found[2];                        // chosen bin, rows of the bins above it
    __shared__ int above_w[kWaves], equal_w[kWaves];
    const int64_t b = blockIdx.x / p.H, h = blockIdx.x % p.H;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = p.lengths ? max(0, min(p.lengths[b], p.keys)) : p.keys;
    int32_t* rows = p.rows + (int64_t)blockIdx.x * p.keep;
    const int count = min(n, p.keep);
    if (h == 0 && tid == 0) p.counts[b] = count;
    for (int i = count + tid; i < p.keep; i += kSelectThreads) rows[i] = -1;
    if (n <= p.keep) {
        for (int i = tid; i < n; i += kSelectThreads) rows[i] = i;
        return;
    }
    for (int i = tid; i < p.sink; i += kSelectThreads) rows[i] = i;
    for (int i = tid; i < p.recent; i += kSelectThreads) rows[p.keep - p.recent + i] = n - p.recent + i;
    const int need = p.keep - p.sink - p.recent, first = p.sink, last = n - p.recent;
    if (need == 0) return;
    const float* w = p.weights + b * p.w_sb + h * p.w_sh;

    uint32_t prefix = 0, mask = 0;
    int left = need;                                     // rows to take among those that match the prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int i = first + tid; i < last; i += kSelectThreads) {
            const uint32_t u = rank_of(w[i]);
            if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & 255], 1u);
        }
        __syncthreads();
        if (wave == 0) {                                 // bins from the top, four a lane
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) sum += c[x] = hist[255 - (4 * lane + x)];
            uint32_t upto = sum;
#pragma unroll
            for (int s = 1; s < 64; s <<= 1) {
                const uint32_t y = __shfl_up(upto, s, 64);
                if (lane >= s) upto += y;
            }
            uint32_t before = upto - sum;
            if (before < (uint32_t)left && upto >= (uint32_t)left) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    if (before < (uint32_t)left && before + c[x] >= (uint32_t)left) {
                        found[0] = 255 - (4 * lane + x);
                        found[1] = before;
                    }
                    before += c[x];
                }
            }
        }
        __syncthreads();
        prefix |= found[0] << shift;
        mask |= 255u << shift;
        left -= (int)found[1];
        __syncthreads();
    }

    // the rows above the prefix and the first `left` equal to it; a wave owns a
    // contiguous part
    const int span = last - first, part = ((span + kWaves - 1) / kWaves + 63) / 64 * 64;
    const int from = first + wave * part, to = min(last, from + part);
    int above = 0, equal = 0;
    for (int i0 = from; i0 < to; i0 += 64) {
        const int i = i0 + lane;
        const uint32_t u = i < to ? rank_of(w[i]) : 0u;
        above += __popcll(__ballot(i < to && u > prefix));
        equal += __popcll(__ballot(i < to && u == prefix));
    }
    if (lane == 0) {
        above_w[wave] = above;
        equal_w[wave] = equal;
    }
    __syncthreads();
    int taken = 0, same = 0;
    for (int x = 0; x < wave; ++x) {
        taken += above_w[x] + min(equal_w[x], max(0, left - same));
        same += equal_w[x];
    }
    int32_t* dst = rows + p.sink + taken;
    for (int i0 = from; i0 < to; i0 += 64) {
        const int i = i0 + lane;
        const uint32_t u = i < to ? rank_of(w[i]) : 0u;
        const uint64_t eq = __ballot(i < to && u == prefix);
        const bool take = i < to && (u > prefix || (u == prefix && same + lanes_below(eq, lane) < left));
        const uint64_t all = __ballot(take);
        if (take) dst[lanes_below(all, lane)] = i;
        dst += __popcll(all);
        same += __popcll(eq);
    }
}

struct CompactParams {
    CacheView c;
    const int32_t* rows; int64_t r_sb, r_sh;
    const int32_t* counts;
    uint16_t* ok; int64_t ok_sb, ok_sn, ok_sh;
    uint16_t* ov; int64_t ov_sb, ov_sn, ov_sh;
    float* weights; int64_t w_sb, w_sh;
    float* ow; int64_t ow_sb, ow_sh;
    int Hw, wkeys, B, Hk, D, keep;
    int move_blocks, weight_blocks;               // workgroups a sequence: K/V rows, weights
};

__device__ __forceinline__ int kept_count(const CompactParams& p, int64_t b) {
    return max(0, min(p.counts[b], p.keep));
}

__device__ __forceinline__ void report_bad_row(int32_t* status) {
    if (status) *status = SLIMKV_STATUS_BAD_SLOT;
}

// blockIdx.y is the sequence; the first move_blocks workgroups move K and V,
// D / 8 lanes a (row, head), the others the weights.
template <bool PAGED>
__global__ void __launch_bounds__(256) compact_kernel(CompactParams p) {
    const int64_t b = blockIdx.y;
    const int count = kept_count(p, b);
    if ((int)blockIdx.x >= p.move_blocks) {
        const int64_t at = (int64_t)(blockIdx.x - p.move_blocks) * 256 + threadIdx.x;
        if (at >= (int64_t)p.Hw * p.keep) return;
        const int h = (int)(at / p.keep), i = (int)(at % p.keep);
        float x = 0.f;
        if (i < count) {
            const int row = p.rows[b * p.r_sb + h * p.r_sh + i];
            if (row >= 0 && row < p.wkeys) x = p.weights[b * p.w_sb + h * p.w_sh + row];
            else report_bad_row(p.c.status);
        }
        p.ow[b * p.ow_sb + h * p.ow_sh + i] = x;
        return;
    }
    const int lanes = p.D / 8, d = 8 * (threadIdx.x % lanes);
    const int64_t item = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
    if (item >= (int64_t)p.keep * p.Hk) return;
    const int i = (int)(item / p.Hk), h = (int)(item % p.Hk);
    u32x4 k = {0u, 0u, 0u, 0u}, v = {0u, 0u, 0u, 0u};
    if (i < count) {
        const int row = p.rows[b * p.r_sb + h * p.r_sh + i];
        if (row < 0 || row >= p.c.keys) {
            report_bad_row(p.c.status);
        } else {
            bool good = true;
            if constexpr (PAGED) {
                good = table_page(p.c.table[b * p.c.t_sb + quotient(row, p.c.block)], p.c.num_blocks) >= 0;
                if (!good) report_bad_page(p.c.status);
            }
            if (good) {
                const RowAt at = cache_row<PAGED>(p.c, b, row);
                k = *reinterpret_cast<const u32x4*>(p.c.k + at.k + h * p.c.k_sh + d);
                v = *reinterpret_cast<const u32x4*>(p.c.v + at.v + h * p.c.v_sh + d);
            }
        }
    }
    *reinterpret_cast<u32x4*>(p.ok + b * p.ok_sb + i * p.ok_sn + h * p.ok_sh + d) = k;
    *reinterpret_cast<u32x4*>(p.ov + b * p.ov_sb + i * p.ov_sn + h * p.ov_sh + d) = v;
}

// In place: blockIdx = ((sequence, KV head), K or V, 32-column part), then the
// weights' workgroups.  256 threads move 64 rows of 64 bytes a step.
template <bool PAGED>
__global__ void __launch_bounds__(256) compact_in_place_kernel(CompactParams p) {
    const int cols = p.D / 32, per_head = 2 * cols;
    const int64_t b = blockIdx.y;
    const int count = kept_count(p, b);
    if ((int)blockIdx.x >= p.move_blocks) {
        const int h = (int)blockIdx.x - p.move_blocks;
        float* w = p.weights + b * p.w_sb + h * p.w_sh;
        const int32_t* rows = p.rows + b * p.r_sb + h * p.r_sh;
        for (int i0 = 0; i0 < count; i0 += 256) {
            const int i = i0 + threadIdx.x;
            const int row = i < count ? rows[i] : -1;
            const int prior = i > 0 && i < count ? rows[i - 1] : -1;
            const bool good = i < count && row > prior && row >= i && row < p.wkeys;
            if (i < count && !good) report_bad_row(p.c.status);
            const float x = good ? w[row] : 0.f;
            __syncthreads();
            if (good) w[i] = x;
            __syncthreads();
        }
        for (int i = count + threadIdx.x; i < p.wkeys; i += 256) w[i] = 0.f;
        return;
    }
    const int h = (int)blockIdx.x / per_head, rest = (int)blockIdx.x % per_head;
    const int kind = rest / cols, d = 32 * (rest % cols) + 8 * (threadIdx.x & 3);
    const int32_t* rows = p.rows + b * p.r_sb + h * p.r_sh;
    uint16_t* base = const_cast<uint16_t*>(kind ? p.c.v + h * p.c.v_sh : p.c.k + h * p.c.k_sh) + d;
    for (int i0 = 0; i0 < count; i0 += 64) {
        const int i = i0 + (threadIdx.x >> 2);
        const int row = i < count ? rows[i] : -1;
        const int prior = i > 0 && i < count ? rows[i - 1] : -1;
        bool good = i < count && row > prior && row >= i && row < p.c.keys;
        if (i < count && !good) report_bad_row(p.c.status);
        uint16_t *src = base, *dst = base;
        if (good) {
            if constexpr (PAGED) {
                const int64_t* table = p.c.table + b * p.c.t_sb;
                if (table_page(table[quotient(row, p.c.block)], p.c.num_blocks) < 0 ||
                    table_page(table[quotient(i, p.c.block)], p.c.num_blocks) < 0) {
                    report_bad_page(p.c.status);
                    good = false;
                }
            }
        }
        if (good) {
            const RowAt from = cache_row<PAGED>(p.c, b, row), to = cache_row<PAGED>(p.c, b, i);
            src = base + (kind ? from.v : from.k);
            dst = base + (kind ? to.v : to.k);
        }
        u32x4 x = {0u, 0u, 0u, 0u};
        if (good && row != i) x = *reinterpret_cast<const u32x4*>(src);
        __syncthreads();                       // the step's rows are read
        if (good && row != i) *reinterpret_cast<u32x4*>(dst) = x;
        __syncthreads();                       // and written before the next step reads
    }
}

}  // namespace

}  // namespace slimkv

using namespace slimkv;

namespace {

int check_select(const slimkv_select_rows_args* a) {
    if (!a) return fail(SLIMKV_EINVAL, "select rows: null pointer");
    if (a->batch < 0 || a->heads <= 0 || a->keys < 0 || a->keys > ((int64_t)1 << 30) || a->keep <= 0 ||
        a->keep > ((int64_t)1 << 30) || a->sink < 0 || a->recent < 0 || a->batch * a->heads > 0x7fffffff || a->batch > 0x7fffffff)
        return fail(SLIMKV_EINVAL, "select rows: invalid sizes");
    if (a->sink + a->recent > a->keep)
        return fail(SLIMKV_EINVAL, "select rows: the first and the recent rows exceed the rows kept");
    return SLIMKV_OK;
}

}  // namespace

extern "C" size_t slimkv_select_rows_workspace(const slimkv_select_rows_args* a) {
    return check_select(a) == SLIMKV_OK ? 16 : 0;
}

extern "C" int slimkv_select_rows(const slimkv_select_rows_args* a, void* workspace, size_t workspace_bytes,
                                  void* stream) {
    const int code = check_select(a);
    if (code != SLIMKV_OK) return code;
    (void)workspace;
    (void)workspace_bytes;
    if (a->batch == 0) return SLIMKV_OK;
    if ((!a->weights && a->keys > 0) || !a->rows || !a->counts) return fail(SLIMKV_EINVAL, "select rows: null pointer");
    SelectParams p{};
    p.weights = a->weights; p.w_sb = a->w_sb; p.w_sh = a->w_sh;
    p.lengths = a->lengths; p.rows = a->rows; p.counts = a->counts;
    p.H = (int)a->heads; p.keys = (int)a->keys; p.keep = (int)a->keep; p.sink = (int)a->sink; p.recent = (int)a->recent;
    hipLaunchKernelGGL(select_kernel, dim3((unsigned)(a->batch * a->heads)), dim3(kSelectThreads), 0,
                       static_cast<hipStream_t>(stream), p);
    return check_hip(hipGetLastError(), "select rows launch");
}

extern "C" int slimkv_compact_rows(const slimkv_compact_rows_args* a, void* stream) {
    if (!a) return fail(SLIMKV_EINVAL, "compact rows: null pointer");
    if (a->head_dim != 64 && a->head_dim != 128)
        return fail(SLIMKV_EUNSUP, "compact rows: head_dim must be 64 or 128");
    if (a->dtype != SLIMKV_DTYPE_BF16 && a->dtype != SLIMKV_DTYPE_F16)
        return fail(SLIMKV_EUNSUP, "compact rows: element type must be bf16 or fp16");
    if (a->batch < 0 || a->batch > 65535 || a->kv_heads <= 0 || a->kv_heads > 4096 || a->keep < 0 ||
        a->keep > ((int64_t)1 << 30) || a->weight_keys < 0 || a->weight_keys > ((int64_t)1 << 30) ||
        (a->weights && a->weight_heads != a->kv_heads && a->weight_heads != 1))
        return fail(SLIMKV_EINVAL, "compact rows: invalid sizes");
    if (a->batch == 0 || a->keep == 0) return SLIMKV_OK;
    if (!a->rows || !a->counts || (!a->in_place && (!a->out_k || !a->out_v || (a->weights && !a->out_weights))))
        return fail(SLIMKV_EINVAL, "compact rows: null pointer");
    CompactParams p{};
    const int view = cache_view(a->cache, a->batch, a->kv_heads, a->head_dim, true, "compact rows", &p.c);
    if (view != SLIMKV_OK) return view;
    if (!a->in_place && (!rows_aligned(a->out_k, {{a->batch, a->ok_sb}, {a->keep, a->ok_sn}, {a->kv_heads, a->ok_sh}}) ||
                         !rows_aligned(a->out_v, {{a->batch, a->ov_sb}, {a->keep, a->ov_sn}, {a->kv_heads, a->ov_sh}})))
        return fail(SLIMKV_EINVAL, "compact rows: output rows must start on 16-byte boundaries");
    p.rows = a->rows; p.r_sb = a->r_sb; p.r_sh = a->r_sh; p.counts = a->counts;
    p.ok = static_cast<uint16_t*>(a->out_k); p.ok_sb = a->ok_sb; p.ok_sn = a->ok_sn; p.ok_sh = a->ok_sh;
    p.ov = static_cast<uint16_t*>(a->out_v); p.ov_sb = a->ov_sb; p.ov_sn = a->ov_sn; p.ov_sh = a->ov_sh;
    p.weights = a->weights; p.w_sb = a->w_sb; p.w_sh = a->w_sh;
    p.ow = a->out_weights; p.ow_sb = a->ow_sb; p.ow_sh = a->ow_sh;
    p.Hw = (int)a->weight_heads; p.wkeys = (int)a->weight_keys;
    p.B = (int)a->batch; p.Hk = (int)a->kv_heads; p.D = (int)a->head_dim; p.keep = (int)a->keep;
    hipStream_t st = static_cast<hipStream_t>(stream);
    int64_t move, weights;
    if (a->in_place) {
        move = a->kv_heads * 2 * (a->head_dim / 32);
        weights = a->weights ? a->weight_heads : 0;
    } else {
        const int64_t per = 256 / (a->head_dim / 8);
        move = (a->keep * a->kv_heads + per - 1) / per;
        weights = a->weights ? (a->weight_heads * a->keep + 255) / 256 : 0;
    }
    if (move + weights > 0x7fffffff) return fail(SLIMKV_EINVAL, "compact rows: too many rows for one call");
    p.move_blocks = (int)move;
    p.weight_blocks = (int)weights;
    const dim3 grid((unsigned)(move + weights), (unsigned)a->batch);
    if (a->in_place) {
        if (p.c.table) hipLaunchKernelGGL(compact_in_place_kernel<true>, grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL(compact_in_place_kernel<false>, grid, dim3(256), 0, st, p);
    } else {
        if (p.c.table) hipLaunchKernelGGL(compact_kernel<true>, grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL(compact_kernel<false>, grid, dim3(256), 0, st, p);
    }
    return check_hip(hipGetLastError(), "compact rows launch");
}
