// What the cache operators share: the cache's rows as a kernel sees them
// (dense rows or pages), the two element types, exact small divisions.
#pragma once

#include "common.hpp"

#include "../../include/slimkv/cache_ops.h"

#include <algorithm>

namespace slimkv {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// The operand types: 16-bit patterns in memory and in the MFMA operands, fp32
// in the accumulators.  mfma32 / mfma16 as the bf16 tiles of common.hpp.
template <bool F16>
struct Elem;

template <>
struct Elem<false> {
    static __device__ __forceinline__ v4f mma32(u32x4 a, u32x4 b, v4f c) { return mfma32(a, b, c); }
    static __device__ __forceinline__ v4f mma16(u32x2 a, u32x2 b, v4f c) {
        return mfma16(__builtin_bit_cast(v4s, a), __builtin_bit_cast(v4s, b), c);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16(a, b); }
    static __device__ __forceinline__ float lo(uint32_t w) { return lo_bf16(w); }
    static __device__ __forceinline__ float hi(uint32_t w) { return hi_bf16(w); }
    // either half infinite or NaN
    static __device__ __forceinline__ bool unbounded(uint32_t w) {
        return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
    }
};

template <>
struct Elem<true> {
    static __device__ __forceinline__ v4f mma32(u32x4 a, u32x4 b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
    static __device__ __forceinline__ v4f mma16(u32x2 a, u32x2 b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0,
                                                     0, 0);
    }
    // two round-to-nearest-even conversions
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_hw{a, b}, f16x2));
    }
    static __device__ __forceinline__ float lo(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[0]; }
    static __device__ __forceinline__ float hi(uint32_t w) { return (float)__builtin_bit_cast(f16x2, w)[1]; }
    static __device__ __forceinline__ bool unbounded(uint32_t w) {
        return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
    }
};

// n / d and n % d for 0 <= n < 2^31: with l = ceil(log2 d) and m = floor(2^(31
// + l) / d) + 1, m d exceeds 2^(31 + l) by at most d <= 2^l, so n m / 2^(31 +
// l) exceeds n / d by less than 1 / d and has its integer part.
struct FastDiv {
    uint32_t d, m, shift;
};

inline FastDiv fast_div(int64_t d) {
    uint32_t l = 0;
    while (((int64_t)1 << l) < d) ++l;
    return FastDiv{(uint32_t)d, (uint32_t)((((uint64_t)1 << (31 + l)) / (uint64_t)d) + 1), 31 + l};
}

__device__ __forceinline__ int quotient(int n, const FastDiv& f) { return (int)(((uint64_t)(uint32_t)n * f.m) >> f.shift); }

// A softmax scale whose fp32 image times a score of -inf stays -inf.
inline bool scale_usable(double scale) { return scale >= 1e-18 && scale <= 1e18; }

// A grid dimension's threads are counted in 32 bits by the launch.
inline bool launchable(int64_t workgroups, int64_t threads) { return workgroups <= 0xffffffff / threads; }

struct CacheView {
    const uint16_t* k; int64_t k_sb, k_sn, k_sh;
    const uint16_t* v; int64_t v_sb, v_sn, v_sh;
    const int64_t* table; int64_t t_sb, num_blocks;
    FastDiv block;
    const int32_t* lengths;
    int keys;
    int32_t* status;
};

__device__ __forceinline__ int cache_length(const CacheView& c, int64_t b) {
    return c.lengths ? max(0, min(c.lengths[b], c.keys)) : c.keys;
}

// The pool block of row `row` of sequence b: an entry outside the pool is
// reported and read as block 0, so every address stays inside the pool.
__device__ __forceinline__ int64_t cache_block(const CacheView& c, int64_t b, int row) {
    const int64_t page = table_page(c.table[b * c.t_sb + quotient(row, c.block)], c.num_blocks);
    if (page < 0) report_bad_page(c.status);
    return page < 0 ? 0 : page;
}

// Offsets of a row's first element in K and V (head 0).
struct RowAt {
    int64_t k, v;
};

template <bool PAGED>
__device__ __forceinline__ RowAt cache_row(const CacheView& c, int64_t b, int row) {
    if constexpr (PAGED) {
        const int64_t page = cache_block(c, b, row);
        const int slot = row - quotient(row, c.block) * (int)c.block.d;
        return RowAt{page * c.k_sb + slot * c.k_sn, page * c.v_sb + slot * c.v_sn};
    } else {
        return RowAt{b * c.k_sb + row * c.k_sn, b * c.v_sb + row * c.v_sn};
    }
}

// Checks of a cache and its kernel view; `what` names the call.
int cache_view(const slimkv_cache_rows& rows, int64_t batch, int64_t kv_heads, int64_t head_dim, bool need_v,
               const char* what, CacheView* view);
// Strides read for 16-byte pieces: multiples of 8 where the dimension has more than one element.
bool rows_aligned(const void* p, std::initializer_list<std::pair<int64_t, int64_t>> size_and_stride);

constexpr int kXcdCount = 8;

// Values that are the same on every lane, in scalar registers: what follows
// from them stays on the scalar unit, and buffer resources need no loop over
// lanes.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
    return (int64_t)((uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32 | (uint32_t)uniform((int)x));
}

// The dealing of a ragged batch to workgroups.  An item is one KV head of one
// sequence: its cache rows in tiles of `rows`, and `extra` tiles after them.  The
// tiles of all items lie in a row, sequence by sequence and head by head, and
// are dealt to at most `runs` workgroups in equal runs, whatever the lengths
// are.  The host keeps their number below 2^31.
struct Dealing {
    int B, Hk, rows, extra, runs;
};

__device__ __forceinline__ int item_tiles(const Dealing& d, int n) {
    return (int)((uint32_t)(n + d.rows - 1) / (uint32_t)d.rows) + d.extra;
}

// Tiles of all items (every lane active).
__device__ __forceinline__ int total_tiles(const CacheView& c, const Dealing& d) {
    const int lane = threadIdx.x & 63;
    int sum = 0;
    for (int b0 = 0; b0 < d.B; b0 += 64) {
        int x = b0 + lane < d.B ? item_tiles(d, cache_length(c, b0 + lane)) : 0;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) x += __shfl_xor(x, s, 64);
        sum += x;
    }
    return uniform(sum) * d.Hk;
}

// Sequence that holds tile `pos`, the position of its first tile, its tiles a
// head and its rows.
struct Place {
    int b, tiles, n, first;
};

__device__ __forceinline__ Place place_of(const CacheView& c, const Dealing& d, int pos) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int b0 = 0; b0 < d.B; b0 += 64) {
        const int n = b0 + lane < d.B ? cache_length(c, b0 + lane) : 0;
        const int x = b0 + lane < d.B ? item_tiles(d, n) : 0;
        int end = x;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int y = __shfl_up(end, s, 64);
            if (lane >= s) end += y;
        }
        end = base + end * d.Hk;
        const uint64_t past = __ballot(pos < end);
        if (past) {
            const int at = __ffsll((unsigned long long)past) - 1;
            const int tiles = uniform(__shfl(x, at, 64));
            return Place{b0 + at, tiles, uniform(__shfl(n, at, 64)), uniform(__shfl(end, at, 64)) - tiles * d.Hk};
        }
        base = uniform(__shfl(end, 63, 64));
    }
    return Place{0, 1, 0, 0};             // not reached: pos < total_tiles
}

// Workgroups that follow one another in the grid go to the XCDs in turn: the
// slots of one XCD follow one another.
__device__ __forceinline__ int slot_of_block() {
    return (int)((blockIdx.x % kXcdCount) * (gridDim.x / kXcdCount) + blockIdx.x / kXcdCount);
}

// The runs of `total` tiles: the first `extra` runs take `each` + 1 of them,
// the others `each`.
struct Deal {
    int runs, each, extra;
    __device__ __forceinline__ Deal(const Dealing& d, int total) {
        runs = min(d.runs, total);
        const int r = max(runs, 1);
        each = (uint32_t)total / (uint32_t)r;
        extra = total - each * r;
    }
    __device__ __forceinline__ int begin(int r) const { return r * each + min(r, extra); }
    __device__ __forceinline__ int run_of(int pos) const {
        const int split = extra * (each + 1);
        return pos < split ? (uint32_t)pos / (uint32_t)(each + 1) : extra + (uint32_t)(pos - split) / (uint32_t)each;
    }
};

}  // namespace slimkv
