// A cache held in 4 bits as the kernels see it (include/slimkv/quant_cache.h):
// where the parts of a page lie, and the conversions of its codes.
#pragma once

#include "cache.hpp"

#include "../../include/slimkv/quant_cache.h"

namespace slimkv {

// gfx950 converts two codes, or two elements, an instruction, each times 2^e or
// by it.  The factor is an fp32 of which only the exponent field counts (sign and
// mantissa may be anything), so a scale byte shifted to bits 23 .. 30 is one;
// byte 255 gives NaN.  Conversions to codes round to the nearest, ties to even,
// and end at 6.  (All codes, scales and 16-bit elements were compared with the
// format's definition.)
template <bool F16>
struct Codes;

template <>
struct Codes<false> {
    template <int BYTE>
    static __device__ __forceinline__ uint32_t values(uint32_t w, uint32_t scale) {
        return __builtin_bit_cast(uint32_t,
                                  __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, __uint_as_float(scale), BYTE));
    }
    template <int BYTE>
    static __device__ __forceinline__ uint32_t codes(uint32_t into, uint32_t pair, uint32_t scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(into, __builtin_bit_cast(bf16x2_hw, pair),
                                                         __uint_as_float(scale), BYTE);
    }
    static constexpr uint32_t kInfinite = 0x7f80u;
    static constexpr int kTopScale = 127 + 127 - 2;
    static __device__ __forceinline__ float value(uint32_t magnitude) { return lo_bf16(magnitude); }
};

template <>
struct Codes<true> {
    template <int BYTE>
    static __device__ __forceinline__ uint32_t values(uint32_t w, uint32_t scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, __uint_as_float(scale), BYTE));
    }
    template <int BYTE>
    static __device__ __forceinline__ uint32_t codes(uint32_t into, uint32_t pair, uint32_t scale) {
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(into, __builtin_bit_cast(f16x2, pair), __uint_as_float(scale),
                                                        BYTE);
    }
    static constexpr uint32_t kInfinite = 0x7c00u;
    static constexpr int kTopScale = 127 + 15 - 2;
    static __device__ __forceinline__ float value(uint32_t magnitude) { return Elem<true>::lo(magnitude); }
};

// Eight values of a dword of codes, as an MFMA operand takes them.
template <bool F16>
__device__ __forceinline__ u32x4 eight_values(uint32_t w, uint32_t scale) {
    using C = Codes<F16>;
    return u32x4{C::template values<0>(w, scale), C::template values<1>(w, scale), C::template values<2>(w, scale),
                 C::template values<3>(w, scale)};
}

struct PoolView {
    uint8_t* pages;
    int64_t p_sb, p_sh;
    const int64_t* table;             // NULL: sequence b is page b
    int64_t t_sb, num_pages;
    FastDiv block;
    int capacity;                     // rows of a sequence
    int32_t* status;
    // byte offsets in a page of one head: V codes, K scales, V scales
    int64_t v_at, ks_at, vs_at;
};

// Checks of a cache and its kernel view; `what` names the call.
int pool_view(const slimkv_quant_pages& pages, int64_t batch, int64_t kv_heads, int64_t head_dim, const char* what,
              PoolView* view);

}  // namespace slimkv
