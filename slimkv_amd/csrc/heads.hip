// Queries and keys of a step or window, each head normalised by its root mean
// square, weighed and rotated to its position (include/slimkv/quant_cache.h):
//   y = x rsqrt(mean(x^2) + eps) w,   out = y cos + rotate_half(y) sin
// in fp32 with one rounding, in one pass over the heads.
//
// Bound by the bytes of the heads, read and written once (8192 tokens of 48 heads of
// 128, 210 MB: 40 us a call, 5.2 TB/s, a copy's rate).  D / 16 lanes hold a
// head, a lane the eight elements 8 i .. and their partners D / 2 above, so that
// the rotation stays in its registers and the norm's sum crosses D / 16 lanes.  A
// wave works on one token: its rows of the rotation tables, twice the bytes of a
// head each, are read once for all heads that the wave takes.

#include "quant.hpp"

namespace slimkv {

namespace {

struct HeadsParams {
    const char* q; int64_t q_sb, q_sl, q_sh;          // strides in bytes
    const char* k; int64_t k_sb, k_sl, k_sh;
    const void* q_weight;
    const void* k_weight;
    const float* cos;
    const float* sin;
    int64_t table_rows;
    const int64_t* positions; int64_t pos_sb, pos_sl;
    char* out_q; int64_t oq_sb, oq_sl, oq_sh;
    char* out_k; int64_t ok_sb, ok_sl, ok_sh;
    int32_t* status;
    int tokens, Hq, H;                                // all tokens; query heads; all heads
    int each;                                         // rounds of heads a wave takes
    FastDiv by_length, by_chunks;                     // chunks of heads a token is cut into
    float eps;
    int weight_f32;
};

template <int CTRL>
__device__ __forceinline__ float lane_sum(float x) {
    return x + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, true));
}

template <bool F16>
__device__ __forceinline__ void unpack(u32x4 w, float (&x)[8]) {
    using E = Elem<F16>;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[2 * e] = E::lo(w[e]);
        x[2 * e + 1] = E::hi(w[e]);
    }
}

// Eight weights from element d on.
template <bool F16>
__device__ __forceinline__ void weights_at(const void* w, int f32, int d, float (&x)[8]) {
    if (f32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = static_cast<const float*>(w)[d + e];
    } else {
        unpack<F16>(*reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(w) + d), x);
    }
}

// Rows of a call that no cache keeps until the next launch reads them go past the
// caches (FAR).
template <bool FAR>
__device__ __forceinline__ void store_row(u32x4 x, char* to) {
    if constexpr (FAR) __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(to));
    else *reinterpret_cast<u32x4*>(to) = x;
}

template <int D, bool F16, bool FAR>
__global__ void __launch_bounds__(256) norm_rope_kernel(HeadsParams p) {
    using E = Elem<F16>;
    constexpr int kLanes = D / 16, kRound = 64 / kLanes;         // lanes a head, heads a round
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int at = blockIdx.x * 4 + wave;
    const int token = quotient(at, p.by_chunks), chunk = at - token * (int)p.by_chunks.d;
    if (token >= p.tokens) return;
    const int64_t b = quotient(token, p.by_length), l = token - b * (int)p.by_length.d;
    const int64_t pos = p.positions[b * p.pos_sb + l * p.pos_sl];
    if (pos < 0 || pos >= p.table_rows) {
        if (p.status) *p.status = SLIMKV_STATUS_BAD_SLOT;
        return;
    }
    const int d = 8 * (lane % kLanes);
    float c1[8], c2[8], s1[8], s2[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        c1[e] = p.cos[pos * D + d + e];
        c2[e] = p.cos[pos * D + D / 2 + d + e];
        s1[e] = p.sin[pos * D + d + e];
        s2[e] = p.sin[pos * D + D / 2 + d + e];
    }
    for (int r = 0; r < p.each; ++r) {
        const int head = (chunk * p.each + r) * kRound + lane / kLanes;
        if (head >= p.H) return;
        const bool key = head >= p.Hq;
        const int hh = key ? head - p.Hq : head;
        const char* src = key ? p.k + b * p.k_sb + l * p.k_sl + hh * p.k_sh : p.q + b * p.q_sb + l * p.q_sl + hh * p.q_sh;
        char* dst = key ? p.out_k + b * p.ok_sb + l * p.ok_sl + hh * p.ok_sh
                        : p.out_q + b * p.oq_sb + l * p.oq_sl + hh * p.oq_sh;
        float x1[8], x2[8];
        unpack<F16>(*reinterpret_cast<const u32x4*>(src + 2 * d), x1);
        unpack<F16>(*reinterpret_cast<const u32x4*>(src + D + 2 * d), x2);
        const void* w = key ? p.k_weight : p.q_weight;
        if (w) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += x1[e] * x1[e] + x2[e] * x2[e];
            sum = lane_sum<0xb1>(sum);                           // quad_perm 1 0 3 2
            sum = lane_sum<0x4e>(sum);                           // quad_perm 2 3 0 1
            if constexpr (D == 128) sum = lane_sum<0x141>(sum);  // row_half_mirror
            const float f = 1.f / sqrtf(sum * (1.f / D) + p.eps);
            float w1[8], w2[8];
            weights_at<F16>(w, p.weight_f32, d, w1);
            weights_at<F16>(w, p.weight_f32, d + D / 2, w2);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x1[e] = x1[e] * f * w1[e];
                x2[e] = x2[e] * f * w2[e];
            }
        }
        float o1[8], o2[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            o1[e] = x1[e] * c1[e] - x2[e] * s1[e];
            o2[e] = x2[e] * c2[e] + x1[e] * s2[e];
        }
        store_row<FAR>(u32x4{E::pack(o1[0], o1[1]), E::pack(o1[2], o1[3]), E::pack(o1[4], o1[5]), E::pack(o1[6], o1[7])},
                       dst + 2 * d);
        store_row<FAR>(u32x4{E::pack(o2[0], o2[1]), E::pack(o2[2], o2[3]), E::pack(o2[4], o2[5]), E::pack(o2[6], o2[7])},
                       dst + D + 2 * d);
    }
}

}  // namespace

}  // namespace slimkv

using namespace slimkv;

extern "C" int slimkv_norm_rope(const slimkv_norm_rope_args* a, void* stream) {
    if (!a) return fail(SLIMKV_EINVAL, "norm rope: null pointer");
    if (a->head_dim != 64 && a->head_dim != 128) return fail(SLIMKV_EUNSUP, "norm rope: head_dim must be 64 or 128");
    if (a->dtype != SLIMKV_DTYPE_BF16 && a->dtype != SLIMKV_DTYPE_F16)
        return fail(SLIMKV_EUNSUP, "norm rope: element type must be bf16 or fp16");
    const int64_t B = a->batch, L = a->length, Hq = a->heads, Hk = a->kv_heads, D = a->head_dim;
    if (B < 0 || B > 65535 || L < 0 || L > ((int64_t)1 << 30) || Hq <= 0 || Hq > 4096 || Hk < 0 || Hk > 4096)
        return fail(SLIMKV_EINVAL, "norm rope: invalid sizes");
    if (!(a->eps >= 0.0 && a->eps <= 1e30)) return fail(SLIMKV_EINVAL, "norm rope: eps must lie in [0, 1e30]");
    if (B == 0 || L == 0) return SLIMKV_OK;
    if (!a->q || !a->out_q || (Hk && (!a->k || !a->out_k)) || !a->cos || !a->sin || !a->positions || a->table_rows <= 0)
        return fail(SLIMKV_EINVAL, "norm rope: null pointer or empty tables");
    if (!rows_aligned(a->q, {{B, a->q_sb}, {L, a->q_sl}, {Hq, a->q_sh}}) ||
        !rows_aligned(a->out_q, {{B, a->oq_sb}, {L, a->oq_sl}, {Hq, a->oq_sh}}) ||
        (Hk && (!rows_aligned(a->k, {{B, a->k_sb}, {L, a->k_sl}, {Hk, a->k_sh}}) ||
                !rows_aligned(a->out_k, {{B, a->ok_sb}, {L, a->ok_sl}, {Hk, a->ok_sh}}))) ||
        !rows_aligned(a->cos, {}) || !rows_aligned(a->sin, {}) || !rows_aligned(a->q_weight, {}) ||
        !rows_aligned(a->k_weight, {}))
        return fail(SLIMKV_EINVAL, "norm rope: rows, tables and weights must start on 16-byte boundaries (strides "
                                   "multiples of 8)");
    HeadsParams p{};
    p.q = static_cast<const char*>(a->q); p.q_sb = 2 * a->q_sb; p.q_sl = 2 * a->q_sl; p.q_sh = 2 * a->q_sh;
    p.k = static_cast<const char*>(a->k); p.k_sb = 2 * a->k_sb; p.k_sl = 2 * a->k_sl; p.k_sh = 2 * a->k_sh;
    p.q_weight = a->q_weight; p.k_weight = a->k_weight;
    p.cos = a->cos; p.sin = a->sin; p.table_rows = a->table_rows;
    p.positions = a->positions; p.pos_sb = a->pos_sb; p.pos_sl = a->pos_sl;
    p.out_q = static_cast<char*>(a->out_q); p.oq_sb = 2 * a->oq_sb; p.oq_sl = 2 * a->oq_sl; p.oq_sh = 2 * a->oq_sh;
    p.out_k = static_cast<char*>(a->out_k); p.ok_sb = 2 * a->ok_sb; p.ok_sl = 2 * a->ok_sl; p.ok_sh = 2 * a->ok_sh;
    p.status = a->status;
    const int64_t tokens = B * L, round = 1024 / D, rounds = (Hq + Hk + round - 1) / round;
    // Two rounds a wave where that leaves every SIMD several waves (8192 tokens of 48 heads: one round 47.7 us, two
    // 43.1, three 43.4, four 44.1).  The sides cross near the border: 10240 and 12288 rounds 14.0 / 13.5 and 15.1 / 14.2,
    // 13108 and 16384 (10 + 2 heads) 15.8 / 16.4 and 17.7 / 18.1, 16385 19.4 / 19.5, 24576 26.4 / 24.0.
    // Past the caches from 64 MB of rows on, twice the L2 (the same call 43.1 / 40.2).  By itself that is faster below as
    // well (5 MB 5.0 / 4.6, 48 MB 24.0 / 22.7), but a step writes the rows before and reads them after: with both
    // (elementwise kernels) 38 MB 51.6 / 54.3, 48 MB 57.1 / 56.8, 64 MB 77.1 / 72.6, 77 MB 89.8 / 84.2, 96 MB 103.7 / 105.7,
    // 192 MB 217.2 / 217.6, 384 MB 416 / 410.
    p.each = tokens * rounds >= 16384 ? 2 : 1;
    const int64_t chunks = (rounds + p.each - 1) / p.each, workgroups = (tokens * chunks + 3) / 4;
    // keeps tokens, and waves, below 2^31 as well
    if (!launchable(workgroups, 256)) return fail(SLIMKV_EINVAL, "norm rope: too many rows for one call");
    const bool far = tokens * (Hq + Hk) * D * 2 >= ((int64_t)64 << 20);
    p.tokens = (int)tokens; p.Hq = (int)Hq; p.H = (int)(Hq + Hk);
    p.by_length = fast_div(L); p.by_chunks = fast_div(chunks);
    p.eps = (float)a->eps; p.weight_f32 = a->weight_f32;
    const dim3 grid((unsigned)workgroups);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool f16 = a->dtype == SLIMKV_DTYPE_F16;
    void (*kernel)(HeadsParams);
    if (D == 128) {
        if (f16) kernel = far ? norm_rope_kernel<128, true, true> : norm_rope_kernel<128, true, false>;
        else kernel = far ? norm_rope_kernel<128, false, true> : norm_rope_kernel<128, false, false>;
    } else {
        if (f16) kernel = far ? norm_rope_kernel<64, true, true> : norm_rope_kernel<64, true, false>;
        else kernel = far ? norm_rope_kernel<64, false, true> : norm_rope_kernel<64, false, false>;
    }
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p);
    return check_hip(hipGetLastError(), "norm rope launch");
}
