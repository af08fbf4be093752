// Attention weight of cache rows: w[j] += sum over query rows p of one KV head
// of exp(scale q_p . k_j - lse_p), from the LSEs that the attention left.
//
// S^T = K . Q^T on the MFMA with K rows as A, held in registers for the whole
// pass (a wave owns 32 keys), and the query rows p = l * G + g as B, 64 at a
// time through LDS.  The weight of a score is one fma and one exp2 against the
// row's LSE; a lane adds the weights of its column's rows in fp32, and the 16
// columns meet once at the end, so nothing is divided, rescaled or atomic.
//
// A workgroup owns (sequence, KV head, 128 keys); where these do not fill the
// CUs the query rows are split as well and the parts are added by a second
// kernel in order.

#include "cache.hpp"

namespace slimkv {

namespace {

constexpr int kWaveKeys = 32;                     // keys a wave owns
constexpr int kBlockKeys = 4 * kWaveKeys;
constexpr int kRows = 64;                         // query rows per LDS tile

struct WeightsParams {
    CacheView c;
    const uint16_t* q; int64_t q_sb, q_sl, q_sh;
    const float* lse; int64_t l_sb, l_sh, l_sl;
    const float* previous; int64_t p_sb, p_sh;
    float* out; int64_t w_sb, w_sh;
    int B, L, Hq, Hk, causal;
    FastDiv G;
    int M, splits, blocks;                        // M = L * G query rows; blocks of keys a (sequence, head)
    float scale_log2;
    float* part;                                  // [splits][B][Hk][keys]
};

// Query rows row0 .. row0 + 63: operand, LSE in log2 and the last key each
// row sees (-1: none).
template <int D>
struct QueryTile {
    uint16_t q[kRows * (D + 16)];
    float lse[kRows];
    int last[kRows];
};

template <int D, bool F16, bool PAGED>
__global__ void __launch_bounds__(256) weights_kernel(WeightsParams p) {
    using E = Elem<F16>;
    constexpr int KS = D / 32, P = D / 8, KR = D / 32, kStride = D + 16;
    __shared__ __attribute__((aligned(16))) QueryTile<D> tiles[2];
    const int64_t item = blockIdx.x / p.blocks;
    const int64_t b = item / p.Hk;
    const int h = (int)(item % p.Hk);
    const int k0 = (int)(blockIdx.x % p.blocks) * kBlockKeys;
    const int n = cache_length(p.c, b);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int kw = k0 + wave * kWaveKeys;

    // query tiles of this split that see a key of the block
    const int tiles_all = (p.M + kRows - 1) / kRows;
    int t0 = (int)((int64_t)blockIdx.y * tiles_all / p.splits);
    const int t1 = k0 < n ? (int)((int64_t)(blockIdx.y + 1) * tiles_all / p.splits) : t0;
    if (p.causal && k0 < n) {
        const int64_t first = (int64_t)max(0, k0 - n + p.L) * p.G.d;      // the first row that sees key k0
        t0 = (int)max<int64_t>(t0, min<int64_t>(first / kRows, t1));
    }

    v4f acc[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
    if (t0 < t1) {
        u32x4 kr[2][KS];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            const RowAt at = cache_row<PAGED>(p.c, b, min(kw + 16 * mt + col, n - 1));
            const uint16_t* src = p.c.k + at.k + h * p.c.k_sh + 8 * grp;
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) kr[mt][kk] = *reinterpret_cast<const u32x4*>(src + 32 * kk);
        }
        u32x4 qr[KR];
        float lse_r;
        int last_r;
        const int kq = threadIdx.x / P, cp = 8 * (threadIdx.x % P);
        auto load = [&](int t) {
#pragma unroll
            for (int r = 0; r < KR; ++r) {
                const int row = min(t * kRows + kq + (256 / P) * r, p.M - 1);
                const int l = quotient(row, p.G), g = row - l * (int)p.G.d;
                qr[r] = *reinterpret_cast<const u32x4*>(p.q + b * p.q_sb + l * p.q_sl +
                                                        (int64_t)(h * (int)p.G.d + g) * p.q_sh + cp);
            }
            const int mine = t * kRows + (threadIdx.x & (kRows - 1)), row = min(mine, p.M - 1);
            const int l = quotient(row, p.G), g = row - l * (int)p.G.d;
            const float x = p.lse[b * p.l_sb + (int64_t)(h * (int)p.G.d + g) * p.l_sh + l * p.l_sl];
            lse_r = x * kLog2e;
            last_r = mine < p.M && x != kNegInf ? (p.causal ? n - p.L + l : n - 1) : -1;
        };
        auto store = [&](QueryTile<D>& t) {
#pragma unroll
            for (int r = 0; r < KR; ++r)
                *reinterpret_cast<u32x4*>(t.q + (kq + (256 / P) * r) * kStride + cp) = qr[r];
            if (threadIdx.x < kRows) {
                t.lse[threadIdx.x] = lse_r;
                t.last[threadIdx.x] = last_r;
            }
        };
        load(t0);
        store(tiles[t0 & 1]);
        if (t0 + 1 < t1) load(t0 + 1);
        __syncthreads();
        for (int t = t0; t < t1; ++t) {
            const QueryTile<D>& w = tiles[t & 1];
#pragma unroll
            for (int nt = 0; nt < kRows / 16; ++nt) {
                if (t * kRows + 16 * nt >= p.M) break;
                v4f s[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) {
                    const u32x4 x = *reinterpret_cast<const u32x4*>(w.q + (16 * nt + col) * kStride + 32 * kk + 8 * grp);
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) s[mt] = E::mma32(kr[mt][kk], x, s[mt]);
                }
                const float lse = w.lse[16 * nt + col];
                const int last = w.last[16 * nt + col] - kw - 4 * grp;
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = fast_exp2(__builtin_fmaf(s[mt][i], p.scale_log2, -lse));
                        acc[mt][i] += 16 * mt + i <= last ? x : 0.f;
                    }
            }
            if (t + 1 < t1) {
                store(tiles[(t + 1) & 1]);
                if (t + 2 < t1) load(t + 2);
            }
            __syncthreads();
        }
    }

    // over the 16 columns; lane col holds keys 4 grp + i of each 16
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int s = 1; s < 16; s <<= 1) acc[mt][i] += shfl_xor_f(acc[mt][i], s);
    if (col >= 8) return;
    const int mt = col >> 2, i = col & 3;
    float sum = 0.f;
#pragma unroll
    for (int x = 0; x < 8; ++x) sum = col == x ? acc[x >> 2][x & 3] : sum;
    const int key = kw + 16 * mt + 4 * grp + i;
    if (key >= p.c.keys) return;
    if (p.splits > 1) {
        p.part[(((int64_t)blockIdx.y * p.B + b) * p.Hk + h) * p.c.keys + key] = key < n ? sum : 0.f;
        return;
    }
    const float before = p.previous ? p.previous[b * p.p_sb + h * p.p_sh + key] : 0.f;
    p.out[b * p.w_sb + h * p.w_sh + key] = key < n ? before + sum : before;
}

__global__ void __launch_bounds__(256) weights_sum_kernel(WeightsParams p) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, all = (int64_t)p.B * p.Hk * p.c.keys;
    if (at >= all) return;
    const int64_t item = at / p.c.keys, key = at % p.c.keys, b = item / p.Hk, h = item % p.Hk;
    float sum = 0.f;
    for (int s = 0; s < p.splits; ++s) sum += p.part[s * all + at];
    const float before = p.previous ? p.previous[b * p.p_sb + h * p.p_sh + key] : 0.f;
    p.out[b * p.w_sb + h * p.w_sh + key] = key < cache_length(p.c, b) ? before + sum : before;
}

// Splits of the query rows: four workgroups a CU where the key blocks alone
// give fewer, a tile of rows at least.
int weight_splits(const slimkv_attention_weights_args* a) {
    const int64_t blocks = (a->cache.keys + kBlockKeys - 1) / kBlockKeys * a->batch * a->kv_heads;
    const int64_t tiles = (a->queries * (a->heads / a->kv_heads) + kRows - 1) / kRows;
    const int64_t want = 4 * device_cu_count();
    if (blocks <= 0 || blocks >= want) return 1;
    return (int)std::max<int64_t>(1, std::min(std::min<int64_t>(want / blocks, tiles), (int64_t)64));
}

int check_weights(const slimkv_attention_weights_args* a) {
    if (!a) return fail(SLIMKV_EINVAL, "attention weights: null pointer");
    if (a->head_dim != 64 && a->head_dim != 128)
        return fail(SLIMKV_EUNSUP, "attention weights: head_dim must be 64 or 128");
    if (a->dtype != SLIMKV_DTYPE_BF16 && a->dtype != SLIMKV_DTYPE_F16)
        return fail(SLIMKV_EUNSUP, "attention weights: element type must be bf16 or fp16");
    if (a->batch < 0 || a->batch > 65535 || a->queries < 0 || a->queries > (1 << 20) || a->heads <= 0 ||
        a->kv_heads <= 0 || a->heads % a->kv_heads || a->heads > 4096 || a->heads / a->kv_heads > 256)
        return fail(SLIMKV_EINVAL, "attention weights: invalid sizes");
    if (!(a->scale > 0.0)) return fail(SLIMKV_EINVAL, "attention weights: the softmax scale must be positive");
    if (a->cache.keys < 0 || a->cache.keys > ((int64_t)1 << 30))
        return fail(SLIMKV_EINVAL, "attention weights: invalid cache length");
    return SLIMKV_OK;
}

template <int D, bool F16>
void launch_weights(const WeightsParams& p, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)p.B * p.Hk * p.blocks), (unsigned)p.splits);
    if (p.c.table) hipLaunchKernelGGL((weights_kernel<D, F16, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((weights_kernel<D, F16, false>), grid, dim3(256), 0, st, p);
}

}  // namespace

}  // namespace slimkv

using namespace slimkv;

extern "C" size_t slimkv_attention_weights_workspace(const slimkv_attention_weights_args* a) {
    if (check_weights(a) != SLIMKV_OK) return 0;
    const int splits = weight_splits(a);
    return splits == 1 ? 16 : (size_t)splits * a->batch * a->kv_heads * a->cache.keys * sizeof(float);
}

extern "C" int slimkv_attention_weights(const slimkv_attention_weights_args* a, void* workspace,
                                        size_t workspace_bytes, void* stream) {
    const int code = check_weights(a);
    if (code != SLIMKV_OK) return code;
    if (a->batch == 0 || a->cache.keys == 0) return SLIMKV_OK;
    if (!a->out || (a->queries > 0 && (!a->q || !a->lse))) return fail(SLIMKV_EINVAL, "attention weights: null pointer");
    WeightsParams p{};
    const int view = cache_view(a->cache, a->batch, a->kv_heads, a->head_dim, false, "attention weights", &p.c);
    if (view != SLIMKV_OK) return view;
    if (a->queries > 0 && !rows_aligned(a->q, {{a->batch, a->q_sb}, {a->queries, a->q_sl}, {a->heads, a->q_sh}}))
        return fail(SLIMKV_EINVAL, "attention weights: query rows must start on 16-byte boundaries");
    p.q = static_cast<const uint16_t*>(a->q); p.q_sb = a->q_sb; p.q_sl = a->q_sl; p.q_sh = a->q_sh;
    p.lse = a->lse; p.l_sb = a->l_sb; p.l_sh = a->l_sh; p.l_sl = a->l_sl;
    p.previous = a->previous; p.p_sb = a->p_sb; p.p_sh = a->p_sh;
    p.out = a->out; p.w_sb = a->w_sb; p.w_sh = a->w_sh;
    p.B = (int)a->batch; p.L = (int)a->queries; p.Hq = (int)a->heads; p.Hk = (int)a->kv_heads; p.causal = a->causal ? 1 : 0;
    p.G = fast_div(a->heads / a->kv_heads);
    p.M = p.L * (int)p.G.d;
    p.splits = weight_splits(a);
    p.blocks = (p.c.keys + kBlockKeys - 1) / kBlockKeys;
    p.scale_log2 = (float)(a->scale * 1.4426950408889634);
    p.part = static_cast<float*>(workspace);
    if (p.splits > 1 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
                         workspace_bytes < slimkv_attention_weights_workspace(a)))
        return fail(SLIMKV_EWORKSPACE, "attention weights: workspace missing, misaligned or too small");
    if ((int64_t)p.B * p.Hk * p.blocks > 0x7fffffff) return fail(SLIMKV_EINVAL, "attention weights: too many rows for one call");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->head_dim == 128) {
        if (a->dtype == SLIMKV_DTYPE_F16) launch_weights<128, true>(p, st);
        else launch_weights<128, false>(p, st);
    } else {
        if (a->dtype == SLIMKV_DTYPE_F16) launch_weights<64, true>(p, st);
        else launch_weights<64, false>(p, st);
    }
    if (p.splits > 1) {
        const int64_t all = (int64_t)p.B * p.Hk * p.c.keys;
        hipLaunchKernelGGL(weights_sum_kernel, dim3((unsigned)((all + 255) / 256)), dim3(256), 0, st, p);
    }
    return check_hip(hipGetLastError(), "attention weights launch");
}
