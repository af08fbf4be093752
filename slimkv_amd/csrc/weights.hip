// Attention weight of cache rows: w[j] += sum over query rows p of one KV head
// of exp(scale q_p . k_j - lse_p), from the LSEs that the attention left.
//
// S^T = K . Q^T on the MFMA with K rows as A, held in registers for the whole
// pass, and the query rows p = l * G + g as B, 16 at a time.  The weight of a
// score is one fma and one exp2 against the row's LSE; a lane adds the weights
// of its column's rows in fp32, and the 16 columns meet once at the end, so
// nothing is divided, rescaled or atomic.
//
// Few query rows (up to 16 a KV head): bound by K's bytes.  A wave owns 32 keys
// and reads the queries where they lie; nothing is shared and nothing waits but
// for memory, and many short waves a CU keep it busy.
//
// Many: bound by the exponentials.  A wave owns 64 keys, so that a query operand
// read from LDS feeds four products (with 32 the LDS reads alone take as long
// as the products), and the query rows pass through LDS 64 at a time.  Where
// the key blocks do not fill the CUs evenly the query rows are split as well and
// the parts are added by a second kernel in order.  A 2048-query chunk over two
// sequences of up to 10240 rows takes 231 us, the last 32 queries over 32771 rows
// 25.6, a token over 16 x 8-32K rows 138 (5.0 TB/s of K).  Figures beside a choice
// compare its two sides as they were when it was made.

#include "cache.hpp"

namespace slimkv {

namespace {

constexpr int kRows = 64;                         // query rows per LDS tile

struct WeightsParams {
    CacheView c;
    const uint16_t* q; int64_t q_sb, q_sl, q_sh;
    const float* lse; int64_t l_sb, l_sh, l_sl;
    const float* previous; int64_t p_sb, p_sh;
    float* out; int64_t w_sb, w_sh;
    int B, L, Hk, causal;
    FastDiv G;
    int M, splits, blocks;                        // M = L * G query rows; blocks of keys a (sequence, head)
    float scale_log2;
    float* part;                                  // [splits][B][Hk][keys]
};

// Query row `row` (clamped to the last): its address, its LSE in log2 (rounded to
// fp32 once more, 2^-24 of it, as the scaled score is) and the last key it sees (-1:
// none, also for a row that counts nothing).
__device__ __forceinline__ const uint16_t* query_address(const WeightsParams& p, int64_t b, int h, int row) {
    const int r = min(row, p.M - 1), l = quotient(r, p.G), g = r - l * (int)p.G.d;
    return p.q + b * p.q_sb + l * p.q_sl + (int64_t)(h * (int)p.G.d + g) * p.q_sh;
}

__device__ __forceinline__ void query_stats(const WeightsParams& p, int64_t b, int h, int n, int row, float* lse, int* last) {
    const int r = min(row, p.M - 1), l = quotient(r, p.G), g = r - l * (int)p.G.d;
    const float x = p.lse[b * p.l_sb + (int64_t)(h * (int)p.G.d + g) * p.l_sh + l * p.l_sl];
    *lse = x * kLog2e;
    *last = row < p.M && x != kNegInf ? (p.causal ? n - p.L + l : n - 1) : -1;
}

// The first query row that sees key k0.
__device__ __forceinline__ int first_row(const WeightsParams& p, int n, int k0) {
    return p.causal ? (int)min<int64_t>((int64_t)max(0, k0 - n + p.L) * p.G.d, p.M) : 0;
}

template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
    return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(v), CTRL, 0xf, 0xf, true));
}

// The 16 columns' sums of 16 MT keys, MT 2 or 4: lane (col, grp) comes with its
// column's share of keys 16 mt + 4 grp + i.  Each step pairs a lane with its
// mirror image in 16, 8, 4 and 2 lanes; a pair splits the keys it still holds,
// each lane sending what the other keeps, so 4 MT - 1 additions do (and one
// more for MT 2, where two lanes end with the same key).  Lane col ends with
// key_of_column(col).
template <int MT>
__device__ __forceinline__ int key_of_column(int col) {
    const int grp = (threadIdx.x & 63) >> 4, v = MT == 4 ? col : col >> 1;
    return 16 * (v >> 2) + 4 * grp + (v & 3);
}

template <int MT>
__device__ __forceinline__ float columns_sum(const v4f (&acc)[MT]) {
    const int col = threadIdx.x & 15;
    float x[4 * MT];
#pragma unroll
    for (int v = 0; v < 4 * MT; ++v) x[v] = acc[v >> 2][v & 3];
    auto halve = [&](auto move, int half, bool upper) {
#pragma unroll
        for (int v = 0; v < 2 * MT; ++v) {
            if (v >= half) break;
            const float keep = upper ? x[v + half] : x[v], send = upper ? x[v] : x[v + half];
            x[v] = keep + move(send);
        }
    };
    halve([](float v) { return dpp_move<0x140>(v); }, 2 * MT, col & 8);                  // row mirror
    halve([](float v) { return dpp_move<0x141>(v); }, MT, col & 4);                      // half-row mirror
    halve([](float v) { return dpp_move<0x1b>(v); }, MT / 2, col & 2);                   // quad [3, 2, 1, 0]
    if constexpr (MT == 4) halve([](float v) { return dpp_move<0xb1>(v); }, 1, col & 1); // quad [1, 0, 3, 2]
    else x[0] += dpp_move<0xb1>(x[0]);
    return x[0];
}

template <int D, bool F16, bool PAGED>
__global__ void __launch_bounds__(256) weights_few_kernel(WeightsParams p) {
    using E = Elem<F16>;
    constexpr int KS = D / 32, MT = 2;
    const int rest = (int)(blockIdx.x % p.blocks), h = (int)(blockIdx.x / p.blocks % p.Hk);
    const int64_t b = blockIdx.x / p.blocks / p.Hk;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const int k0 = rest * 4 * 16 * MT + wave * 16 * MT;
    const int n = cache_length(p.c, b);
    const int key = k0 + key_of_column<MT>(col);                           // the key this lane writes
    const bool mine = (MT == 4 || !(col & 1)) && key < p.c.keys;
    float before = 0.f;
    if (p.previous && mine) before = p.previous[b * p.p_sb + h * p.p_sh + key];
    v4f acc[MT] = {};
    if (k0 < n) {
        u32x4 kr[MT][KS];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const RowAt at = cache_row<PAGED>(p.c, b, min(k0 + 16 * mt + col, n - 1));
            const uint16_t* src = p.c.k + at.k + h * p.c.k_sh + 8 * grp;
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) kr[mt][kk] = *reinterpret_cast<const u32x4*>(src + 32 * kk);
        }
        if (first_row(p, n, k0) < p.M) {
            const uint16_t* src = query_address(p, b, h, col) + 8 * grp;
            u32x4 x[KS];
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) x[kk] = *reinterpret_cast<const u32x4*>(src + 32 * kk);
            float lse;
            int last;
            query_stats(p, b, h, n, col, &lse, &last);
            last -= k0 + 4 * grp;
            v4f s[MT] = {};
#pragma unroll
            for (int kk = 0; kk < KS; ++kk)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[mt] = E::mma32(kr[mt][kk], x[kk], s[mt]);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float w = fast_exp2(__builtin_fmaf(s[mt][i], p.scale_log2, -lse));
                    acc[mt][i] += 16 * mt + i <= last ? w : 0.f;
                }
        }
    }
    const float sum = columns_sum<MT>(acc);
    if (mine) p.out[b * p.w_sb + h * p.w_sh + key] = key < n ? before + sum : before;
}

// The slot of piece c of row r is c ^ twist(r): the operand reads (16 rows, one
// piece) then spread over all banks.  With rows padded by 32 bytes instead, half
// of a 2048-query chunk's time went to bank conflicts (363 us, 294 so).
template <int D>
__device__ __forceinline__ int twist(int r) { return D == 128 ? r & 15 : (r >> 1) & 7; }

// Query rows row0 .. row0 + 63: operand, LSE in log2, the last key each row
// sees, and the least of these.
template <int D>
struct alignas(16) QueryTile {
    uint16_t q[kRows * D];                        // a row's 16-byte pieces exchanged by an XOR with its number
    float lse[kRows];
    int last[kRows];
    int least;
};

template <int D, bool F16, bool PAGED>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) weights_many_kernel(WeightsParams p) {
    using E = Elem<F16>;
    constexpr int KS = D / 32, P = D / 8, KR = D / 32, MT = 4, NT = kRows / 16;
    __shared__ __attribute__((aligned(16))) QueryTile<D> tiles[2];
    const int h = (int)(blockIdx.x % p.Hk), rest = (int)(blockIdx.x / p.Hk);
    const int64_t b = rest / p.blocks;
    const int n = cache_length(p.c, b);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int kb = (rest % p.blocks) * 4 * 16 * MT, k0 = kb + wave * 16 * MT;

    // query tiles of this split that see a key of the block
    const int tiles_all = (p.M + kRows - 1) / kRows;
    const int from = (int)((int64_t)blockIdx.y * tiles_all / p.splits), to = (int)((int64_t)(blockIdx.y + 1) * tiles_all / p.splits);
    const int t1 = kb < n ? to : from, t0 = min(t1, max(from, first_row(p, n, kb) / kRows));
    v4f acc[MT] = {};
    if (t0 < t1) {
        u32x4 kr[MT][KS];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const RowAt at = cache_row<PAGED>(p.c, b, min(k0 + 16 * mt + col, n - 1));
            const uint16_t* src = p.c.k + at.k + h * p.c.k_sh + 8 * grp;
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) kr[mt][kk] = *reinterpret_cast<const u32x4*>(src + 32 * kk);
        }
        u32x4 qr[KR];
        float lse_r;
        int last_r;
        const int kq = threadIdx.x / P, cp = 8 * (threadIdx.x % P);
        // The rows a thread loads of a tile lie 64 rows after those of the tile
        // before: 64 / G queries and 64 % G heads on.  Found anew for each tile,
        // their addresses took a third of the VALU instructions (254 us, 248 so).
        const int G = (int)p.G.d, dl = quotient(kRows, p.G), dg = kRows - dl * G;
        const uint16_t* qp[KR];
        const float* lp;
        int qg[KR], lg, ll;
        auto place = [&](int t) {
#pragma unroll
            for (int r = 0; r < KR; ++r) {
                const int row = min(t * kRows + kq + (256 / P) * r, p.M - 1), l = quotient(row, p.G);
                qg[r] = row - l * G;
                qp[r] = p.q + b * p.q_sb + l * p.q_sl + (int64_t)(h * G + qg[r]) * p.q_sh + cp;
            }
            const int row = min(t * kRows + lane, p.M - 1);
            ll = quotient(row, p.G);
            lg = row - ll * G;
            lp = p.lse + b * p.l_sb + (int64_t)(h * G + lg) * p.l_sh + ll * p.l_sl;
        };
        const int64_t q_step = dl * p.q_sl + dg * p.q_sh, q_wrap = q_step + p.q_sl - G * p.q_sh;
        const int64_t l_step = dl * p.l_sl + dg * p.l_sh, l_wrap = l_step + p.l_sl - G * p.l_sh;
        auto load = [&](int t) {
            if (t == t0 || (t + 1) * kRows > p.M) {                      // the last tile's rows are clamped
                place(t);
            } else if (dg == 0) {
#pragma unroll
                for (int r = 0; r < KR; ++r) qp[r] += q_step;
                ll += dl;
                lp += l_step;
            } else {
#pragma unroll
                for (int r = 0; r < KR; ++r) {
                    const bool wrap = qg[r] + dg >= G;
                    qp[r] += wrap ? q_wrap : q_step;
                    qg[r] += wrap ? dg - G : dg;
                }
                const bool wrap = lg + dg >= G;
                lp += wrap ? l_wrap : l_step;
                ll += dl + wrap;
                lg += wrap ? dg - G : dg;
            }
#pragma unroll
            for (int r = 0; r < KR; ++r) qr[r] = *reinterpret_cast<const u32x4*>(qp[r]);
            const float x = *lp;
            lse_r = x * kLog2e;
            last_r = t * kRows + lane < p.M && x != kNegInf ? (p.causal ? n - p.L + ll : n - 1) : -1;
        };
        auto store = [&](QueryTile<D>& t) {
#pragma unroll
            for (int r = 0; r < KR; ++r) {
                const int row = kq + (256 / P) * r;
                *reinterpret_cast<u32x4*>(t.q + row * D + 8 * ((int)(threadIdx.x % P) ^ twist<D>(row))) = qr[r];
            }
            if (wave == 0) {
                t.lse[lane] = lse_r;
                t.last[lane] = last_r;
                int least = last_r;
#pragma unroll
                for (int s = 1; s < 64; s <<= 1) least = min(least, __shfl_xor(least, s, 64));
                if (lane == 0) t.least = least;
            }
        };
        load(t0);
        store(tiles[t0 & 1]);
        if (t0 + 1 < t1) load(t0 + 1);
        __syncthreads();
        for (int t = t0; t < t1; ++t) {
            const QueryTile<D>& w = tiles[t & 1];
            const bool all = __builtin_amdgcn_readfirstlane(w.least) >= k0 + 16 * MT - 1;
            u32x4 x[NT][KS];
            auto read = [&](int nt) {
#pragma unroll
                for (int kk = 0; kk < KS; ++kk)
                    x[nt][kk] = *reinterpret_cast<const u32x4*>(w.q + (16 * nt + col) * D + 8 * ((4 * kk + grp) ^ twist<D>(col)));
            };
            auto product = [&](int nt, v4f(&s)[MT]) {
#pragma unroll
                for (int kk = 0; kk < KS; ++kk)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
                        s[mt] = E::mma32(kr[mt][kk], x[nt][kk], kk ? s[mt] : v4f{0.f, 0.f, 0.f, 0.f});
            };
            if (all) {
                // the weights of 16 rows between the products of the next 16:
                // one product, one fma, one exp2 and one addition in turn
                v4f s[2][MT];
                float lse[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) lse[nt] = w.lse[16 * nt + col];
                read(0);
                read(1);
                __builtin_amdgcn_sched_barrier(0);
                product(0, s[0]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (nt + 2 < NT) read(nt + 2);
                    if (nt + 1 < NT) product(nt + 1, s[(nt + 1) & 1]);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[mt][i] += fast_exp2(__builtin_fmaf(s[nt & 1][mt][i], p.scale_log2, -lse[nt]));
                    if (nt + 1 < NT) {
                        __builtin_amdgcn_sched_group_barrier(0x100, KS, 0);
#pragma unroll
                        for (int x = 0; x < KS * MT; ++x) {
                            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(0x002, 12 / KS, 0);
                        }
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            } else {
                read(0);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (t * kRows + 16 * nt >= p.M) break;
                    if (nt + 1 < NT) read(nt + 1);
                    const float lse = w.lse[16 * nt + col];
                    const int last = w.last[16 * nt + col] - k0 - 4 * grp;
                    v4f s[MT];
                    product(nt, s);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float e = fast_exp2(__builtin_fmaf(s[mt][i], p.scale_log2, -lse));
                            acc[mt][i] += 16 * mt + i <= last ? e : 0.f;
                        }
                }
            }
            if (t + 1 < t1) {
                store(tiles[(t + 1) & 1]);
                if (t + 2 < t1) load(t + 2);
            }
            __syncthreads();
        }
    }
    const float sum = columns_sum<MT>(acc);
    const int key = k0 + key_of_column<MT>(col);
    if (key >= p.c.keys) return;
    if (p.splits > 1) {
        p.part[(((int64_t)blockIdx.y * p.B + b) * p.Hk + h) * p.c.keys + key] = sum;
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

// Up to 16 query rows a KV head go to the kernel without LDS, more to the other
// (8 sequences of 32768 rows, 8 KV heads: 16 query rows 100 / 122 us, 32 rows 127
// / 123, 64 rows 183 / 121; one sequence 16.2 / 17.7, 20.3 / 17.6, 28.1 / 17.1).
// Its query rows are split until sixteen workgroups a CU are there, since ragged
// lengths leave part of them nothing to do (a 2048-query chunk of two sequences,
// one a quarter of the other: 286 us at eight, 264 at sixteen, 281 at thirty-two).
struct WeightsPlan {
    bool few;
    int64_t blocks;                                // of keys, a (sequence, head)
    int splits;
};

WeightsPlan plan_weights(const slimkv_attention_weights_args* a) {
    WeightsPlan w{};
    const int64_t M = a->queries * (a->heads / a->kv_heads), tiles = (M + kRows - 1) / kRows;
    w.few = M <= 16;
    const int64_t keys = w.few ? 128 : 256;        // of a workgroup
    w.blocks = (a->cache.keys + keys - 1) / keys;
    const int64_t workgroups = w.blocks * a->batch * a->kv_heads, want = 16 * device_cu_count();
    w.splits = w.few || workgroups <= 0 ? 1 : (int)std::max<int64_t>(1, std::min(want / workgroups, tiles / 4));
    return w;
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
    if (!scale_usable(a->scale)) return fail(SLIMKV_EINVAL, "attention weights: the softmax scale must lie in [1e-18, 1e18]");
    if (a->cache.keys < 0 || a->cache.keys > ((int64_t)1 << 30))
        return fail(SLIMKV_EINVAL, "attention weights: invalid cache length");
    return SLIMKV_OK;
}

template <int D, bool F16>
void launch_weights(const WeightsParams& p, bool few, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)p.B * p.Hk * p.blocks), (unsigned)p.splits);
    void (*kernel)(WeightsParams);
    if (few) kernel = p.c.table ? weights_few_kernel<D, F16, true> : weights_few_kernel<D, F16, false>;
    else kernel = p.c.table ? weights_many_kernel<D, F16, true> : weights_many_kernel<D, F16, false>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p);
}

}  // namespace

}  // namespace slimkv

using namespace slimkv;

extern "C" size_t slimkv_attention_weights_workspace(const slimkv_attention_weights_args* a) {
    if (check_weights(a) != SLIMKV_OK) return 0;
    const int splits = plan_weights(a).splits;
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
    p.B = (int)a->batch; p.L = (int)a->queries; p.Hk = (int)a->kv_heads; p.causal = a->causal ? 1 : 0;
    p.G = fast_div(a->heads / a->kv_heads);
    p.M = p.L * (int)p.G.d;
    const WeightsPlan plan = plan_weights(a);
    p.splits = plan.splits;
    p.blocks = (int)plan.blocks;
    p.scale_log2 = (float)(a->scale * 1.4426950408889634);
    p.part = static_cast<float*>(workspace);
    if (p.splits > 1 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
                         workspace_bytes < slimkv_attention_weights_workspace(a)))
        return fail(SLIMKV_EWORKSPACE, "attention weights: workspace missing, misaligned or too small");
    if (!launchable((int64_t)p.B * p.Hk * p.blocks, 256)) return fail(SLIMKV_EINVAL, "attention weights: too many rows for one call");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->head_dim == 128) {
        if (a->dtype == SLIMKV_DTYPE_F16) launch_weights<128, true>(p, plan.few, st);
        else launch_weights<128, false>(p, plan.few, st);
    } else {
        if (a->dtype == SLIMKV_DTYPE_F16) launch_weights<64, true>(p, plan.few, st);
        else launch_weights<64, false>(p, plan.few, st);
    }
    if (p.splits > 1) {
        const int64_t all = (int64_t)p.B * p.Hk * p.c.keys;
        hipLaunchKernelGGL(weights_sum_kernel, dim3((unsigned)((all + 255) / 256)), dim3(256), 0, st, p);
    }
    return check_hip(hipGetLastError(), "attention weights launch");
}
