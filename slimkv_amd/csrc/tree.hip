// Attention of a tree of drafted tokens over a cache: every query row sees all
// rows of its sequence's cache and the drafted tokens its mask names.
//
// The T * G query rows of one KV head (row p = t * G + g) are the columns of
// the score MFMA, as in the prefill kernel: S^T = K . Q^T with K rows as A and
// the query rows held in registers as B, softmax statistics per lane column,
// O^T = V^T . P^T with P^T straight from the score registers.  A workgroup of
// four waves holds 16 RW NT rows: RW waves side by side on rows, 4 / RW waves
// on the keys of a tile, joined at the end of an item.
//
// Key tiles of 64 rows -- the cache's, then the drafted tokens' -- pass through
// LDS, the next one in registers.  The drafted tokens of a tile are masked by
// their bytes; cache rows past the length read as zero and are masked.
//
// Schedule.  The tiles of all (sequence, KV head) items lie in a row and are
// dealt to `runs` workgroups in equal runs, whatever the lengths are; a run
// that holds part of an item leaves its unnormalised output, maxima and sums
// in the workspace for the merge kernel.  Each run exists once per block of
// query rows, side by side on one XCD, so that the blocks share the tiles in
// its L2.

#include "cache.hpp"

namespace slimkv {

namespace {

constexpr int kKeys = 64;                 // keys per tile
constexpr int kMergeRows = 8;             // query rows per merge workgroup
constexpr int kMaxDrafted = 1024;

struct TreeParams {
    CacheView c;
    const uint16_t* q; int64_t q_sb, q_sl, q_sh;
    const uint16_t* dk; int64_t dk_sb, dk_sn, dk_sh;
    const uint16_t* dv; int64_t dv_sb, dv_sn, dv_sh;
    const uint8_t* mask; int64_t m_sb, m_sl;
    uint16_t* out; int64_t o_sb, o_sl, o_sh;
    float* lse;
    int B, T, Hq, Hk, G, M;               // M = T * G query rows of a KV head
    int row_blocks, runs, least;          // least: tiles a run takes at least
    int64_t slots;                        // runs * row_blocks
    float scale_log2;
    float* part;
};

// Tiles of one KV head of a sequence with n cache rows.
__device__ __forceinline__ int item_tiles(int n, int T) {
    return (n + kKeys - 1) / kKeys + (T + kKeys - 1) / kKeys;
}

// Tiles of all items (wave-uniform result, every lane active).
__device__ __forceinline__ int64_t total_tiles(const TreeParams& p) {
    const int lane = threadIdx.x & 63;
    int64_t sum = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        int x = b0 + lane < p.B ? item_tiles(cache_length(p.c, b0 + lane), p.T) : 0;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) x += __shfl_xor(x, s, 64);
        sum += x;
    }
    return sum * p.Hk;
}

// Sequence that holds tile `pos`, the position of its first tile and its tiles
// a head.
struct Place {
    int b, tiles, n;
    int64_t first;
};

__device__ __forceinline__ Place place_of(const TreeParams& p, int64_t pos) {
    const int lane = threadIdx.x & 63;
    int64_t base = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        const int n = b0 + lane < p.B ? cache_length(p.c, b0 + lane) : 0;
        const int x = b0 + lane < p.B ? item_tiles(n, p.T) : 0;
        int64_t end = x;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int64_t y = __shfl_up(end, s, 64);
            if (lane >= s) end += y;
        }
        end = base + end * p.Hk;
        const uint64_t past = __ballot(pos < end);
        if (past) {
            const int at = __ffsll((unsigned long long)past) - 1;
            const int tiles = __shfl(x, at, 64);
            return Place{b0 + at, tiles, __shfl(n, at, 64), __shfl(end, at, 64) - (int64_t)tiles * p.Hk};
        }
        base = __shfl(end, 63, 64);
    }
    return Place{0, 1, 0, 0};             // not reached: pos < total_tiles
}

__device__ __forceinline__ int used_runs(const TreeParams& p, int64_t total) {
    const int64_t most = (total + p.least - 1) / p.least;
    return (int)(most < p.runs ? most : p.runs);
}

__device__ __forceinline__ int64_t run_begin(int64_t total, int runs, int r) { return r * total / runs; }

template <int D, int RW, int NT>
struct Shape {
    static constexpr int KW = 4 / RW;                      // waves side by side on a tile's keys
    static constexpr int MT = 4 / KW;                      // 16-key tiles a wave takes of a tile
    static constexpr int kRows = 16 * RW * NT;             // query rows of a workgroup
    static constexpr int KR = D / 32;                      // rows a thread loads of a tile (one 16-byte piece each)
    static constexpr int kKStride = D + 16;                // K tile row (16-bit elements)
    static constexpr int kVStride = kKeys + 8;             // V^T tile row
    static constexpr int kPart = kRows * (D + 2);          // floats of one partial
};

// Where a tile's rows lie: row `first` is the tile's first, rows from `n` on do
// not exist.
struct Tile {
    int first, n;
    bool draft;
};

template <int KR>
struct TileRegs {
    u32x4 k[KR], v[KR];
};

// The tile's rows KR kq + r (kq = thread / pieces a row), 16 bytes each of K
// and V.  Rows past the last one read it again; store_tile zeroes them.
template <int D, bool PAGED>
__device__ __forceinline__ void load_tile(TileRegs<D / 32>& t, const TreeParams& p, const Tile& w, int64_t b, int h) {
    constexpr int KR = D / 32, P = D / 8;
    const int kq = threadIdx.x / P, c = 8 * (threadIdx.x % P);
#pragma unroll
    for (int r = 0; r < KR; ++r) {
        const int row = min(w.first + KR * kq + r, w.n - 1);
        const uint16_t *ks, *vs;
        if (w.draft) {
            ks = p.dk + b * p.dk_sb + row * p.dk_sn + h * p.dk_sh;
            vs = p.dv + b * p.dv_sb + row * p.dv_sn + h * p.dv_sh;
        } else {
            const RowAt at = cache_row<PAGED>(p.c, b, row);
            ks = p.c.k + at.k + h * p.c.k_sh;
            vs = p.c.v + at.v + h * p.c.v_sh;
        }
        t.k[r] = *reinterpret_cast<const u32x4*>(ks + c);
        t.v[r] = *reinterpret_cast<const u32x4*>(vs + c);
    }
}

__device__ __forceinline__ uint32_t pair_of(uint32_t a, uint32_t b, bool high) {
    return __builtin_amdgcn_perm(b, a, high ? 0x07060302u : 0x05040100u);
}

// V^T keeps, per 32-key step, the keys a lane group reads together side by
// side: key 16 half + 4 g + j of the step at 8 g + 4 half + j.
__device__ __forceinline__ int vt_pos(int key) {
    const int step = key >> 5, half = (key >> 4) & 1, g = (key >> 2) & 3, j = key & 3;
    return 32 * step + 8 * g + 4 * half + j;
}

// K row-major, V transposed.  A drafted row may hold infinities or NaN that
// some query rows must not see: `wild` is then set for the tile.
template <int D, bool F16>
__device__ __forceinline__ void store_tile(const TileRegs<D / 32>& t, const Tile& w, uint16_t* ks, uint16_t* vts,
                                           int* wild) {
    constexpr int KR = D / 32, P = D / 8, kKStride = D + 16, kVStride = kKeys + 8;
    const int kq = threadIdx.x / P, c = 8 * (threadIdx.x % P);
    u32x4 v[KR];
    bool bad = false;
#pragma unroll
    for (int r = 0; r < KR; ++r) {
        const bool in = w.first + KR * kq + r < w.n;
        *reinterpret_cast<u32x4*>(ks + (KR * kq + r) * kKStride + c) = t.k[r];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[r][e] = in ? t.v[r][e] : 0u;
            if (w.draft) bad |= Elem<F16>::unbounded(v[r][e]);
        }
    }
    if (w.draft && bad) wild[w.first / kKeys] = 1;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        uint16_t* dst = vts + (c + e) * kVStride + vt_pos(KR * kq);
#pragma unroll
        for (int r = 0; r < KR; r += 2)
            *reinterpret_cast<uint32_t*>(dst + r) = pair_of(v[r][e >> 1], v[r + 1][e >> 1], e & 1);
    }
}

template <int D, bool F16, int RW, int NT, bool PAGED>
__global__ void __launch_bounds__(256) tree_kernel(TreeParams p) {
    using S = Shape<D, RW, NT>;
    using E = Elem<F16>;
    constexpr int KS = D / 32, MD = D / 16, MT = S::MT;
    constexpr int kBuf = kKeys * S::kKStride + D * S::kVStride;        // 16-bit elements of one tile
    constexpr int kJoin = S::KW > 1 ? (S::KW - 1) * S::kPart : 0;      // floats of the key waves' join
    constexpr int kBytes = 4 * kBuf > 4 * kJoin ? 4 * kBuf : 4 * kJoin;
    __shared__ __attribute__((aligned(16))) char lds[kBytes];
    __shared__ int wild[kMaxDrafted / kKeys];             // drafted tiles with values that are not finite
    uint16_t* bufs = reinterpret_cast<uint16_t*>(lds);

    const int64_t slot = (int64_t)(blockIdx.x % kXcdCount) * (gridDim.x / kXcdCount) + blockIdx.x / kXcdCount;
    if (slot >= p.slots) return;
    const int run = (int)(slot / p.row_blocks), rb = (int)(slot % p.row_blocks);
    const int64_t total = total_tiles(p);
    const int runs = used_runs(p, total);
    if (run >= runs) return;
    int64_t pos = run_begin(total, runs, run);
    const int64_t end = run_begin(total, runs, run + 1);

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int rw = wave % RW, kw = wave / RW;
    const int row0 = rb * S::kRows + rw * 16 * NT;        // the wave's first query row

    while (pos < end) {
        const Place at = place_of(p, pos);
        const int64_t b = at.b;
        const int h = (int)((pos - at.first) / at.tiles);
        const int t0 = (int)(pos - at.first - (int64_t)h * at.tiles);
        const int t1 = (int)min<int64_t>(at.tiles, t0 + end - pos);
        const int cached = (at.n + kKeys - 1) / kKeys;     // the first drafted tile
        auto tile = [&](int t) {
            return t < cached ? Tile{t * kKeys, at.n, false} : Tile{(t - cached) * kKeys, p.T, true};
        };

        TileRegs<S::KR> tr;
        load_tile<D, PAGED>(tr, p, tile(t0), b, h);
        u32x4 qr[NT][KS];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int row = row0 + 16 * nt + col;
            const int r = min(row, p.M - 1), t = r / p.G, g = r - t * p.G;
            const uint16_t* src = p.q + b * p.q_sb + t * p.q_sl + (int64_t)(h * p.G + g) * p.q_sh + 8 * grp;
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                const u32x4 x = *reinterpret_cast<const u32x4*>(src + 32 * kk);
                const bool ok = row < p.M;
                qr[nt][kk] = u32x4{ok ? x.x : 0u, ok ? x.y : 0u, ok ? x.z : 0u, ok ? x.w : 0u};
            }
        }
        v4f o[MD][NT];
        float m[NT], l[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt] = kNegInf;
            l[nt] = 0.f;
#pragma unroll
            for (int md = 0; md < MD; ++md) o[md][nt] = v4f{0.f, 0.f, 0.f, 0.f};
        }

        __syncthreads();                                   // the item before is done with the buffers
        if (threadIdx.x < kMaxDrafted / kKeys) wild[threadIdx.x] = 0;
        __syncthreads();
        store_tile<D, F16>(tr, tile(t0), bufs + (t0 & 1) * kBuf, bufs + (t0 & 1) * kBuf + kKeys * S::kKStride, wild);
        if (t0 + 1 < t1) load_tile<D, PAGED>(tr, p, tile(t0 + 1), b, h);
        __syncthreads();

        for (int t = t0; t < t1; ++t) {
            const Tile w = tile(t);
            const uint16_t* ks = bufs + (t & 1) * kBuf;
            const uint16_t* vts = ks + kKeys * S::kKStride;
            const int key0 = kw * 16 * MT;                 // the wave's first key in the tile

            v4f s[MT][NT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[mt][nt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < KS; ++kk)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const u32x4 a = *reinterpret_cast<const u32x4*>(ks + (key0 + 16 * mt + col) * S::kKStride + 32 * kk +
                                                                    8 * grp);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) s[mt][nt] = E::mma32(a, qr[nt][kk], s[mt][nt]);
                }

            if (w.draft) {                                 // by the mask's bytes, or j <= t without one
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const int tq = min(row0 + 16 * nt + col, p.M - 1) / p.G;
                    const uint8_t* mrow = p.mask + b * p.m_sb + tq * p.m_sl;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int j = w.first + key0 + 16 * mt + 4 * grp + i;
                            const bool seen = j < p.T && (p.mask ? mrow[min(j, p.T - 1)] != 0 : j <= tq);
                            s[mt][nt][i] = seen ? s[mt][nt][i] : kNegInf;
                        }
                }
            } else if (w.first + kKeys > w.n) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool seen = w.first + key0 + 16 * mt + 4 * grp + i < w.n;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) s[mt][nt][i] = seen ? s[mt][nt][i] : kNegInf;
                    }
            }

#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float mx = kNegInf;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[mt][nt][i]);
                mx = rows_max(mx);
                const float m_new = fmaxf(m[nt], mx * p.scale_log2);
                const float base = m_new == kNegInf ? 0.f : m_new;
                const float alpha = fast_exp2(m[nt] - base);
                m[nt] = m_new;
                float sum = 0.f;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[mt][nt][i] = fast_exp2(__builtin_fmaf(s[mt][nt][i], p.scale_log2, -base));
                        sum += s[mt][nt][i];
                    }
                if (__ballot(alpha != 1.f)) {
#pragma unroll
                    for (int md = 0; md < MD; ++md) o[md][nt] *= alpha;
                    l[nt] *= alpha;
                }
                l[nt] += sum;                              // fp32, of the unrounded weights
            }

            if (w.draft && wild[w.first / kKeys]) {
                // drafted values that are not finite: weight by weight, so that a
                // row takes nothing from a token it does not see
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        for (int g = 0; g < 4; ++g) {
                            const int j = w.first + key0 + 16 * mt + 4 * g + i;
                            if (j >= p.T) continue;
                            const uint16_t* vrow = p.dv + b * p.dv_sb + j * p.dv_sn + h * p.dv_sh + 4 * grp;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                const float pj = __shfl(s[mt][nt][i], col + 16 * g, 64);
#pragma unroll
                                for (int md = 0; md < MD; ++md) {
                                    const u32x2 x = *reinterpret_cast<const u32x2*>(vrow + 16 * md);
                                    const float vals[4] = {E::lo(x.x), E::hi(x.x), E::lo(x.y), E::hi(x.y)};
#pragma unroll
                                    for (int e = 0; e < 4; ++e) o[md][nt][e] += pj == 0.f ? 0.f : pj * vals[e];
                                }
                            }
                        }
            } else if constexpr (MT == 1) {                // 16 keys: half a step
#pragma unroll
                for (int md = 0; md < MD; ++md) {
                    const u32x2 a = *reinterpret_cast<const u32x2*>(vts + (16 * md + col) * S::kVStride +
                                                                    32 * (kw >> 1) + 8 * grp + 4 * (kw & 1));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        o[md][nt] = E::mma16(a, u32x2{E::pack(s[0][nt][0], s[0][nt][1]), E::pack(s[0][nt][2], s[0][nt][3])},
                                             o[md][nt]);
                }
            } else {
#pragma unroll
                for (int ss = 0; ss < MT / 2; ++ss) {
                    u32x4 pb[NT];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        pb[nt] = u32x4{E::pack(s[2 * ss][nt][0], s[2 * ss][nt][1]), E::pack(s[2 * ss][nt][2], s[2 * ss][nt][3]),
                                       E::pack(s[2 * ss + 1][nt][0], s[2 * ss + 1][nt][1]),
                                       E::pack(s[2 * ss + 1][nt][2], s[2 * ss + 1][nt][3])};
#pragma unroll
                    for (int md = 0; md < MD; ++md) {
                        const u32x4 a = *reinterpret_cast<const u32x4*>(vts + (16 * md + col) * S::kVStride + key0 +
                                                                        32 * ss + 8 * grp);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) o[md][nt] = E::mma32(a, pb[nt], o[md][nt]);
                    }
                }
            }

            if (t + 1 < t1) {
                uint16_t* next = bufs + ((t + 1) & 1) * kBuf;
                store_tile<D, F16>(tr, tile(t + 1), next, next + kKeys * S::kKStride, wild);
                if (t + 2 < t1) load_tile<D, PAGED>(tr, p, tile(t + 2), b, h);
            }
            __syncthreads();
        }

        // the key waves' states joined in the first one's registers
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) l[nt] = rows_sum(l[nt]);
        if constexpr (S::KW > 1) {
            float* join = reinterpret_cast<float*>(lds);
            if (kw > 0) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float* e = join + (kw - 1) * S::kPart;
                    const int row = rw * 16 * NT + 16 * nt + col;
#pragma unroll
                    for (int md = 0; md < MD; ++md) *reinterpret_cast<v4f*>(e + row * D + 16 * md + 4 * grp) = o[md][nt];
                    if (grp == 0) {
                        e[S::kRows * D + row] = m[nt];
                        e[S::kRows * D + S::kRows + row] = l[nt];
                    }
                }
            }
            __syncthreads();
            if (kw == 0) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const int row = rw * 16 * NT + 16 * nt + col;
                    float top = m[nt];
#pragma unroll
                    for (int x = 0; x < S::KW - 1; ++x) top = fmaxf(top, join[x * S::kPart + S::kRows * D + row]);
                    const float base = top == kNegInf ? 0.f : top;
                    const float own = fast_exp2(m[nt] - base);
                    l[nt] *= own;
#pragma unroll
                    for (int md = 0; md < MD; ++md) o[md][nt] *= own;
                    m[nt] = top;
#pragma unroll
                    for (int x = 0; x < S::KW - 1; ++x) {
                        const float* e = join + x * S::kPart;
                        const float f = fast_exp2(e[S::kRows * D + row] - base);
                        l[nt] += f * e[S::kRows * D + S::kRows + row];
#pragma unroll
                        for (int md = 0; md < MD; ++md)
                            o[md][nt] += f * *reinterpret_cast<const v4f*>(e + row * D + 16 * md + 4 * grp);
                    }
                }
            }
        }

        if (kw == 0) {
            if (t0 > 0 || t1 < at.tiles) {
                float* part = p.part + (2 * slot + (t0 == 0)) * S::kPart;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const int row = rw * 16 * NT + 16 * nt + col;
                    if (rb * S::kRows + row >= p.M) continue;
#pragma unroll
                    for (int md = 0; md < MD; ++md) *reinterpret_cast<v4f*>(part + row * D + 16 * md + 4 * grp) = o[md][nt];
                    if (grp == 0) {
                        part[S::kRows * D + row] = m[nt];
                        part[S::kRows * D + S::kRows + row] = l[nt];
                    }
                }
            } else {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const int row = row0 + 16 * nt + col;
                    if (row >= p.M) continue;
                    const int tq = row / p.G, g = row - tq * p.G;
                    const float inv = l[nt] == 0.f ? 0.f : 1.f / l[nt];
                    uint16_t* dst = p.out + b * p.o_sb + tq * p.o_sl + (int64_t)(h * p.G + g) * p.o_sh + 4 * grp;
#pragma unroll
                    for (int md = 0; md < MD; ++md)
                        *reinterpret_cast<u32x2*>(dst + 16 * md) = u32x2{E::pack(o[md][nt][0] * inv, o[md][nt][1] * inv),
                                                                         E::pack(o[md][nt][2] * inv, o[md][nt][3] * inv)};
                    if (p.lse && grp == 0)
                        p.lse[(b * p.Hq + h * p.G + g) * p.T + tq] =
                            l[nt] == 0.f ? kNegInf : (m[nt] + __log2f(l[nt])) * kLn2;
                }
            }
        }
        pos += t1 - t0;
    }
}

// Merges the runs of every item that lies in more than one: D / 4 lanes a row,
// kMergeRows rows of one (sequence, KV head) a workgroup.
template <int D, bool F16>
__global__ void __launch_bounds__(kMergeRows * D / 4) tree_merge_kernel(TreeParams p, int rows_wg, int chunks) {
    using E = Elem<F16>;
    const int item = blockIdx.x / chunks;
    const int64_t b = item / p.Hk;
    const int h = item % p.Hk;
    const int row = (blockIdx.x % chunks) * kMergeRows + threadIdx.x / (D / 4), c = 4 * (threadIdx.x % (D / 4));

    // first tile of the item: tiles of the sequences before it
    const int lane = threadIdx.x & 63;
    int64_t before = 0, all = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        const int x = b0 + lane < p.B ? item_tiles(cache_length(p.c, b0 + lane), p.T) : 0;
        int lower = b0 + lane < b ? x : 0, any = x;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            lower += __shfl_xor(lower, s, 64);
            any += __shfl_xor(any, s, 64);
        }
        before += lower;
        all += any;
    }
    const int tiles = item_tiles(cache_length(p.c, b), p.T);
    const int64_t total = all * p.Hk, first = before * p.Hk + (int64_t)h * tiles, last = first + tiles - 1;
    const int runs = used_runs(p, total);
    auto run_of = [&](int64_t pos) {
        int r = (int)(pos * runs / total);
        while (run_begin(total, runs, r + 1) <= pos) ++r;
        return r;
    };
    const int r0 = run_of(first), r1 = run_of(last);
    if (r0 == r1 || row >= p.M) return;
    const int rb = row / rows_wg, in = row - rb * rows_wg;
    const int64_t size = (int64_t)rows_wg * (D + 2);
    auto entry = [&](int r) {
        const bool starts = run_begin(total, runs, r) <= first;
        return p.part + (2 * ((int64_t)r * p.row_blocks + rb) + starts) * size;
    };
    float M = kNegInf;
    for (int r = r0; r <= r1; ++r) M = fmaxf(M, entry(r)[rows_wg * D + in]);
    const float base = M == kNegInf ? 0.f : M;
    float L = 0.f;
    v4f acc = {0.f, 0.f, 0.f, 0.f};
    for (int r = r0; r <= r1; ++r) {
        const float* e = entry(r);
        const float f = fast_exp2(e[rows_wg * D + in] - base);
        L += f * e[rows_wg * D + rows_wg + in];
        acc += f * *reinterpret_cast<const v4f*>(e + in * D + c);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int tq = row / p.G, g = row - tq * p.G;
    *reinterpret_cast<u32x2*>(p.out + b * p.o_sb + tq * p.o_sl + (int64_t)(h * p.G + g) * p.o_sh + c) =
        u32x2{E::pack(acc[0] * inv, acc[1] * inv), E::pack(acc[2] * inv, acc[3] * inv)};
    if (p.lse && c == 0) p.lse[(b * p.Hq + h * p.G + g) * p.T + tq] = L == 0.f ? kNegInf : (M + __log2f(L)) * kLn2;
}

struct TreePlan {
    int rw, nt, row_blocks, runs;
    int64_t slots;
    int rows() const { return 16 * rw * nt; }
    size_t bytes(int64_t D) const { return (size_t)slots * 2 * rows() * (D + 2) * sizeof(float); }
};

// Query rows a workgroup holds: the fewest of 16, 32, 64 and 128 that hold all
// of them (128 for more).  Runs: two workgroups a CU over all row blocks.
TreePlan plan_tree(const slimkv_tree_attention_args* a) {
    TreePlan t{};
    const int64_t M = a->drafted * (a->heads / a->kv_heads);
    t.rw = M <= 32 ? 1 : M <= 64 ? 2 : 4;
    t.nt = M <= 16 ? 1 : 2;
    t.row_blocks = std::max(1, (int)((M + t.rows() - 1) / t.rows()));
    t.runs = std::max(1, 2 * device_cu_count() / t.row_blocks);
    t.slots = (int64_t)t.runs * t.row_blocks;
    return t;
}

int check_tree(const slimkv_tree_attention_args* a) {
    if (!a || (!a->q && a->drafted > 0 && a->batch > 0)) return fail(SLIMKV_EINVAL, "tree attention: null pointer");
    if (a->head_dim != 64 && a->head_dim != 128) return fail(SLIMKV_EUNSUP, "tree attention: head_dim must be 64 or 128");
    if (a->dtype != SLIMKV_DTYPE_BF16 && a->dtype != SLIMKV_DTYPE_F16)
        return fail(SLIMKV_EUNSUP, "tree attention: element type must be bf16 or fp16");
    if (a->batch < 0 || a->batch > 65535 || a->drafted < 0 || a->drafted > kMaxDrafted || a->heads <= 0 || a->kv_heads <= 0 ||
        a->heads % a->kv_heads || a->heads > 4096 || a->heads / a->kv_heads > 256)
        return fail(SLIMKV_EINVAL, "tree attention: invalid sizes");
    if (!(a->scale > 0.0)) return fail(SLIMKV_EINVAL, "tree attention: the softmax scale must be positive");
    return SLIMKV_OK;
}

template <int D, bool F16, int RW, int NT>
void launch_tree(const TreeParams& p, const TreePlan& plan, hipStream_t st) {
    const dim3 grid((unsigned)((plan.slots + kXcdCount - 1) / kXcdCount * kXcdCount));
    if (p.c.table) hipLaunchKernelGGL((tree_kernel<D, F16, RW, NT, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((tree_kernel<D, F16, RW, NT, false>), grid, dim3(256), 0, st, p);
    const int chunks = (p.M + kMergeRows - 1) / kMergeRows;
    hipLaunchKernelGGL((tree_merge_kernel<D, F16>), dim3((unsigned)(p.B * p.Hk * chunks)), dim3(kMergeRows * D / 4), 0, st,
                       p, plan.rows(), chunks);
}

template <int D, bool F16>
void launch_rows(const TreeParams& p, const TreePlan& plan, hipStream_t st) {
    if (plan.rw == 4) launch_tree<D, F16, 4, 2>(p, plan, st);
    else if (plan.rw == 2) launch_tree<D, F16, 2, 2>(p, plan, st);
    else if (plan.nt == 2) launch_tree<D, F16, 1, 2>(p, plan, st);
    else launch_tree<D, F16, 1, 1>(p, plan, st);
}

}  // namespace

bool rows_aligned(const void* p, std::initializer_list<std::pair<int64_t, int64_t>> size_and_stride) {
    if (reinterpret_cast<uintptr_t>(p) & 15) return false;
    for (const auto& s : size_and_stride)
        if (s.first > 1 && s.second % 8) return false;
    return true;
}

int cache_view(const slimkv_cache_rows& r, int64_t batch, int64_t kv_heads, int64_t head_dim, bool need_v,
               const char* what, CacheView* view) {
    const std::string w(what);
    if (r.keys < 0 || r.keys > ((int64_t)1 << 30)) return fail(SLIMKV_EINVAL, w + ": invalid cache length");
    if (r.keys > 0 && (!r.k || (need_v && !r.v))) return fail(SLIMKV_EINVAL, w + ": null cache pointer");
    if (r.table && (r.block_size <= 0 || r.num_blocks <= 0 || r.num_blocks > ((int64_t)1 << 40) || r.t_cols <= 0 ||
                    (batch > 1 && r.t_sb < r.t_cols && r.t_sb != 0) || r.block_size > ((int64_t)1 << 30) ||
                    r.t_cols > ((int64_t)1 << 30) || r.keys > r.t_cols * r.block_size))
        return fail(SLIMKV_EINVAL, w + ": invalid page layout (cache rows past the block table?)");
    const int64_t outer = r.table ? r.num_blocks : batch, rows = r.table ? r.block_size : r.keys;
    if (r.keys > 0 && (!rows_aligned(r.k, {{outer, r.k_sb}, {rows, r.k_sn}, {kv_heads, r.k_sh}}) ||
                       (need_v && !rows_aligned(r.v, {{outer, r.v_sb}, {rows, r.v_sn}, {kv_heads, r.v_sh}}))))
        return fail(SLIMKV_EINVAL, w + ": cache rows must start on 16-byte boundaries (strides multiples of 8)");
    (void)head_dim;
    view->k = static_cast<const uint16_t*>(r.k); view->k_sb = r.k_sb; view->k_sn = r.k_sn; view->k_sh = r.k_sh;
    view->v = static_cast<const uint16_t*>(r.v); view->v_sb = r.v_sb; view->v_sn = r.v_sn; view->v_sh = r.v_sh;
    view->table = r.table; view->t_sb = r.t_sb; view->num_blocks = r.num_blocks;
    view->block = fast_div(r.table ? r.block_size : 1);
    view->lengths = r.lengths; view->keys = (int)r.keys; view->status = r.status;
    return SLIMKV_OK;
}

}  // namespace slimkv

using namespace slimkv;

extern "C" int slimkv_cache_abi_version(void) { return 1; }

extern "C" size_t slimkv_tree_attention_workspace(const slimkv_tree_attention_args* a) {
    if (check_tree(a) != SLIMKV_OK) return 0;
    return std::max<size_t>(plan_tree(a).bytes(a->head_dim), 16);
}

extern "C" int slimkv_tree_attention(const slimkv_tree_attention_args* a, void* workspace, size_t workspace_bytes,
                                     void* stream) {
    const int code = check_tree(a);
    if (code != SLIMKV_OK) return code;
    if (a->batch == 0 || a->drafted == 0) return SLIMKV_OK;
    if (!a->draft_k || !a->draft_v || !a->out) return fail(SLIMKV_EINVAL, "tree attention: null pointer");
    TreeParams p{};
    const int view = cache_view(a->cache, a->batch, a->kv_heads, a->head_dim, true, "tree attention", &p.c);
    if (view != SLIMKV_OK) return view;
    const int64_t B = a->batch, T = a->drafted, Hq = a->heads, Hk = a->kv_heads;
    if (!rows_aligned(a->q, {{B, a->q_sb}, {T, a->q_sl}, {Hq, a->q_sh}}) ||
        !rows_aligned(a->draft_k, {{B, a->dk_sb}, {T, a->dk_sn}, {Hk, a->dk_sh}}) ||
        !rows_aligned(a->draft_v, {{B, a->dv_sb}, {T, a->dv_sn}, {Hk, a->dv_sh}}) ||
        !rows_aligned(a->out, {{B, a->o_sb}, {T, a->o_sl}, {Hq, a->o_sh}}))
        return fail(SLIMKV_EINVAL, "tree attention: rows must start on 16-byte boundaries (strides multiples of 8)");
    const TreePlan plan = plan_tree(a);
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < plan.bytes(a->head_dim))
        return fail(SLIMKV_EWORKSPACE, "tree attention: workspace missing, misaligned or too small");
    p.q = static_cast<const uint16_t*>(a->q); p.q_sb = a->q_sb; p.q_sl = a->q_sl; p.q_sh = a->q_sh;
    p.dk = static_cast<const uint16_t*>(a->draft_k); p.dk_sb = a->dk_sb; p.dk_sn = a->dk_sn; p.dk_sh = a->dk_sh;
    p.dv = static_cast<const uint16_t*>(a->draft_v); p.dv_sb = a->dv_sb; p.dv_sn = a->dv_sn; p.dv_sh = a->dv_sh;
    p.mask = a->mask; p.m_sb = a->m_sb; p.m_sl = a->m_sl;
    p.out = static_cast<uint16_t*>(a->out); p.o_sb = a->o_sb; p.o_sl = a->o_sl; p.o_sh = a->o_sh;
    p.lse = a->lse;
    p.B = (int)B; p.T = (int)T; p.Hq = (int)Hq; p.Hk = (int)Hk; p.G = (int)(Hq / Hk);
    p.M = p.T * p.G;
    p.row_blocks = plan.row_blocks; p.runs = plan.runs; p.slots = plan.slots;
    p.least = 2;
    p.scale_log2 = (float)(a->scale * 1.4426950408889634);
    p.part = static_cast<float*>(workspace);
    if ((int64_t)p.B * p.Hk * ((p.M + kMergeRows - 1) / kMergeRows) > 0x7fffffff)
        return fail(SLIMKV_EINVAL, "tree attention: too many rows for one call");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->head_dim == 128) {
        if (a->dtype == SLIMKV_DTYPE_F16) launch_rows<128, true>(p, plan, st);
        else launch_rows<128, false>(p, plan, st);
    } else {
        if (a->dtype == SLIMKV_DTYPE_F16) launch_rows<64, true>(p, plan, st);
        else launch_rows<64, false>(p, plan, st);
    }
    return check_hip(hipGetLastError(), "tree attention launch");
}
