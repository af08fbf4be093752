// What the attentions of drafted tokens share, over a cache of full-width rows and
// over one held in 4 bits: query rows as MFMA columns, the drafted tokens' tiles
// and masks, the softmax step, the split of a ragged batch into runs and their
// merge.
#pragma once

#include "cache.hpp"

namespace slimkv {

namespace {

constexpr int kKeys = 64;                 // keys per tile
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
    int row_blocks;
    Dealing deal;
    float scale_log2;
    float* part;
};

// ---------------------------------------------------------------------------
// what both kernels share
// ---------------------------------------------------------------------------

// The page numbers of a stretch of the cache, in LDS: a tile's loads then wait
// for no table read.  Holds table columns [first, first + kPages).
constexpr int kPages = 1024;

struct Pages {
    int32_t page[kPages];
};

// Tiles a stretch holds at any block size: 64 c rows span at most 64 c / block
// + 2 columns.
__device__ __forceinline__ int page_tiles(const CacheView& c) {
    return (int)min<int64_t>((int64_t)(kPages - 2) * c.block.d / kKeys, 1 << 24);
}

// Columns of tiles [t, t + page_tiles) that rows below n need; every thread of
// the workgroup, between barriers.
__device__ __forceinline__ void load_pages(const CacheView& c, int64_t b, int t, int n, Pages& s) {
    const int first = quotient(t * kKeys, c.block), last = quotient(n - 1, c.block);
    const int count = min(last - first + 1, kPages);
    for (int i = threadIdx.x; i < count; i += 256) {
        const int64_t page = table_page(c.table[b * c.t_sb + first + i], c.num_blocks);
        if (page < 0) report_bad_page(c.status);
        s.page[i] = page < 0 ? 0 : (int)page;
    }
}

// Row `row` (below the length) through the stretch that begins with tile t.
__device__ __forceinline__ RowAt paged_row(const CacheView& c, const Pages& s, int t, int row) {
    const int col = quotient(row, c.block);
    const int64_t page = s.page[col - quotient(t * kKeys, c.block)];
    const int64_t slot = row - col * (int)c.block.d;
    return RowAt{page * c.k_sb + slot * c.k_sn, page * c.v_sb + slot * c.v_sn};
}

// Order LDS accesses of one wave: its LDS instructions execute in issue order,
// so only the compiler's reordering has to be prevented.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Which drafted tokens first .. first + 63 the tokens of `rows` query rows from
// row0 on see, one 64-bit word a token in the wave's own LDS: lane j reads the
// byte of token first + j and the ballot makes the word.
__device__ __forceinline__ void drafted_seen(const TreeParams& p, int64_t b, int row0, int rows, int first,
                                             uint64_t* words) {
    const int lane = threadIdx.x & 63, j = first + lane;
    const int from = min(row0, p.M - 1) / p.G, to = min(row0 + rows - 1, p.M - 1) / p.G;
    wave_fence();
    for (int t0 = from; t0 <= to; t0 += 4) {               // four tokens' bytes in flight
        bool sees[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int tq = min(t0 + i, to);
            sees[i] = j < p.T && (p.mask ? p.mask[b * p.m_sb + tq * p.m_sl + min(j, p.T - 1)] != 0 : j <= tq);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t word = __ballot(sees[i]);
            if (lane == 0) words[min(t0 + i, to) - from] = word;
        }
    }
    wave_fence();
}

// Drafted values that are not finite stay out of the matrix product (0 there,
// with the flag set), since a zero weight would not keep them from rows that
// do not see them.
template <bool F16>
__device__ __forceinline__ u32x4 finite_only(u32x4 x, bool* wild) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t w = x[e];
        if (Elem<F16>::unbounded(w)) {
            *wild = true;
            const uint32_t all = F16 ? 0x7c00u : 0x7f80u;
            x[e] = ((w & all) == all ? 0u : w & 0xffffu) | ((w >> 16 & all) == all ? 0u : w & 0xffff0000u);
        }
    }
    return x;
}

// They are then added to the rows that do see them: any positive weight makes
// an infinity or NaN of them.  Tokens [j0, j1); lane (col, grp) holds columns
// 16 md + 4 grp + e of row row0 + col.
template <int MD, bool F16>
__device__ __forceinline__ void add_unbounded(const TreeParams& p, int64_t b, int h, int j0, int j1, int row,
                                              v4f (&o)[MD]) {
    const int tq = min(row, p.M - 1) / p.G, grp = (threadIdx.x & 63) >> 4;
#pragma unroll 1
    for (int j = j0; j < j1; ++j) {
        const bool seen = p.mask ? p.mask[b * p.m_sb + tq * p.m_sl + j] != 0 : j <= tq;
        const uint16_t* v = p.dv + b * p.dv_sb + j * p.dv_sn + h * p.dv_sh + 4 * grp;
#pragma unroll
        for (int md = 0; md < MD; ++md) {
            const u32x2 x = *reinterpret_cast<const u32x2*>(v + 16 * md);
            const float f[4] = {Elem<F16>::lo(x.x), Elem<F16>::hi(x.x), Elem<F16>::lo(x.y), Elem<F16>::hi(x.y)};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (seen && !(__builtin_fabsf(f[e]) < __builtin_inff())) o[md][e] += f[e];
        }
    }
}

// Query rows row0 + 16 nt + col as MFMA operands, zero past the last one.  Step
// kk of lane group grp holds elements 32 kk + 8 grp + [0, 8), or, where a group's
// steps lie side by side (GROUPED), 8 (KS grp + kk) + [0, 8); the keys' operands
// follow the same order.
template <int KS, int NT, bool GROUPED = false>
__device__ __forceinline__ void load_queries(const TreeParams& p, int64_t b, int h, int row0, u32x4 (&qr)[NT][KS]) {
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    constexpr int kGroup = GROUPED ? 8 * KS : 8, kStep = GROUPED ? 8 : 32;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = row0 + 16 * nt + col;
        const int r = min(row, p.M - 1), t = r / p.G, g = r - t * p.G;
        const uint16_t* src = p.q + b * p.q_sb + t * p.q_sl + (int64_t)(h * p.G + g) * p.q_sh + kGroup * grp;
        const bool ok = row < p.M;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(src + kStep * kk);
            qr[nt][kk] = u32x4{ok ? x.x : 0u, ok ? x.y : 0u, ok ? x.z : 0u, ok ? x.w : 0u};
        }
    }
}

// A score's exponent against the row's base.  Fused, it is rounded once, but the
// largest score then ends at the rounding of its product, which is in the base: up
// to half a step of it either way, past the exponents of fp16 from 2^28 on and of
// fp32 from 2^31.  From kFarBase on the products are rounded before the
// difference, as they were for the base, and the largest ends at zero.
constexpr float kFarBase = 1048576.f;
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}
__device__ __forceinline__ float far_exponent(float s, float scale_log2, float base) {
#pragma clang fp contract(off)
    return __builtin_fabsf(base) >= kFarBase ? rounded_product(s, scale_log2) - base : __builtin_fmaf(s, scale_log2, -base);
}

// The base of a maximum, in log2.  fp16 weights against the maximum itself would be
// subnormal from 2^-14 of it on and nothing from 2^-25, while their sum kept them:
// 15 less, weights of up to 2^15 go down to 2^-39 of the largest in what the type
// holds.  The sum and the output carry the same factor, and base + log2 of the sum
// is the LSE for any base.  Maxima whose rounding could take a weight past the type
// stay their own base.
template <bool F16>
__device__ __forceinline__ float base_of(float top) {
    if constexpr (F16) return __builtin_fabsf(top) < kFarBase ? top - 15.f : top;
    return top;
}

// One online-softmax step of a column's scores: the scores become weights, the
// state moves to the new base.  The weights' sum is fp32 and of the unrounded
// weights; a lane keeps the sum of its own keys.
template <int MT, int MD, bool F16>
__device__ __forceinline__ void softmax_step(v4f (&s)[MT], float scale_log2, float& m, float& l, v4f (&o)[MD]) {
    float mx = kNegInf;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[mt][i]);
    mx = rows_max(mx);
    const float m_new = fmaxf(m, base_of<F16>(rounded_product(mx, scale_log2)));
    const float base = m_new == kNegInf ? 0.f : m_new;
    const float alpha = fast_exp2(m - base);
    m = m_new;
    float sum = 0.f;
    auto weigh = [&](auto exponent) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[mt][i] = fast_exp2(exponent(s[mt][i]));
                sum += s[mt][i];
            }
    };
    if (__ballot(__builtin_fabsf(base) >= kFarBase)) weigh([&](float x) { return far_exponent(x, scale_log2, base); });
    else weigh([&](float x) { return __builtin_fmaf(x, scale_log2, -base); });
    if (__ballot(alpha != 1.f)) {
#pragma unroll
        for (int md = 0; md < MD; ++md) o[md] *= alpha;
        l *= alpha;
    }
    l += sum;
}

// A finished row set: the output where the item lies in this run alone, else a
// partial entry of `rows` rows.  l is summed over the lane groups.
template <int MD, bool F16>
__device__ __forceinline__ void finish_rows(const TreeParams& p, int64_t b, int h, int row, int in, int rows, bool whole,
                                            float* part, float m, float l, const v4f (&o)[MD]) {
    using E = Elem<F16>;
    constexpr int D = 16 * MD;
    const int grp = (threadIdx.x & 63) >> 4;
    if (row >= p.M) return;
    if (!whole) {
#pragma unroll
        for (int md = 0; md < MD; ++md) *reinterpret_cast<v4f*>(part + in * D + 16 * md + 4 * grp) = o[md];
        if (grp == 0) {
            part[rows * D + in] = m;
            part[rows * D + rows + in] = l;
        }
        return;
    }
    const int tq = row / p.G, g = row - tq * p.G;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t* dst = p.out + b * p.o_sb + tq * p.o_sl + (int64_t)(h * p.G + g) * p.o_sh + 4 * grp;
#pragma unroll
    for (int md = 0; md < MD; ++md)
        *reinterpret_cast<u32x2*>(dst + 16 * md) =
            u32x2{E::pack(o[md][0] * inv, o[md][1] * inv), E::pack(o[md][2] * inv, o[md][3] * inv)};
    if (p.lse && grp == 0) p.lse[(b * p.Hq + h * p.G + g) * p.T + tq] = l == 0.f ? kNegInf : (m + __log2f(l)) * kLn2;
}

// Joins the states of KW key waves in those of wave 0: the others leave theirs
// in LDS (entries of `rows` rows).  Every wave calls it.
template <int MD, int NT, int KW>
__device__ __forceinline__ void join_keys(float* lds, int rows, int row0, int kw, float (&m)[NT], float (&l)[NT],
                                          v4f (&o)[NT][MD]) {
    constexpr int D = 16 * MD;
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const int size = rows * (D + 2);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) l[nt] = rows_sum(l[nt]);
    if constexpr (KW == 1) return;
    if (kw > 0) {
        float* e = lds + (kw - 1) * size;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int row = row0 + 16 * nt + col;
#pragma unroll
            for (int md = 0; md < MD; ++md) *reinterpret_cast<v4f*>(e + row * D + 16 * md + 4 * grp) = o[nt][md];
            if (grp == 0) {
                e[rows * D + row] = m[nt];
                e[rows * D + rows + row] = l[nt];
            }
        }
    }
    __syncthreads();
    if (kw > 0) return;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = row0 + 16 * nt + col;
        float top = m[nt];
#pragma unroll
        for (int x = 0; x < KW - 1; ++x) top = fmaxf(top, lds[x * size + rows * D + row]);
        const float base = top == kNegInf ? 0.f : top;
        const float own = fast_exp2(m[nt] - base);
        l[nt] *= own;
#pragma unroll
        for (int md = 0; md < MD; ++md) o[nt][md] *= own;
        m[nt] = top;
#pragma unroll
        for (int x = 0; x < KW - 1; ++x) {
            const float* e = lds + x * size;
            const float f = fast_exp2(e[rows * D + row] - base);
            l[nt] += f * e[rows * D + rows + row];
#pragma unroll
            for (int md = 0; md < MD; ++md) o[nt][md] += f * *reinterpret_cast<const v4f*>(e + row * D + 16 * md + 4 * grp);
        }
    }
}

// The run of a workgroup, item by item.
struct Item {
    int64_t b;
    int h, n, t0, t1, tiles;
};

__device__ __forceinline__ Item item_at(const TreeParams& p, int pos, int end) {
    const Place at = place_of(p.c, p.deal, pos);
    Item it;
    it.b = at.b;
    it.n = at.n;
    it.tiles = at.tiles;
    it.h = (uint32_t)(pos - at.first) / (uint32_t)at.tiles;
    it.t0 = pos - at.first - it.h * at.tiles;
    it.t1 = min(at.tiles, it.t0 + end - pos);
    return it;
}

// The rows of 16 keys in LDS, as a wave loads them straight from memory (no
// registers) or through registers.  A row's 16-byte pieces are exchanged by an
// XOR with its number, so that the score operand (16 rows, one piece) and the
// transposed reads of V (16 rows, two pieces) spread over all banks.
template <int D>
struct Rows16 {
    static constexpr int kRowBytes = 2 * D;
    static constexpr int kBytes = 16 * kRowBytes;                // K or V of 16 keys
    static constexpr int P = D / 8;                              // pieces a row
    static constexpr int kLoads = kBytes / 1024;                 // 1024 bytes a wave-wide load
    // piece c of row r lies at slot c ^ twist(r)
    static __device__ __forceinline__ int twist(int r) { return D == 128 ? r & 15 : (r >> 1) & 7; }
};

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) v4s lds_v4s;

// 16 bytes a lane to 1024 consecutive bytes of LDS at dst (wave-uniform), from
// base + offset or from src.  Written out because the compiler, which orders LDS
// reads of its own behind every such load it knows of, would empty the pipeline;
// the waits are the caller's.  No register is written.  ONCE: rows that no other
// workgroup reads are loaded non-temporal (16 sequences of 8-32K paged rows, one
// token 255 us without, 228 with; 26 tokens 318 / 290; 63 tokens over one cache,
// three blocks of query rows reading each row, 276 / 297).
template <bool ONCE>
__device__ __forceinline__ void load_to_lds(const char* base, uint32_t offset, char* dst) {
    const uint32_t at = (uint32_t)uniform((int)(uintptr_t)(lds_void*)dst);
    if constexpr (ONCE)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(at), "v"(offset), "s"(base)
                     : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(offset), "s"(base)
                     : "memory", "m0");
}
template <bool ONCE>
__device__ __forceinline__ void load_to_lds(const char* src, char* dst) {
    const uint32_t at = (uint32_t)uniform((int)(uintptr_t)(lds_void*)dst);
    if constexpr (ONCE)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(at), "v"(src) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(src) : "memory", "m0");
}

__device__ __forceinline__ u32x2 read_transposed(const char* p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)p));
}

// Score operand: row col of 16 rows at `ks`, pieces 4 kk + grp (GROUPED: those of
// load_queries).
template <int D, bool GROUPED = false>
__device__ __forceinline__ u32x4 key_operand(const char* ks, int kk) {
    using R = Rows16<D>;
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const int piece = GROUPED ? D / 32 * grp + kk : 4 * kk + grp;
    return *reinterpret_cast<const u32x4*>(ks + col * R::kRowBytes + 16 * (piece ^ R::twist(col)));
}

// Columns 16 md + col of rows 4 grp .. 4 grp + 3 of the 16 rows at `vs`.
template <int D>
__device__ __forceinline__ u32x2 value_operand(const char* vs, int md) {
    using R = Rows16<D>;
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const int row = 4 * grp + (col >> 2);                        // the row this lane names for the transpose
    return read_transposed(vs + row * R::kRowBytes + 16 * ((2 * md + ((col & 3) >> 1)) ^ R::twist(row)) + 8 * (col & 1));
}

// Where the rows of a cache lie: in one tensor, in blocks of a multiple of 16
// rows (the 16 rows that a wave loads at a time share one), in blocks of any
// size.
constexpr int kDense = 0, kBlocks16 = 1, kAnyBlocks = 2;

// A wave's view of the cache rows of one item: 16 consecutive rows into LDS.
// Where the 16 rows lie in one tensor or in one block, their first row is found
// on the scalar unit and a lane adds the same offsets each time.
template <int D, int PAGED>
struct RowLoader {
    using R = Rows16<D>;
    const char *kb, *vb;
    uint32_t ko[R::kLoads], vo[R::kLoads];
    int lrow, lslot;

    __device__ __forceinline__ RowLoader(const TreeParams& p) {
        const int lane = threadIdx.x & 63;
        lrow = lane / R::P;
        lslot = lane % R::P;
#pragma unroll
        for (int x = 0; x < R::kLoads; ++x) {
            const int r = x * (64 / R::P) + lrow, piece = 16 * (lslot ^ R::twist(r));
            ko[x] = 2 * r * (uint32_t)p.c.k_sn + piece;
            vo[x] = 2 * r * (uint32_t)p.c.v_sn + piece;
        }
    }
    __device__ __forceinline__ void item(const TreeParams& p, int64_t b, int h) {
        kb = reinterpret_cast<const char*>(p.c.k + h * p.c.k_sh + (PAGED ? 0 : b * p.c.k_sb));
        vb = reinterpret_cast<const char*>(p.c.v + h * p.c.v_sh + (PAGED ? 0 : b * p.c.v_sb));
    }
    // K (V false) or V of rows row .. row + 15
    template <bool V>
    __device__ __forceinline__ void load(const TreeParams& p, const Pages& pages, int stretch, int row, char* dst) const {
        if (p.row_blocks == 1) load_rows<V, true>(p, pages, stretch, row, dst);
        else load_rows<V, false>(p, pages, stretch, row, dst);
    }
    template <bool V, bool ONCE>
    __device__ __forceinline__ void load_rows(const TreeParams& p, const Pages& pages, int stretch, int row,
                                              char* dst) const {
        const char* base = V ? vb : kb;
        if constexpr (PAGED != kAnyBlocks) {
            int64_t at;
            if constexpr (PAGED) {
                const RowAt r = paged_row(p.c, pages, stretch, row);
                at = uniform(V ? r.v : r.k);
            } else {
                at = row * (V ? p.c.v_sn : p.c.k_sn);
            }
            base += 2 * at;
#pragma unroll
            for (int x = 0; x < R::kLoads; ++x) load_to_lds<ONCE>(base, V ? vo[x] : ko[x], dst + 1024 * x);
        } else {
#pragma unroll
            for (int x = 0; x < R::kLoads; ++x) {
                const int r = x * (64 / R::P) + lrow, piece = 16 * (lslot ^ R::twist(r));
                const RowAt at = paged_row(p.c, pages, stretch, row + r);
                load_to_lds<ONCE>(base + 2 * (V ? at.v : at.k) + piece, dst + 1024 * x);
            }
        }
    }
};

// A workgroup's LDS.  The rows come first, so that every address a load to LDS
// names fits the 16 bits its base register holds for certain.
template <int BYTES, int ROWS>
struct alignas(1024) TreeLds {
    char rows[BYTES];
    Pages pages;
    uint64_t seen[4][ROWS];       // drafted_seen's words, by wave
    int wild;                     // drafted values that are not finite
    static_assert(BYTES <= 65536, "addresses past 16 bits");
};

// The 16 rows from key0 on (draft: drafted ones) through registers, for rows
// that end before the 16th and for drafted values that are not finite: what
// does not exist becomes zero.
template <int D, bool F16, int PAGED>
struct StagedRows {
    using R = Rows16<D>;
    u32x4 k[R::kLoads], v[R::kLoads];

    __device__ __forceinline__ void load(const TreeParams& p, const Item& it, const Pages& pages, int stretch, bool draft,
                                         int key0) {
        const int lane = threadIdx.x & 63, lrow = lane / R::P, lslot = lane % R::P, rows = draft ? p.T : it.n;
#pragma unroll
        for (int y = 0; y < R::kLoads; ++y) {
            const int row = min(key0 + y * (64 / R::P) + lrow, rows - 1);
            const uint16_t *ks, *vs;
            if (draft) {
                ks = p.dk + it.b * p.dk_sb + row * p.dk_sn + it.h * p.dk_sh;
                vs = p.dv + it.b * p.dv_sb + row * p.dv_sn + it.h * p.dv_sh;
            } else {
                RowAt at;
                if constexpr (PAGED) at = paged_row(p.c, pages, stretch, row);
                else at = RowAt{it.b * p.c.k_sb + row * p.c.k_sn, it.b * p.c.v_sb + row * p.c.v_sn};
                ks = p.c.k + at.k + it.h * p.c.k_sh;
                vs = p.c.v + at.v + it.h * p.c.v_sh;
            }
            k[y] = *reinterpret_cast<const u32x4*>(ks + 8 * lslot);
            v[y] = *reinterpret_cast<const u32x4*>(vs + 8 * lslot);
        }
    }
    __device__ __forceinline__ void load_drafted(const TreeParams& p, const Item& it, int key0) {
        const int lane = threadIdx.x & 63, lrow = lane / R::P, lslot = lane % R::P;
#pragma unroll
        for (int y = 0; y < R::kLoads; ++y) {
            const int row = min(key0 + y * (64 / R::P) + lrow, p.T - 1);
            k[y] = *reinterpret_cast<const u32x4*>(p.dk + it.b * p.dk_sb + row * p.dk_sn + it.h * p.dk_sh + 8 * lslot);
            v[y] = *reinterpret_cast<const u32x4*>(p.dv + it.b * p.dv_sb + row * p.dv_sn + it.h * p.dv_sh + 8 * lslot);
        }
    }
    // Returns whether a value was taken out.
    __device__ __forceinline__ bool store(bool draft, int left, char* dst, int apart) {
        const int lane = threadIdx.x & 63, lrow = lane / R::P, lslot = lane % R::P;
        bool bad = false;
#pragma unroll
        for (int y = 0; y < R::kLoads; ++y) {
            const int r = y * (64 / R::P) + lrow;
            const bool in = r < left;
            u32x4 x = v[y];
            if (draft) x = finite_only<F16>(x, &bad);
            char* at = dst + r * R::kRowBytes + 16 * (lslot ^ R::twist(r));
            *reinterpret_cast<u32x4*>(at) = k[y];
            *reinterpret_cast<u32x4*>(at + apart) = u32x4{in ? x.x : 0u, in ? x.y : 0u, in ? x.z : 0u, in ? x.w : 0u};
        }
        return bad;
    }
};

// Merges the runs of every item that lies in more than one.  D / 4 lanes hold a
// row; SHARE groups of them take every SHARE-th run of it, four runs' loads
// side by side, and meet in LDS.
template <int D, bool F16, int SHARE>
__global__ void __launch_bounds__(256) tree_merge_kernel(TreeParams p, int rows_wg, int chunks) {
    using E = Elem<F16>;
    constexpr int kGroups = 256 / (D / 4), kRowsWg = kGroups / SHARE;
    __shared__ v4f join_o[SHARE > 1 ? kGroups : 1][D / 4];
    __shared__ float join_m[kGroups], join_l[kGroups];
    const int item = blockIdx.x / chunks;
    const int64_t b = item / p.Hk;
    const int h = item % p.Hk;
    const int group = threadIdx.x / (D / 4), part = group % SHARE, c = 4 * (threadIdx.x % (D / 4));
    const int row = (blockIdx.x % chunks) * kRowsWg + group / SHARE;

    const int tiles = item_tiles(p.deal, cache_length(p.c, b));
    int r0, r1;                                          // the item's runs
    if (p.deal.splits) {
        const int each = (uint32_t)(tiles + p.deal.splits - 1) / (uint32_t)p.deal.splits;
        r0 = item * p.deal.splits;
        r1 = r0 + (uint32_t)(tiles - 1) / (uint32_t)each;
    } else {
        // first tile of the item: tiles of the sequences before it
        const int lane = threadIdx.x & 63;
        int before = 0, all = 0;
        for (int b0 = 0; b0 < p.B; b0 += 64) {
            const int x = b0 + lane < p.B ? item_tiles(p.deal, cache_length(p.c, b0 + lane)) : 0;
            int lower = b0 + lane < b ? x : 0, any = x;
#pragma unroll
            for (int s = 1; s < 64; s <<= 1) {
                lower += __shfl_xor(lower, s, 64);
                any += __shfl_xor(any, s, 64);
            }
            before += lower;
            all += any;
        }
        const Deal deal(p.deal, uniform(all) * p.Hk);
        const int first = uniform(before) * p.Hk + h * tiles;
        r0 = deal.run_of(first);
        r1 = deal.run_of(first + tiles - 1);
    }
    if (r0 == r1) return;
    const int live = min(row, p.M - 1), rb = live / rows_wg, in = live - rb * rows_wg;
    const int64_t size = (int64_t)rows_wg * (D + 2);
    float M = kNegInf, L = 0.f;
    v4f acc = {0.f, 0.f, 0.f, 0.f};
    for (int r = r0 + part; r <= r1; r += 4 * SHARE) {
        float m[4], l[4];
        v4f o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int ri = min(r + i * SHARE, r1);
            // the run that starts the item keeps it in its second entry
            const float* e = p.part + (2 * ((int64_t)ri * p.row_blocks + rb) + (ri == r0)) * size;
            m[i] = e[rows_wg * D + in];
            l[i] = e[rows_wg * D + rows_wg + in];
            o[i] = *reinterpret_cast<const v4f*>(e + in * D + c);
        }
        float top = M;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (r + i * SHARE > r1) m[i] = kNegInf;
            top = fmaxf(top, m[i]);
        }
        const float base = top == kNegInf ? 0.f : top;
        const float old = fast_exp2(M - base);
        L *= old;
        acc *= old;
        M = top;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in_range = r + i * SHARE <= r1;
            const float f = in_range ? fast_exp2(m[i] - base) : 0.f;
            L += in_range ? f * l[i] : 0.f;
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[x] += in_range ? f * o[i][x] : 0.f;
        }
    }
    if constexpr (SHARE > 1) {
        join_o[group][c / 4] = acc;
        join_m[group] = M;
        join_l[group] = L;
        __syncthreads();
        if (part) return;
        float top = kNegInf;
#pragma unroll
        for (int i = 0; i < SHARE; ++i) top = fmaxf(top, join_m[group + i]);
        const float base = top == kNegInf ? 0.f : top;
        L = 0.f;
        acc = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < SHARE; ++i) {
            const float f = fast_exp2(join_m[group + i] - base);
            L += f * join_l[group + i];
            acc += f * join_o[group + i][c / 4];
        }
        M = top;
    }
    if (row >= p.M) return;
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
    bool whole() const { return runs == 1; }      // no item lies in two runs: nothing to merge
    size_t bytes(int64_t D) const { return whole() ? 0 : (size_t)slots * 2 * rows() * (D + 2) * sizeof(float); }
};

// Query rows (M a KV head) a workgroup holds: the fewest of 16, 32, 64 and 128
// that hold all of them (128 for more).  Runs: two workgroups a CU over all row
// blocks.
inline TreePlan plan_tree(int64_t M) {
    TreePlan t{};
    t.rw = M <= 32 ? 1 : M <= 64 ? 2 : 4;
    t.nt = M <= 16 ? 1 : 2;
    t.row_blocks = std::max(1, (int)((M + t.rows() - 1) / t.rows()));
    t.runs = std::max(1, 2 * device_cu_count() / t.row_blocks);
    t.slots = (int64_t)t.runs * t.row_blocks;
    return t;
}

// The merge's workgroups.  Runs an item has at most, on average: every group of
// lanes its own row where they are few, all groups one row where they are many.
struct MergePlan {
    bool shared;
    int chunks;                    // workgroups an item
};

inline MergePlan plan_merge(const TreePlan& plan, int64_t items, int64_t M, int64_t D) {
    const bool shared = plan.runs / items >= 8;
    const int64_t rows = shared ? 1 : 256 / (D / 4);
    return MergePlan{shared, (int)((M + rows - 1) / rows)};
}

template <int D, bool F16>
void launch_merge(const TreeParams& p, const TreePlan& plan, hipStream_t st) {
    if (plan.whole()) return;
    const MergePlan merge = plan_merge(plan, (int64_t)p.B * p.Hk, p.M, D);
    const dim3 merge_grid((unsigned)(p.B * p.Hk * merge.chunks));
    constexpr int kGroups = 256 / (D / 4);
    if (merge.shared)
        hipLaunchKernelGGL((tree_merge_kernel<D, F16, kGroups>), merge_grid, dim3(256), 0, st, p, plan.rows(), merge.chunks);
    else
        hipLaunchKernelGGL((tree_merge_kernel<D, F16, 1>), merge_grid, dim3(256), 0, st, p, plan.rows(), merge.chunks);
}

}  // namespace

}  // namespace slimkv
