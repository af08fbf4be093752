// Attention of a tree of drafted tokens over a cache: every query row sees all
// rows of its sequence's cache and the drafted tokens its mask names.
//
// The T * G query rows of one KV head (row p = t * G + g) are the columns of
// the score MFMA: S^T = K . Q^T with K rows as A and the query rows held in
// registers as B, so the softmax statistics stay in a lane's column, and O^T =
// V^T . P^T with P^T straight from the score registers.  Weights are rounded once
// to the element type, since the matrix instruction takes both operands in it: at
// most half a step of sum p |v|, of either sign; their sum is fp32 and of the
// unrounded ones.  K and V rows go from memory straight to LDS, row by row; V is
// transposed by the LDS read.
//
// Up to 32 query rows a KV head the cache's bytes are the bound: tree_few_kernel,
// whose waves share nothing but the end (16 sequences of 8-32K paged rows, a
// token each: a call of 234 us for 1.34 GB, 5.7 TB/s; a copy moves 4.9-5.3).  More
// rows are bound by the matrix cores and by how well loads hide behind them:
// tree_many_kernel, 64 or 128 rows a workgroup (26 tokens on the same cache 293
// us, 4.6 TB/s; 63 tokens of 40 heads over 131071 rows 255 us, 664 TFLOP/s of
// needed work, 809 with the rows that fill up the last block of 128).  Figures
// beside a choice compare its two sides as they were when it was made.
//
// Schedule.  The tiles of 64 rows of all (sequence, KV head) items -- the cache's
// rows, then the drafted tokens' -- lie in a row and are dealt to two workgroups a
// CU in equal runs, whatever the lengths are (four a CU: 26 tokens 358 us instead
// of 318, six short chains 29 instead of 23); a run that holds part of an item
// leaves its unnormalised output, maxima and sums in the workspace for the merge
// kernel.  Each run exists once per block of query rows, side by side on one XCD,
// so that the blocks share the tiles in its L2.

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

// Query rows row0 + 16 nt + col as MFMA operands, zero past the last one.
template <int KS, int NT>
__device__ __forceinline__ void load_queries(const TreeParams& p, int64_t b, int h, int row0, u32x4 (&qr)[NT][KS]) {
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = row0 + 16 * nt + col;
        const int r = min(row, p.M - 1), t = r / p.G, g = r - t * p.G;
        const uint16_t* src = p.q + b * p.q_sb + t * p.q_sl + (int64_t)(h * p.G + g) * p.q_sh + 8 * grp;
        const bool ok = row < p.M;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(src + 32 * kk);
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

// Score operand: row col of 16 rows at `ks`, pieces 4 kk + grp.
template <int D>
__device__ __forceinline__ u32x4 key_operand(const char* ks, int kk) {
    using R = Rows16<D>;
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    return *reinterpret_cast<const u32x4*>(ks + col * R::kRowBytes + 16 * ((4 * kk + grp) ^ R::twist(col)));
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

// ---------------------------------------------------------------------------
// up to 32 query rows a KV head: bound by the cache's bytes
// ---------------------------------------------------------------------------

// A wave owns 16 keys of each tile and works for itself on its own LDS ring,
// without a barrier: the next two tiles are on their way while one is computed.
template <int D, bool F16, int NT, int PAGED>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) tree_few_kernel(TreeParams p) {
    using E = Elem<F16>;
    using R = Rows16<D>;
    constexpr int KS = D / 32, MD = D / 16, kRows = 16 * NT, kPart = kRows * (D + 2), kWave = 4 * R::kBytes;
    constexpr int kBytes = 4 * kWave > 12 * kPart ? 4 * kWave : 12 * kPart;      // rings, or the join of three waves
    __shared__ TreeLds<kBytes, kRows> sh;
    char* lds = sh.rows;
    Pages& pages = sh.pages;
    auto& seen = sh.seen;
    int& wild = sh.wild;

    const int run = slot_of_block();
    const Deal deal(p.deal, total_tiles(p.c, p.deal));
    if (run >= deal.runs) return;
    int pos = deal.begin(run);
    const int end = deal.begin(run + 1);
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    char* ring = lds + wave * kWave;
    RowLoader<D, PAGED> loader(p);

    while (pos < end) {
        const Item it = item_at(p, pos, end);
        const int64_t b = it.b;
        const int whole_tiles = it.n / kKeys, cached = (it.n + kKeys - 1) / kKeys;
        const int streamed = max(it.t0, min(it.t1, whole_tiles));        // tiles [t0, streamed) by the ring
        int stretch = it.t0;                                             // first tile of the pages held
        loader.item(p, b, it.h);
        __syncthreads();                                                 // the item before is done with LDS
        if (threadIdx.x == 0) wild = 0;
        if constexpr (PAGED) {
            if (it.t0 < cached) load_pages(p.c, b, it.t0, it.n, pages);
        }
        __syncthreads();

        auto fetch = [&](int t) {
            char* dst = ring + (t & 1) * 2 * R::kBytes;
            loader.template load_rows<false, true>(p, pages, stretch, t * kKeys + 16 * wave, dst);
            loader.template load_rows<true, true>(p, pages, stretch, t * kKeys + 16 * wave, dst + R::kBytes);
        };
        u32x4 qr[NT][KS];
        load_queries<KS, NT>(p, b, it.h, 0, qr);
        // the first of the tiles that pass through registers, asked for early
        StagedRows<D, F16, PAGED> staged;
        auto rows_of = [&](int t) { return t >= cached ? p.T : it.n; };
        auto key_of = [&](int t) { return (t >= cached ? t - cached : t) * kKeys + 16 * wave; };
        const bool early = streamed < it.t1 && key_of(streamed) < rows_of(streamed) &&
                           !(PAGED && streamed < cached && streamed >= stretch + page_tiles(p.c));
        if (early) staged.load(p, it, pages, stretch, streamed >= cached, key_of(streamed));
        if (it.t0 < streamed) fetch(it.t0);
        if (it.t0 + 1 < streamed) fetch(it.t0 + 1);

        v4f o[NT][MD];
        float m[NT], l[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt] = kNegInf;
            l[nt] = 0.f;
#pragma unroll
            for (int md = 0; md < MD; ++md) o[nt][md] = v4f{0.f, 0.f, 0.f, 0.f};
        }

        // 16 keys at ks; visible(nt, i): key 4 grp + i for column col
        auto compute = [&](const char* ks, auto visible) {
            v4f s[NT][1];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[nt][0] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                const u32x4 a = key_operand<D>(ks, kk);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][0] = E::mma32(a, qr[nt][kk], s[nt][0]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[nt][0][i] = visible(nt, i) ? s[nt][0][i] : kNegInf;
                softmax_step<1, MD, F16>(s[nt], p.scale_log2, m[nt], l[nt], o[nt]);
            }
#pragma unroll
            for (int md = 0; md < MD; ++md) {
                const u32x2 a = value_operand<D>(ks + R::kBytes, md);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    o[nt][md] = E::mma16(a, u32x2{E::pack(s[nt][0][0], s[nt][0][1]), E::pack(s[nt][0][2], s[nt][0][3])},
                                         o[nt][md]);
            }
        };

        for (int t = it.t0; t < streamed; ++t) {
            // the loads of tile t are done once only the next tile's are open
            if (t + 1 < streamed) {
                if constexpr (D == 128) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
                else asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            compute(ring + (t & 1) * 2 * R::kBytes, [](int, int) { return true; });
            if (t + 2 < streamed) {
                if constexpr (PAGED) {
                    if (t + 2 >= stretch + page_tiles(p.c)) {
                        __syncthreads();
                        stretch = t + 2;
                        load_pages(p.c, b, stretch, it.n, pages);
                        __syncthreads();
                    }
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // tile t is read
                fetch(t + 2);
            }
        }

        // the cache's last rows and the drafted tokens
        for (int t = streamed; t < it.t1; ++t) {
            const bool draft = t >= cached;
            if constexpr (PAGED) {
                if (!draft && t >= stretch + page_tiles(p.c)) {
                    __syncthreads();
                    stretch = t;
                    load_pages(p.c, b, stretch, it.n, pages);
                    __syncthreads();
                }
            }
            const int key0 = key_of(t), left = rows_of(t) - key0;
            if (left <= 0) continue;
            if (t > streamed || !early) staged.load(p, it, pages, stretch, draft, key0);
            if (draft) drafted_seen(p, b, 0, kRows, key0 - 16 * wave, seen[wave]);
            wave_fence();
            if (staged.store(draft, left, ring, R::kBytes)) wild = 1;
            wave_fence();
            uint32_t bits[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                bits[nt] = draft ? (uint32_t)(seen[wave][min(16 * nt + col, p.M - 1) / p.G] >> (16 * wave + 4 * grp)) & 15u
                                 : (1u << max(0, min(4, left - 4 * grp))) - 1;
            compute(ring, [&](int nt, int i) { return (bits[nt] >> i & 1u) != 0; });
            wave_fence();
        }

        __syncthreads();
        join_keys<MD, NT, 4>(reinterpret_cast<float*>(lds), kRows, 0, wave, m, l, o);
        if (wave == 0) {
            float* part = p.part + (2 * (int64_t)run + (it.t0 == 0)) * kPart;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int row = 16 * nt + col;
                if (wild) add_unbounded<MD, F16>(p, b, it.h, 0, p.T, row, o[nt]);
                finish_rows<MD, F16>(p, b, it.h, row, row, kRows, it.t0 == 0 && it.t1 == it.tiles, part, m[nt], l[nt], o[nt]);
            }
        }
        pos += it.t1 - it.t0;
    }
}

// ---------------------------------------------------------------------------
// more than 32 query rows a KV head: bound by the matrix cores
// ---------------------------------------------------------------------------

// A tile of 64 rows lies in LDS as four groups of 16 (K, then V), each loaded by
// one wave, two tiles side by side.
template <int D, bool F16, int RW, int PAGED>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) tree_many_kernel(TreeParams p) {
    using R = Rows16<D>;
    using E = Elem<F16>;
    constexpr int NT = 2, KS = D / 32, MD = D / 16;
    constexpr int KW = 4 / RW, MT = 4 / KW;                // waves side by side on a tile's keys, 16-key groups of each
    constexpr int kRows = 16 * RW * NT, kPart = kRows * (D + 2);
    constexpr int kTile = 8 * R::kBytes, kApart = 4 * R::kBytes;
    constexpr int kJoin = KW > 1 ? 4 * (KW - 1) * kPart : 0;
    constexpr int kBytes = 2 * kTile > kJoin ? 2 * kTile : kJoin;
    __shared__ TreeLds<kBytes, 16 * NT> sh;
    char* lds = sh.rows;
    Pages& pages = sh.pages;
    auto& seen = sh.seen;
    int& wild = sh.wild;

    const int slot = slot_of_block();
    const int run = (uint32_t)slot / (uint32_t)p.row_blocks, rb = slot - run * p.row_blocks;
    const Deal deal(p.deal, total_tiles(p.c, p.deal));
    if (run >= deal.runs) return;
    int pos = deal.begin(run);
    const int end = deal.begin(run + 1);

    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int rw = wave % RW, kw = wave / RW;
    const int row0 = rb * kRows + rw * 16 * NT;           // the wave's first query row
    const int key0 = kw * 16 * MT;                        // the wave's first key in a tile
    RowLoader<D, PAGED> loader(p);

    while (pos < end) {
        const Item it = item_at(p, pos, end);
        const int64_t b = it.b;
        const int whole_tiles = it.n / kKeys, cached = (it.n + kKeys - 1) / kKeys;
        const int streamed = max(it.t0, min(it.t1, whole_tiles));        // tiles [t0, streamed) straight to LDS
        int stretch = it.t0;
        loader.item(p, b, it.h);
        __syncthreads();                                   // the item before is done with LDS
        if (threadIdx.x == 0) wild = 0;
        if constexpr (PAGED) {
            if (it.t0 < cached) load_pages(p.c, b, it.t0, it.n, pages);
            __syncthreads();
        }
        auto fetch_k = [&](int t) {
            if constexpr (PAGED) {
                if (t >= stretch + page_tiles(p.c)) {      // V of the tiles before is on its way
                    __syncthreads();
                    stretch = t;
                    load_pages(p.c, b, stretch, it.n, pages);
                    __syncthreads();
                }
            }
            loader.template load<false>(p, pages, stretch, t * kKeys + 16 * wave, lds + (t & 1) * kTile + wave * R::kBytes);
        };
        auto fetch_v = [&](int t) {
            loader.template load<true>(p, pages, stretch, t * kKeys + 16 * wave,
                                       lds + (t & 1) * kTile + kApart + wave * R::kBytes);
        };
        if (it.t0 < streamed) {
            fetch_k(it.t0);
            fetch_v(it.t0);
        }
        if (it.t0 + 1 < streamed) fetch_k(it.t0 + 1);
        u32x4 qr[NT][KS];
        load_queries<KS, NT>(p, b, it.h, row0, qr);
        v4f o[NT][MD];
        float m[NT], l[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt] = kNegInf;
            l[nt] = 0.f;
#pragma unroll
            for (int md = 0; md < MD; ++md) o[nt][md] = v4f{0.f, 0.f, 0.f, 0.f};
        }

        // the wave's MT groups of 16 keys of the tile at `tile`: scores, softmax, values
        auto scores = [&](const char* tile, v4f(&s)[NT][MT]) {
            const char* ks = tile + kw * MT * R::kBytes;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][mt] = v4f{0.f, 0.f, 0.f, 0.f};
            u32x4 a[KS][MT];                               // two k-steps' rows asked for ahead of their products
            auto read = [&](int kk) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) a[kk][mt] = key_operand<D>(ks + mt * R::kBytes, kk);
            };
            read(0);
            read(1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                if (kk + 2 < KS) read(kk + 2);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) s[nt][mt] = E::mma32(a[kk][mt], qr[nt][kk], s[nt][mt]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto softmax = [&](v4f(&s)[NT][MT], u32x4(&pb)[MT / 2][NT]) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                softmax_step<MT, MD, F16>(s[nt], p.scale_log2, m[nt], l[nt], o[nt]);
#pragma unroll
                for (int ss = 0; ss < MT / 2; ++ss)
                    pb[ss][nt] =
                        u32x4{E::pack(s[nt][2 * ss][0], s[nt][2 * ss][1]), E::pack(s[nt][2 * ss][2], s[nt][2 * ss][3]),
                              E::pack(s[nt][2 * ss + 1][0], s[nt][2 * ss + 1][1]),
                              E::pack(s[nt][2 * ss + 1][2], s[nt][2 * ss + 1][3])};
            }
        };
        auto values = [&](const char* tile, const u32x4(&pb)[MT / 2][NT]) {
            const char* vs = tile + kApart + kw * MT * R::kBytes;
            constexpr int kGroups = MT / 2 * MD / 4;       // four 16-column operands a group, one group ahead
            u32x4 a[kGroups][4];
            auto read = [&](int g) {
                const int ss = g / (MD / 4), m0 = g % (MD / 4) * 4;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const u32x2 lo = value_operand<D>(vs + 2 * ss * R::kBytes, m0 + i);
                    const u32x2 hi = value_operand<D>(vs + (2 * ss + 1) * R::kBytes, m0 + i);
                    a[g][i] = u32x4{lo.x, lo.y, hi.x, hi.y};
                }
            };
            read(0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const int ss = g / (MD / 4), m0 = g % (MD / 4) * 4;
                if (g + 1 < kGroups) read(g + 1);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) o[nt][m0 + i] = E::mma32(a[g][i], pb[ss][nt], o[nt][m0 + i]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };

        // K of tile t + 2 is asked for once all waves are past the scores of
        // tile t, V of tile t + 1 once all are past the values of tile t - 1,
        // so every load has one and a half tiles' time.  A wave waits for its
        // own rows, by the number of younger loads, then for the others' at
        // the barrier (whose LDS reads are done by then).
        for (int t = it.t0; t < streamed; ++t) {
            const bool more = t + 1 < streamed;
            v4f s[NT][MT];
            u32x4 pb[MT / 2][NT];
            if (!more) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(R::kLoads) : "memory");
            else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * R::kLoads) : "memory");
            if (more) fetch_v(t + 1);
            scores(lds + (t & 1) * kTile, s);
            softmax(s, pb);
            if (!more) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * R::kLoads) : "memory");
            if (t + 2 < streamed) fetch_k(t + 2);
            values(lds + (t & 1) * kTile, pb);
        }
        // the cache's last rows and the drafted tokens
        for (int t = streamed; t < it.t1; ++t) {
            const bool draft = t >= cached;
            const int first = (draft ? t - cached : t) * kKeys;
            __syncthreads();
            if constexpr (PAGED) {
                if (!draft && t >= stretch + page_tiles(p.c)) {
                    stretch = t;
                    load_pages(p.c, b, stretch, it.n, pages);
                    __syncthreads();
                }
            }
            {
                StagedRows<D, F16, PAGED> staged;
                const int key = first + 16 * wave;
                staged.load(p, it, pages, stretch, draft, key);
                if (draft) drafted_seen(p, b, row0, 16 * NT, first, seen[wave]);
                if (staged.store(draft, (draft ? p.T : it.n) - key, lds + wave * R::kBytes, kApart)) wild = 1;
            }
            __syncthreads();
            v4f s[NT][MT];
            u32x4 pb[MT / 2][NT];
            scores(lds, s);
            const int from = min(row0, p.M - 1) / p.G, left = it.n - first - key0 - 4 * grp;
            const uint64_t all = left <= 0 ? 0 : left >= 64 ? ~(uint64_t)0 : ((uint64_t)1 << left) - 1;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint64_t word =
                    draft ? seen[wave][min(row0 + 16 * nt + col, p.M - 1) / p.G - from] >> (key0 + 4 * grp) : all;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[nt][mt][i] = word >> (16 * mt + i) & 1 ? s[nt][mt][i] : kNegInf;
            }
            softmax(s, pb);
            values(lds, pb);
        }
        __syncthreads();

        join_keys<MD, NT, KW>(reinterpret_cast<float*>(lds), kRows, rw * 16 * NT, kw, m, l, o);
        if (kw == 0) {
            float* part = p.part + (2 * (int64_t)slot + (it.t0 == 0)) * kPart;
            const int j0 = max(0, it.t0 - cached) * kKeys, j1 = min(p.T, max(0, it.t1 - cached) * kKeys);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int in = rw * 16 * NT + 16 * nt + col, row = rb * kRows + in;
                if (wild) add_unbounded<MD, F16>(p, b, it.h, j0, j1, row, o[nt]);
                finish_rows<MD, F16>(p, b, it.h, row, in, kRows, it.t0 == 0 && it.t1 == it.tiles, part, m[nt], l[nt],
                                     o[nt]);
            }
        }
        pos += it.t1 - it.t0;
    }
}

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
    const int tiles = item_tiles(p.deal, cache_length(p.c, b));
    const Deal deal(p.deal, uniform(all) * p.Hk);
    const int first = uniform(before) * p.Hk + h * tiles, r0 = deal.run_of(first), r1 = deal.run_of(first + tiles - 1);
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
    if (!scale_usable(a->scale)) return fail(SLIMKV_EINVAL, "tree attention: the softmax scale must lie in [1e-18, 1e18]");
    return SLIMKV_OK;
}

template <int D, bool F16, int PAGED>
auto tree_kernel(const TreePlan& plan) -> void (*)(TreeParams) {
    if (plan.rw == 4) return tree_many_kernel<D, F16, 4, PAGED>;
    if (plan.rw == 2) return tree_many_kernel<D, F16, 2, PAGED>;
    return plan.nt == 2 ? tree_few_kernel<D, F16, 2, PAGED> : tree_few_kernel<D, F16, 1, PAGED>;
}

// The merge's workgroups.  Runs an item has at most, on average: every group of
// lanes its own row where they are few, all groups one row where they are many.
struct MergePlan {
    bool shared;
    int chunks;                    // workgroups an item
};

MergePlan plan_merge(const TreePlan& plan, int64_t items, int64_t M, int64_t D) {
    const bool shared = plan.runs / items >= 8;
    const int64_t rows = shared ? 1 : 256 / (D / 4);
    return MergePlan{shared, (int)((M + rows - 1) / rows)};
}

template <int D, bool F16>
void launch_tree(const TreeParams& p, const TreePlan& plan, hipStream_t st) {
    const dim3 grid((unsigned)((plan.slots + kXcdCount - 1) / kXcdCount * kXcdCount));
    void (*kernel)(TreeParams);
    if (!p.c.table) kernel = tree_kernel<D, F16, kDense>(plan);
    else if (p.c.block.d % 16 == 0) kernel = tree_kernel<D, F16, kBlocks16>(plan);
    else kernel = tree_kernel<D, F16, kAnyBlocks>(plan);
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p);
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
    if (r.table && (r.block_size <= 0 || r.num_blocks <= 0 || r.num_blocks > 0x7fffffff || r.t_cols <= 0 ||
                    (batch > 1 && r.t_sb < r.t_cols && r.t_sb != 0) || r.block_size > ((int64_t)1 << 30) ||
                    r.t_cols > ((int64_t)1 << 30) || r.keys > r.t_cols * r.block_size))
        return fail(SLIMKV_EINVAL, w + ": invalid page layout (cache rows past the block table?)");
    const int64_t outer = r.table ? r.num_blocks : batch, rows = r.table ? r.block_size : r.keys;
    if (r.keys > 0 && (!rows_aligned(r.k, {{outer, r.k_sb}, {rows, r.k_sn}, {kv_heads, r.k_sh}}) ||
                       (need_v && !rows_aligned(r.v, {{outer, r.v_sb}, {rows, r.v_sn}, {kv_heads, r.v_sh}}))))
        return fail(SLIMKV_EINVAL, w + ": cache rows must start on 16-byte boundaries (strides multiples of 8)");
    for (int64_t s : {r.k_sn, need_v ? r.v_sn : r.k_sn})
        if (rows > 1 && (s < head_dim || s >= (1 << 23)))
            return fail(SLIMKV_EUNSUP, w + ": cache rows must lie [head_dim, 2^23) elements apart");
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
    for (int64_t s : {a->dk_sn, a->dv_sn})
        if (T > 1 && (s < a->head_dim || s >= (1 << 23)))
            return fail(SLIMKV_EUNSUP, "tree attention: drafted rows must lie [head_dim, 2^23) elements apart");
    const TreePlan plan = plan_tree(a);
    if (!plan.whole() &&
        (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < plan.bytes(a->head_dim)))
        return fail(SLIMKV_EWORKSPACE, "tree attention: workspace missing, misaligned or too small");
    p.q = static_cast<const uint16_t*>(a->q); p.q_sb = a->q_sb; p.q_sl = a->q_sl; p.q_sh = a->q_sh;
    p.dk = static_cast<const uint16_t*>(a->draft_k); p.dk_sb = a->dk_sb; p.dk_sn = a->dk_sn; p.dk_sh = a->dk_sh;
    p.dv = static_cast<const uint16_t*>(a->draft_v); p.dv_sb = a->dv_sb; p.dv_sn = a->dv_sn; p.dv_sh = a->dv_sh;
    p.mask = a->mask; p.m_sb = a->m_sb; p.m_sl = a->m_sl;
    p.out = static_cast<uint16_t*>(a->out); p.o_sb = a->o_sb; p.o_sl = a->o_sl; p.o_sh = a->o_sh;
    p.lse = a->lse;
    p.B = (int)B; p.T = (int)T; p.Hq = (int)Hq; p.Hk = (int)Hk; p.G = (int)(Hq / Hk);
    p.M = p.T * p.G;
    p.row_blocks = plan.row_blocks;
    p.deal = Dealing{p.B, p.Hk, kKeys, (p.T + kKeys - 1) / kKeys, plan.runs};
    p.scale_log2 = (float)(a->scale * 1.4426950408889634);
    p.part = static_cast<float*>(workspace);
    if (B * Hk * p.M > 0x7fffffff || (!plan.whole() && !launchable(B * Hk * plan_merge(plan, B * Hk, p.M, a->head_dim).chunks, 256)) ||
        B * Hk * ((a->cache.keys + T) / kKeys + 2) > 0x7fffffff)
        return fail(SLIMKV_EINVAL, "tree attention: too many rows for one call");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->head_dim == 128) {
        if (a->dtype == SLIMKV_DTYPE_F16) launch_tree<128, true>(p, plan, st);
        else launch_tree<128, false>(p, plan, st);
    } else {
        if (a->dtype == SLIMKV_DTYPE_F16) launch_tree<64, true>(p, plan, st);
        else launch_tree<64, false>(p, plan, st);
    }
    return check_hip(hipGetLastError(), "tree attention launch");
}
