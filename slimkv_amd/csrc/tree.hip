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

#include "tree.hpp"

namespace slimkv {

namespace {

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

template <int D, bool F16>
void launch_tree(const TreeParams& p, const TreePlan& plan, hipStream_t st) {
    const dim3 grid((unsigned)((plan.slots + kXcdCount - 1) / kXcdCount * kXcdCount));
    void (*kernel)(TreeParams);
    if (!p.c.table) kernel = tree_kernel<D, F16, kDense>(plan);
    else if (p.c.block.d % 16 == 0) kernel = tree_kernel<D, F16, kBlocks16>(plan);
    else kernel = tree_kernel<D, F16, kAnyBlocks>(plan);
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p);
    launch_merge<D, F16>(p, plan, st);
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
    return std::max<size_t>(plan_tree(a->drafted * (a->heads / a->kv_heads)).bytes(a->head_dim), 16);
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
    const TreePlan plan = plan_tree(a->drafted * (a->heads / a->kv_heads));
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
    p.deal = Dealing{p.B, p.Hk, kKeys, (p.T + kKeys - 1) / kKeys, plan.runs, 0};
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
