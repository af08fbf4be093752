// Attention of new tokens over a cache held in 4 bits: every query row sees all
// rows of its sequence's cache and the drafted tokens its mask names
// (include/slimkv/quant_cache.h has the format).
//
// The mathematics and the split are those of the attention over full-width rows
// (tree.hpp): the T * G query rows of one KV head are the columns of the score
// MFMA, S^T = K . Q^T, O^T = V^T . P^T with P^T straight from the score registers,
// and the tiles of all (sequence, KV head) items are dealt to two workgroups a CU in
// equal runs.  The cached rows come as codes and scales and become MFMA operands
// in registers, two elements an instruction, exactly (a 4-bit float times a power
// of two fits the element type):
//   K   a lane reads 16 (D = 64: 8) bytes of one row, one block of 32 elements
//       (half of one), so one scale serves them.  The order of the elements in the
//       product is free as long as the queries follow it (load_queries GROUPED).
//   V   the product wants a lane's keys side by side.  The pages hold groups of 16
//       rows so that a lane reads its column's codes of its four keys; a byte is two
//       columns of one key and one block, and pairs of keys are then joined.
// So the rows pass no LDS where they serve one wave's columns.

#include "quant.hpp"
#include "tree.hpp"

namespace slimkv {

namespace {

struct QuantParams {
    TreeParams t;
    PoolView z;
};

// 16 rows of K and V as a lane holds them: K of row `col`, elements D / 4 grp on;
// V of rows 4 grp .. 4 grp + 3, columns col + 16 md; their scales.
template <int D>
struct Group {
    typedef uint32_t vec __attribute__((ext_vector_type(D / 32)));
    vec k, v, vs;
    uint32_t ks;
};

// What a lane adds to a group's address.
template <int D>
struct GroupOffsets {
    uint32_t k, v, ks, vs;
    __device__ __forceinline__ GroupOffsets() {
        const uint32_t lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
        k = col * (D / 2) + grp * (D / 8);
        v = lane * (D / 8);
        ks = col * (D / 32) + (D == 128 ? grp : grp >> 1);
        vs = grp * (D / 8);
    }
};

typedef const __attribute__((address_space(4))) int64_t* table_entries;

// A wave's way to the groups of one item: the page numbers on the scalar unit.
template <int D>
struct GroupLoader {
    GroupOffsets<D> off;
    const uint8_t* head;              // page 0 of the item's head (no table: the sequence's page)
    const int64_t* entries;

    __device__ __forceinline__ void item(const PoolView& z, int64_t b, int h) {
        head = z.pages + h * z.p_sh + (z.table ? 0 : b * z.p_sb);
        entries = z.table ? z.table + b * z.t_sb : nullptr;
    }
    // The table entry of the page that holds row `row`, as it stands there.
    __device__ __forceinline__ int64_t entry(const PoolView& z, int row) const {
        return entries ? ((table_entries)(uintptr_t)entries)[quotient(row, z.block)] : 0;
    }
    // The group of rows row .. row + 15.
    __device__ __forceinline__ void load(const PoolView& z, int64_t entry, int row, Group<D>& x) const {
        typedef typename Group<D>::vec vec;
        int64_t page = 0, slot = row;
        if (entries) {
            page = table_page(entry, z.num_pages);
            if (page < 0) {
                report_bad_page(z.status);
                page = 0;
            }
            slot = row - quotient(row, z.block) * (int)z.block.d;
        }
        const uint8_t* base = head + page * z.p_sb;
        const uint8_t* codes = base + slot * (D / 2);
        const uint8_t* scales = base + slot * (D / 32);
        x.k = *reinterpret_cast<const vec*>(codes + off.k);
        x.v = *reinterpret_cast<const vec*>(codes + z.v_at + off.v);
        x.ks = (scales + z.ks_at)[off.ks];
        x.vs = *reinterpret_cast<const vec*>(scales + z.vs_at + off.vs);
    }
};

// Score operand of step kk.
template <int D, bool F16>
__device__ __forceinline__ u32x4 key_values(const Group<D>& x, int kk) {
    return eight_values<F16>(x.k[kk], x.ks << 23);
}

// The scales of the lane's four V rows behind `left` of the group's rows: none,
// since a block behind the end may hold anything.
template <int D>
__device__ __forceinline__ void drop_scales(Group<D>& x, int left) {
    const int grp = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (4 * grp + j < left) continue;
        if constexpr (D == 128) x.vs[j] = 0;
        else x.vs[j / 2] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
    }
}

// Value operands: the lane's four keys of column 16 md + col, two elements a
// dword, for all md.
template <int D, bool F16>
__device__ __forceinline__ void value_values(const Group<D>& x, u32x2 (&out)[D / 16]) {
    using C = Codes<F16>;
    uint32_t pair[4][D / 32];           // key j: columns 32 pr + col (low) and 32 pr + 16 + col (high)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (D == 128) {
            const uint32_t w = x.v[j], f = x.vs[j];
            pair[j][0] = C::template values<0>(w, f << 23);
            pair[j][1] = C::template values<1>(w, f << 15);
            pair[j][2] = C::template values<2>(w, f << 7);
            pair[j][3] = C::template values<3>(w, f >> 1);
        } else {
            const uint32_t w = x.v[j / 2], f = x.vs[j / 2];
            if (j & 1) {
                pair[j][0] = C::template values<2>(w, f << 7);
                pair[j][1] = C::template values<3>(w, f >> 1);
            } else {
                pair[j][0] = C::template values<0>(w, f << 23);
                pair[j][1] = C::template values<1>(w, f << 15);
            }
        }
    }
#pragma unroll
    for (int pr = 0; pr < D / 32; ++pr) {
        out[2 * pr] = u32x2{__builtin_amdgcn_perm(pair[1][pr], pair[0][pr], 0x05040100u),
                            __builtin_amdgcn_perm(pair[3][pr], pair[2][pr], 0x05040100u)};
        out[2 * pr + 1] = u32x2{__builtin_amdgcn_perm(pair[1][pr], pair[0][pr], 0x07060302u),
                                __builtin_amdgcn_perm(pair[3][pr], pair[2][pr], 0x07060302u)};
    }
}

// A workgroup's LDS: tiles or staged rows, joined states.
template <int BYTES, int ROWS>
struct alignas(1024) QuantLds {
    char rows[BYTES];
    uint64_t seen[4][ROWS];       // drafted_seen's words, by wave
    int wild;                     // drafted values that are not finite
};

// ---------------------------------------------------------------------------
// up to 32 query rows a KV head
// ---------------------------------------------------------------------------

constexpr int kUnit = 4;                       // groups of 16 rows that a wave takes of a tile
constexpr int kFewRows = 4 * 16 * kUnit;       // rows of a tile

// A wave owns 64 rows of each tile and works for itself in its registers: the next
// tile's codes are on their way while one is computed.
template <int D, bool F16, int NT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) quant_few_kernel(QuantParams qp) {
    const TreeParams& p = qp.t;
    const PoolView& z = qp.z;
    using E = Elem<F16>;
    using R = Rows16<D>;
    constexpr int KS = D / 32, MD = D / 16, kRows = 16 * NT, kPart = kRows * (D + 2), kWave = 2 * R::kBytes;
    constexpr int kBytes = 4 * kWave > 12 * kPart ? 4 * kWave : 12 * kPart;      // staged rows, or the join of three waves
    __shared__ QuantLds<kBytes, kRows> sh;

    const int run = slot_of_block();
    const Deal deal(p.deal, total_tiles(p.c, p.deal));
    if (run >= deal.runs) return;
    int pos = deal.begin(run);
    const int end = deal.begin(run + 1);
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    char* staging = sh.rows + wave * kWave;
    GroupLoader<D> loader;

    while (pos < end) {
        const Item it = item_at(p, pos, end);
        const int64_t b = it.b;
        const int cached = (it.n + kFewRows - 1) / kFewRows;
        const int stop = max(it.t0, min(it.t1, cached));                 // tiles [t0, stop) of the cache
        loader.item(z, b, it.h);
        __syncthreads();                                                 // the item before is done with LDS
        if (threadIdx.x == 0) sh.wild = 0;
        __syncthreads();
        u32x4 qr[NT][KS];
        load_queries<KS, NT, true>(p, b, it.h, 0, qr);

        v4f o[NT][MD];
        float m[NT], l[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt] = kNegInf;
            l[nt] = 0.f;
#pragma unroll
            for (int md = 0; md < MD; ++md) o[nt][md] = v4f{0.f, 0.f, 0.f, 0.f};
        }

        // the wave's rows of tile t, those past the last group again the last one
        const int last_row = (it.n - 1) & ~15;
        auto row_of = [&](int t, int u) { return min(t * kFewRows + (wave * kUnit + u) * 16, last_row); };
        struct Unit {
            Group<D> x[kUnit];
        };
        auto load = [&](int t, Unit& unit) {
#pragma unroll
            for (int u = 0; u < kUnit; ++u) {
                const int row = row_of(t, u);
                loader.load(z, loader.entry(z, row), row, unit.x[u]);
            }
        };
        auto compute = [&](int t, Unit& unit) {
            const int left = it.n - (t * kFewRows + wave * kUnit * 16);
            if (left <= 0) return;
            v4f s[NT][kUnit];
#pragma unroll
            for (int u = 0; u < kUnit; ++u) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][u] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) {
                    const u32x4 a = key_values<D, F16>(unit.x[u], kk);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) s[nt][u] = E::mma32(a, qr[nt][kk], s[nt][u]);
                }
            }
            if (left < kUnit * 16) {
#pragma unroll
                for (int u = 0; u < kUnit; ++u) {
                    drop_scales<D>(unit.x[u], left - 16 * u);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[nt][u][i] = 16 * u + 4 * grp + i < left ? s[nt][u][i] : kNegInf;
                }
            }
            u32x4 pb[kUnit / 2][NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                softmax_step<kUnit, MD, F16>(s[nt], p.scale_log2, m[nt], l[nt], o[nt]);
#pragma unroll
                for (int ss = 0; ss < kUnit / 2; ++ss)
                    pb[ss][nt] =
                        u32x4{E::pack(s[nt][2 * ss][0], s[nt][2 * ss][1]), E::pack(s[nt][2 * ss][2], s[nt][2 * ss][3]),
                              E::pack(s[nt][2 * ss + 1][0], s[nt][2 * ss + 1][1]),
                              E::pack(s[nt][2 * ss + 1][2], s[nt][2 * ss + 1][3])};
            }
#pragma unroll
            for (int ss = 0; ss < kUnit / 2; ++ss) {
                u32x2 lo[MD], hi[MD];
                value_values<D, F16>(unit.x[2 * ss], lo);
                value_values<D, F16>(unit.x[2 * ss + 1], hi);
#pragma unroll
                for (int md = 0; md < MD; ++md)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        o[nt][md] = E::mma32(u32x4{lo[md].x, lo[md].y, hi[md].x, hi[md].y}, pb[ss][nt], o[nt][md]);
            }
        };

        if (it.t0 < stop) {
            Unit even, odd;
            load(it.t0, even);
            for (int t = it.t0;;) {
                load(min(t + 1, stop - 1), odd);
                compute(t, even);
                if (++t >= stop) break;
                load(min(t + 1, stop - 1), even);
                compute(t, odd);
                if (++t >= stop) break;
            }
        }

        // the drafted tokens, 16 a wave
        for (int t = stop; t < it.t1; ++t) {
            const int first = (t - cached) * kKeys, key0 = first + 16 * wave;
            if (!p.dk || p.T <= key0) continue;
            StagedRows<D, F16, kDense> staged;
            staged.load_drafted(p, it, key0);
            drafted_seen(p, b, 0, kRows, first, sh.seen[wave]);
            wave_fence();
            if (staged.store(true, p.T - key0, staging, R::kBytes)) sh.wild = 1;
            wave_fence();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint32_t bits =
                    (uint32_t)(sh.seen[wave][min(16 * nt + col, p.M - 1) / p.G] >> (16 * wave + 4 * grp)) & 15u;
                v4f s[1] = {v4f{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) s[0] = E::mma32(key_operand<D, true>(staging, kk), qr[nt][kk], s[0]);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[0][i] = bits >> i & 1u ? s[0][i] : kNegInf;
                softmax_step<1, MD, F16>(s, p.scale_log2, m[nt], l[nt], o[nt]);
                const u32x2 pb = {E::pack(s[0][0], s[0][1]), E::pack(s[0][2], s[0][3])};
#pragma unroll
                for (int md = 0; md < MD; ++md)
                    o[nt][md] = E::mma16(value_operand<D>(staging + R::kBytes, md), pb, o[nt][md]);
            }
            wave_fence();
        }

        __syncthreads();
        join_keys<MD, NT, 4>(reinterpret_cast<float*>(sh.rows), kRows, 0, wave, m, l, o);
        if (wave == 0) {
            float* part = p.part + (2 * (int64_t)run + (it.t0 == 0)) * kPart;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int row = 16 * nt + col;
                if (sh.wild) add_unbounded<MD, F16>(p, b, it.h, 0, p.T, row, o[nt]);
                finish_rows<MD, F16>(p, b, it.h, row, row, kRows, it.t0 == 0 && it.t1 == it.tiles, part, m[nt], l[nt], o[nt]);
            }
        }
        pos += it.t1 - it.t0;
    }
}

// ---------------------------------------------------------------------------
// more than 32 query rows a KV head: bound by the matrix cores
// ---------------------------------------------------------------------------

// Four waves share a tile of 64 rows.  Each turns one group of 16 into operands
// and leaves them in LDS in the order in which lanes take them (16 bytes a lane side
// by side: no bank is asked twice), two tiles side by side.
template <int D, bool F16, int RW>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) quant_many_kernel(QuantParams qp) {
    const TreeParams& p = qp.t;
    const PoolView& z = qp.z;
    using R = Rows16<D>;
    using E = Elem<F16>;
    constexpr int NT = 2, KS = D / 32, MD = D / 16;
    constexpr int KW = 4 / RW, MT = 4 / KW;                // waves side by side on a tile's keys, 16-key groups of each
    constexpr int kRows = 16 * RW * NT, kPart = kRows * (D + 2);
    constexpr int kTile = 8 * R::kBytes, kApart = 4 * R::kBytes;
    constexpr int kJoin = KW > 1 ? 4 * (KW - 1) * kPart : 0;
    constexpr int kBytes = 2 * kTile > kJoin ? 2 * kTile : kJoin;
    __shared__ QuantLds<kBytes, 16 * NT> sh;
    char* lds = sh.rows;

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
    GroupLoader<D> loader;

    while (pos < end) {
        const Item it = item_at(p, pos, end);
        const int64_t b = it.b;
        const int cached = (it.n + kKeys - 1) / kKeys;
        const int stop = max(it.t0, min(it.t1, cached));
        loader.item(z, b, it.h);
        __syncthreads();                                   // the item before is done with LDS
        if (threadIdx.x == 0) sh.wild = 0;
        u32x4 qr[NT][KS];
        load_queries<KS, NT, true>(p, b, it.h, row0, qr);
        v4f o[NT][MD];
        float m[NT], l[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt] = kNegInf;
            l[nt] = 0.f;
#pragma unroll
            for (int md = 0; md < MD; ++md) o[nt][md] = v4f{0.f, 0.f, 0.f, 0.f};
        }

        // the wave's group of tile t: asked for, and left in LDS as operands
        Group<D> raw;
        const int last_row = (it.n - 1) & ~15;
        auto fetch = [&](int t) {
            const int row = min(t * kKeys + 16 * wave, last_row);
            loader.load(z, loader.entry(z, row), row, raw);
        };
        auto put = [&](int t) {
            char* tile = lds + (t & 1) * kTile;
            drop_scales<D>(raw, it.n - (t * kKeys + 16 * wave));
#pragma unroll
            for (int kk = 0; kk < KS; ++kk)
                *reinterpret_cast<u32x4*>(tile + (wave * KS + kk) * 1024 + 16 * lane) = key_values<D, F16>(raw, kk);
            u32x2 v[MD];
            value_values<D, F16>(raw, v);
#pragma unroll
            for (int md = 0; md < MD; ++md)
                *reinterpret_cast<u32x2*>(tile + kApart + ((wave >> 1) * MD + md) * 1024 + 16 * lane + 8 * (wave & 1)) = v[md];
        };

        // the wave's MT groups of 16 keys: scores, softmax, values; the operands by key(mt, kk) and value(ss, md)
        auto scores = [&](auto key, v4f(&s)[NT][MT]) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][mt] = v4f{0.f, 0.f, 0.f, 0.f};
            u32x4 a[KS][MT];                               // two steps' rows asked for ahead of their products
            auto read = [&](int kk) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) a[kk][mt] = key(mt, kk);
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
        auto values = [&](auto value, const u32x4(&pb)[MT / 2][NT]) {
            constexpr int kGroups = MT / 2 * MD / 4;       // four 16-column operands a group, one group ahead
            u32x4 a[kGroups][4];
            auto read = [&](int g) {
                const int ss = g / (MD / 4), m0 = g % (MD / 4) * 4;
#pragma unroll
                for (int i = 0; i < 4; ++i) a[g][i] = value(ss, m0 + i);
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

        if (it.t0 < stop) {
            fetch(it.t0);
            put(it.t0);
            if (it.t0 + 1 < stop) fetch(it.t0 + 1);
        }
        __syncthreads();
        for (int t = it.t0; t < stop; ++t) {
            if (t + 1 < stop) put(t + 1);
            if (t + 2 < stop) fetch(t + 2);
            const char* tile = lds + (t & 1) * kTile;
            v4f s[NT][MT];
            u32x4 pb[MT / 2][NT];
            scores([&](int mt, int kk) {
                return *reinterpret_cast<const u32x4*>(tile + ((kw * MT + mt) * KS + kk) * 1024 + 16 * lane);
            }, s);
            const int left = it.n - t * kKeys - key0;
            if (left < 16 * MT) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[nt][mt][i] = 16 * mt + 4 * grp + i < left ? s[nt][mt][i] : kNegInf;
            }
            softmax(s, pb);
            values([&](int ss, int md) {
                return *reinterpret_cast<const u32x4*>(tile + kApart + ((kw * (MT / 2) + ss) * MD + md) * 1024 + 16 * lane);
            }, pb);
            __syncthreads();
        }
        // the drafted tokens
        for (int t = stop; p.dk && t < it.t1; ++t) {
            const int first = (t - cached) * kKeys;
            __syncthreads();
            {
                StagedRows<D, F16, kDense> staged;
                const int key = first + 16 * wave;
                staged.load_drafted(p, it, key);
                drafted_seen(p, b, row0, 16 * NT, first, sh.seen[wave]);
                if (staged.store(true, p.T - key, lds + wave * R::kBytes, kApart)) sh.wild = 1;
            }
            __syncthreads();
            const char* ks = lds + kw * MT * R::kBytes;
            v4f s[NT][MT];
            u32x4 pb[MT / 2][NT];
            scores([&](int mt, int kk) { return key_operand<D, true>(ks + mt * R::kBytes, kk); }, s);
            const int from = min(row0, p.M - 1) / p.G;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint64_t word = sh.seen[wave][min(row0 + 16 * nt + col, p.M - 1) / p.G - from] >> (key0 + 4 * grp);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[nt][mt][i] = word >> (16 * mt + i) & 1 ? s[nt][mt][i] : kNegInf;
            }
            softmax(s, pb);
            values([&](int ss, int md) {
                const u32x2 lo = value_operand<D>(ks + kApart + 2 * ss * R::kBytes, md);
                const u32x2 hi = value_operand<D>(ks + kApart + (2 * ss + 1) * R::kBytes, md);
                return u32x4{lo.x, lo.y, hi.x, hi.y};
            }, pb);
        }
        __syncthreads();

        join_keys<MD, NT, KW>(reinterpret_cast<float*>(lds), kRows, rw * 16 * NT, kw, m, l, o);
        if (kw == 0) {
            float* part = p.part + (2 * (int64_t)slot + (it.t0 == 0)) * kPart;
            const int j0 = max(0, it.t0 - cached) * kKeys, j1 = min(p.T, max(0, it.t1 - cached) * kKeys);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int in = rw * 16 * NT + 16 * nt + col, row = rb * kRows + in;
                if (sh.wild) add_unbounded<MD, F16>(p, b, it.h, j0, j1, row, o[nt]);
                finish_rows<MD, F16>(p, b, it.h, row, in, kRows, it.t0 == 0 && it.t1 == it.tiles, part, m[nt], l[nt],
                                     o[nt]);
            }
        }
        pos += it.t1 - it.t0;
    }
}

int check_attention(const slimkv_quantized_attention_args* a) {
    if (!a || (!a->q && a->tokens > 0 && a->batch > 0)) return fail(SLIMKV_EINVAL, "quantized attention: null pointer");
    if (a->head_dim != 64 && a->head_dim != 128)
        return fail(SLIMKV_EUNSUP, "quantized attention: head_dim must be 64 or 128");
    if (a->dtype != SLIMKV_DTYPE_BF16 && a->dtype != SLIMKV_DTYPE_F16)
        return fail(SLIMKV_EUNSUP, "quantized attention: element type must be bf16 or fp16");
    if (a->batch < 0 || a->batch > 65535 || a->tokens < 0 || a->tokens > kMaxDrafted || a->heads <= 0 || a->kv_heads <= 0 ||
        a->heads % a->kv_heads || a->heads > 4096 || a->heads / a->kv_heads > 256)
        return fail(SLIMKV_EINVAL, "quantized attention: invalid sizes");
    if (!scale_usable(a->scale))
        return fail(SLIMKV_EINVAL, "quantized attention: the softmax scale must lie in [1e-18, 1e18]");
    return SLIMKV_OK;
}

int64_t query_rows(const slimkv_quantized_attention_args* a) { return a->tokens * (a->heads / a->kv_heads); }

template <int D, bool F16>
void launch_attention(const QuantParams& p, const TreePlan& plan, hipStream_t st) {
    const dim3 grid((unsigned)((plan.slots + kXcdCount - 1) / kXcdCount * kXcdCount));
    void (*kernel)(QuantParams) = plan.rw == 4   ? quant_many_kernel<D, F16, 4>
                                  : plan.rw == 2 ? quant_many_kernel<D, F16, 2>
                                  : plan.nt == 2 ? quant_few_kernel<D, F16, 2>
                                                 : quant_few_kernel<D, F16, 1>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p);
    launch_merge<D, F16>(p.t, plan, st);
}

}  // namespace

}  // namespace slimkv

using namespace slimkv;

extern "C" size_t slimkv_quantized_attention_workspace(const slimkv_quantized_attention_args* a) {
    if (check_attention(a) != SLIMKV_OK) return 0;
    return std::max<size_t>(plan_tree(query_rows(a)).bytes(a->head_dim), 16);
}

extern "C" int slimkv_quantized_attention(const slimkv_quantized_attention_args* a, void* workspace,
                                          size_t workspace_bytes, void* stream) {
    const int code = check_attention(a);
    if (code != SLIMKV_OK) return code;
    if (a->batch == 0 || a->tokens == 0) return SLIMKV_OK;
    const bool draft = a->draft_k != nullptr;
    if (!a->out || draft != (a->draft_v != nullptr) || (!draft && a->mask))
        return fail(SLIMKV_EINVAL, "quantized attention: null pointer (drafted K and V come together, a mask with them)");
    QuantParams qp{};
    TreeParams& p = qp.t;
    const int64_t B = a->batch, T = a->tokens, Hq = a->heads, Hk = a->kv_heads, D = a->head_dim;
    const int view = pool_view(a->cache, B, Hk, D, "quantized attention", &qp.z);
    if (view != SLIMKV_OK) return view;
    if (a->keys < 0 || a->keys > qp.z.capacity)
        return fail(SLIMKV_EINVAL, "quantized attention: keys must lie within the cache's rows");
    if (!rows_aligned(a->q, {{B, a->q_sb}, {T, a->q_sl}, {Hq, a->q_sh}}) ||
        (draft && (!rows_aligned(a->draft_k, {{B, a->dk_sb}, {T, a->dk_sn}, {Hk, a->dk_sh}}) ||
                   !rows_aligned(a->draft_v, {{B, a->dv_sb}, {T, a->dv_sn}, {Hk, a->dv_sh}}))) ||
        !rows_aligned(a->out, {{B, a->o_sb}, {T, a->o_sl}, {Hq, a->o_sh}}))
        return fail(SLIMKV_EINVAL, "quantized attention: rows must start on 16-byte boundaries (strides multiples of 8)");
    for (int64_t s : {a->dk_sn, a->dv_sn})
        if (draft && T > 1 && (s < D || s >= (1 << 23)))
            return fail(SLIMKV_EUNSUP, "quantized attention: drafted rows must lie [head_dim, 2^23) elements apart");
    const TreePlan plan = plan_tree(query_rows(a));
    if (!plan.whole() &&
        (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < plan.bytes(D)))
        return fail(SLIMKV_EWORKSPACE, "quantized attention: workspace missing, misaligned or too small");
    p.c.lengths = a->lengths; p.c.keys = (int)a->keys;
    p.q = static_cast<const uint16_t*>(a->q); p.q_sb = a->q_sb; p.q_sl = a->q_sl; p.q_sh = a->q_sh;
    p.dk = static_cast<const uint16_t*>(a->draft_k); p.dk_sb = a->dk_sb; p.dk_sn = a->dk_sn; p.dk_sh = a->dk_sh;
    p.dv = static_cast<const uint16_t*>(a->draft_v); p.dv_sb = a->dv_sb; p.dv_sn = a->dv_sn; p.dv_sh = a->dv_sh;
    p.mask = a->mask; p.m_sb = a->m_sb; p.m_sl = a->m_sl;
    p.out = static_cast<uint16_t*>(a->out); p.o_sb = a->o_sb; p.o_sl = a->o_sl; p.o_sh = a->o_sh;
    p.lse = a->lse;
    p.B = (int)B; p.T = (int)T; p.Hq = (int)Hq; p.Hk = (int)Hk; p.G = (int)(Hq / Hk);
    p.M = p.T * p.G;
    p.row_blocks = plan.row_blocks;
    const int tile = plan.rw == 1 ? kFewRows : kKeys;
    // without drafted tokens a tile without work, so that a sequence without rows has a run that writes its output
    p.deal = Dealing{p.B, p.Hk, tile, draft ? (p.T + kKeys - 1) / kKeys : 1, plan.runs};
    p.scale_log2 = (float)(a->scale * 1.4426950408889634);
    p.part = static_cast<float*>(workspace);
    if (B * Hk * p.M > 0x7fffffff || (!plan.whole() && !launchable(B * Hk * plan_merge(plan, B * Hk, p.M, D).chunks, 256)) ||
        B * Hk * ((a->keys + T) / kKeys + 2) > 0x7fffffff)
        return fail(SLIMKV_EINVAL, "quantized attention: too many rows for one call");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (D == 128) {
        if (a->dtype == SLIMKV_DTYPE_F16) launch_attention<128, true>(qp, plan, st);
        else launch_attention<128, false>(qp, plan, st);
    } else {
        if (a->dtype == SLIMKV_DTYPE_F16) launch_attention<64, true>(qp, plan, st);
        else launch_attention<64, false>(qp, plan, st);
    }
    return check_hip(hipGetLastError(), "quantized attention launch");
}
