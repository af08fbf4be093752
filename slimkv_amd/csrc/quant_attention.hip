// Attention of new tokens over a cache held in 4 bits: every query row sees all
// rows of its sequence's cache and the drafted tokens its mask names
// (include/slimkv/quant_cache.h has the format).
//
// The mathematics and the split are those of the attention over full-width rows
// (tree.hpp): the T * G query rows of one KV head are the columns of the score
// MFMA, S^T = K . Q^T, O^T = V^T . P^T with P^T straight from the score registers,
// and the tiles of all (sequence, KV head) items are dealt to two workgroups a CU in
// equal runs.  The cached rows come as codes and scales and become MFMA operands
// in registers, two elements an instruction, as rows are read back: exactly in bf16,
// and in fp16 what fp16 wrote (bf16 writes some that fp16 rounds or that pass its
// end):
//   K   a lane reads 16 (D = 64: 8) bytes of one row, one block of 32 elements
//       (half of one), so one scale serves them.  The order of the elements in the
//       product is free as long as the queries follow it (load_queries GROUPED).
//   V   the product wants a lane's keys side by side.  The pages hold groups of 16
//       rows so that a lane reads its column's codes of its four keys; a byte is two
//       columns of one key and one block, and pairs of keys are then joined.
// So the rows pass no LDS where they serve one wave's columns.
//
// Up to 32 query rows a KV head the cache's bytes are the bound, 136 a row and head
// of 128 (quant_few_kernel: 16 sequences of 8-32K rows, a token each, 357 MB in 64
// us, 5.6 TB/s, the call with its merge 71; a copy moves 5.2, non-temporal reads alone
// 7.2).  More rows are bound by the instructions of the softmax and of the conversions
// beside the products and by the power that they take together (quant_many_kernel: 26
// tokens on the same cache 202 us a call, 690 TFLOP/s of needed work, 850 with the rows
// that fill up the last tiles; 63 tokens of 40 heads over 131071 rows 214 us, 790 and
// 960; four windows of 1024 tokens over 32768 rows 2.07 ms, 1080, and over none 140 us,
// 245, since drafted tiles behind a block's last token are worked on as well; the
// library's 8192^3 product reaches 1100-1140).  Figures beside a choice compare its two
// sides as they were when it was made.
//
// Not taken: the product that takes 4-bit operands itself
// (v_mfma_scale_f32_16x16x128_f8f6f4, the queries cut into exact 8-bit parts).  Its
// sums are off by up to 1e-4 of sum |q k|, those of 16-bit products by 1e-7.

#include "quant.hpp"
#include "tree.hpp"

namespace slimkv {

namespace {

struct QuantParams {
    TreeParams t;
    PoolView z;
};

// The kernel's arguments, read where they are used: kept in scalar registers
// over the whole kernel they push each other out.
__device__ __forceinline__ const QuantParams& parameters() {
    auto args = (const __attribute__((address_space(4))) QuantParams*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(args));
    return *(const QuantParams*)args;
}

// The tiles that a workgroup has to work on, item by item; of a split item its part
// of that alone.
struct Share {
    int pos, end, splits;

    // False: none.
    __device__ __forceinline__ bool take(const TreeParams& p, int run) {
        splits = p.deal.splits;
        pos = run;
        end = run + 1;
        if (splits) return run < p.B * p.Hk * splits;
        const Deal deal(p.deal, total_tiles(p.c, p.deal));
        pos = deal.begin(run);
        end = deal.begin(run + 1);
        return run < deal.runs;
    }
    __device__ __forceinline__ Item item(const TreeParams& p) const {
        if (!splits) return item_at(p, pos, end);
        const int item = (uint32_t)pos / (uint32_t)splits;
        Item it;
        it.b = (uint32_t)item / (uint32_t)p.Hk;
        it.h = item - (int)it.b * p.Hk;
        it.n = uniform(cache_length(p.c, it.b));
        it.tiles = item_tiles(p.deal, it.n);
        const int each = (uint32_t)(it.tiles + splits - 1) / (uint32_t)splits;
        it.t0 = min(it.tiles, (pos - item * splits) * each);
        it.t1 = min(it.tiles, it.t0 + each);
        return it;
    }
    __device__ __forceinline__ void done(const Item& it) { pos += splits ? 1 : it.t1 - it.t0; }
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

// Where groups of 16 rows lie, 64 of them at a time, one a lane: no load of codes
// waits for the table, whose next 64 entries are on their way meanwhile.
struct Places {
    const int64_t* entries;           // the sequence's row of the table; none: one page
    int64_t entry;                    // asked for
    uint32_t page, slot;              // held

    // The lane's next group begins at `row`.
    __device__ __forceinline__ void ask(const PoolView& z, int row) {
        entry = entries ? entries[quotient(row, z.block)] : 0;
    }
    __device__ __forceinline__ void take(const PoolView& z, int row) {
        page = 0;
        slot = row;
        if (entries) {
            const int64_t at = table_page(entry, z.num_pages);
            if (at < 0) report_bad_page(z.status);
            page = at < 0 ? 0u : (uint32_t)at;
            slot = row - quotient(row, z.block) * (int)z.block.d;
        }
    }
};

// A wave's way to the groups of one item.
template <int D>
struct GroupLoader {
    const uint8_t* head;              // page 0 of the item's head (no table: the sequence's page)
    int64_t p_sb, v_at, ks_at, vs_at;
    Places places;

    __device__ __forceinline__ GroupLoader(const PoolView& z, int64_t b, int h)
        : head(z.pages + h * z.p_sh + (z.table ? 0 : b * z.p_sb)), p_sb(z.p_sb), v_at(z.v_at), ks_at(z.ks_at),
          vs_at(z.vs_at) {
        places.entries = z.table ? z.table + b * z.t_sb : nullptr;
    }
    struct Parts {
        const uint8_t *codes, *scales;
    };
    // K's codes and scales of the group that lane `at` holds the place of, but for the page's offsets.
    __device__ __forceinline__ Parts parts(int at) const {
        const uint32_t page = __builtin_amdgcn_readlane(places.page, at), slot = __builtin_amdgcn_readlane(places.slot, at);
        const uint8_t* base = head + page * p_sb;
        return Parts{base + (int64_t)slot * (D / 2), base + (int64_t)slot * (D / 32)};
    }
    // ONCE: codes that no other workgroup reads are loaded non-temporal (16 sequences of 8-32K rows, one token 79.5 us
    // without, 71.3 with; 26 tokens 202.5 / 199.8).
    template <bool ONCE>
    __device__ __forceinline__ void load(const GroupOffsets<D>& off, int at, Group<D>& x) const {
        typedef typename Group<D>::vec vec;
        const Parts from = parts(at);
        const vec* k = reinterpret_cast<const vec*>(from.codes + off.k);
        const vec* v = reinterpret_cast<const vec*>(from.codes + v_at + off.v);
        x.k = ONCE ? __builtin_nontemporal_load(k) : *k;
        x.v = ONCE ? __builtin_nontemporal_load(v) : *v;
        x.ks = (from.scales + ks_at)[off.ks];
        x.vs = *reinterpret_cast<const vec*>(from.scales + vs_at + off.vs);
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
__device__ __forceinline__ void drop_scales(typename Group<D>::vec& scales, int left) {
    const int grp = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (4 * grp + j < left) continue;
        if constexpr (D == 128) scales[j] = 0;
        else scales[j / 2] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
    }
}

// Value operands of columns 32 pr + col and 32 pr + 16 + col: the lane's four keys,
// two elements a dword.
template <int D, bool F16>
__device__ __forceinline__ void value_values(const typename Group<D>::vec& codes, const typename Group<D>::vec& scales,
                                             int pr, u32x2 (&out)[2]) {
    using C = Codes<F16>;
    uint32_t pair[4];                   // key j: both columns
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int byte = D == 128 ? pr : 2 * (j & 1) + pr;
        const uint32_t w = codes[D == 128 ? j : j / 2], f = scales[D == 128 ? j : j / 2];
        pair[j] = byte == 0   ? C::template values<0>(w, f << 23)
                  : byte == 1 ? C::template values<1>(w, f << 15)
                  : byte == 2 ? C::template values<2>(w, f << 7)
                              : C::template values<3>(w, f >> 1);
    }
    out[0] = u32x2{__builtin_amdgcn_perm(pair[1], pair[0], 0x05040100u), __builtin_amdgcn_perm(pair[3], pair[2], 0x05040100u)};
    out[1] = u32x2{__builtin_amdgcn_perm(pair[1], pair[0], 0x07060302u), __builtin_amdgcn_perm(pair[3], pair[2], 0x07060302u)};
}

// A workgroup's LDS: tiles or staged rows, joined states.
template <int BYTES, int WAVES, int ROWS>
struct alignas(1024) QuantLds {
    char rows[BYTES];
    uint64_t seen[WAVES][ROWS];   // drafted_seen's words, by wave
    int wild;                     // drafted values that are not finite
};

// The softmax of NT columns' scores, in two steps with one branch between them, so
// that the exponentials lie in one block with the products that take them and
// with the conversion of V.  First the maxima: where none moves (and none is so
// large that products are rounded first, as in softmax_step) nothing else happens.
template <int NT, int MT, int MD, bool F16>
struct Softmax {
    float factor[NT], base[NT];       // exponent of score s: factor s - base
    float m[NT], l[NT];
    v4f o[NT][MD];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt] = kNegInf;
            l[nt] = 0.f;
#pragma unroll
            for (int md = 0; md < MD; ++md) o[nt][md] = v4f{0.f, 0.f, 0.f, 0.f};
        }
    }
    __device__ __forceinline__ void move(v4f (&s)[NT][MT], float scale_log2) {
        float top[NT];
        bool moves = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float mx = kNegInf;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[nt][mt][i]);
            mx = rows_max(mx);
            top[nt] = fmaxf(m[nt], base_of<F16>(rounded_product(mx, scale_log2)));
            factor[nt] = scale_log2;
            base[nt] = top[nt] == kNegInf ? 0.f : top[nt];
            moves |= top[nt] != m[nt] || __builtin_fabsf(base[nt]) >= kFarBase;
        }
        if (!__ballot(moves)) return;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float alpha = fast_exp2(m[nt] - base[nt]);
            m[nt] = top[nt];
            l[nt] *= alpha;
#pragma unroll
            for (int md = 0; md < MD; ++md) o[nt][md] *= alpha;
            if (__builtin_fabsf(base[nt]) >= kFarBase) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[nt][mt][i] = far_exponent(s[nt][mt][i], scale_log2, base[nt]);
                factor[nt] = 1.f;
                base[nt] = 0.f;
            }
        }
    }
    // Two weights, rounded to the element type, since the matrix instruction takes both operands in it: at most half a step
    // of sum p |v|, of either sign (16 sequences of 8-32K rows: the outputs' error against 64 bits 0.00167 where the
    // output's own rounding is 0.00166; six short chains 0.00177 / 0.00165).  Their sum before that joins `sum`.
    __device__ __forceinline__ uint32_t weigh(int nt, float a, float b, float& sum) const {
        const float pa = fast_exp2(__builtin_fmaf(a, factor[nt], -base[nt]));
        const float pb = fast_exp2(__builtin_fmaf(b, factor[nt], -base[nt]));
        sum += pa + pb;
        return Elem<F16>::pack(pa, pb);
    }
    // The weights of a column's scores as operands of two groups of 16 keys each.
    __device__ __forceinline__ void weigh(const v4f (&s)[NT][MT], u32x4 (&pb)[MT / 2][NT]) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float sum = 0.f;
#pragma unroll
            for (int x = 0; x < 2 * MT; ++x) pb[x / 4][nt][x % 4] = weigh(nt, s[nt][x / 2][2 * (x & 1)], s[nt][x / 2][2 * (x & 1) + 1], sum);
            l[nt] += sum;
        }
    }
};

// ---------------------------------------------------------------------------
// up to 32 query rows a KV head
// ---------------------------------------------------------------------------

// Groups of 16 rows that a wave takes of a tile: four with up to 16 query rows, two
// with up to 32 (four spill 73 registers).
constexpr int few_groups(int nt) { return nt == 1 ? 4 : 2; }

// A wave owns 64 (32) rows of each tile and works for itself in its registers: the
// next tile's codes are on their way while one is computed.
template <int D, bool F16, int NT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) quant_few_kernel(QuantParams) {
    using E = Elem<F16>;
    using R = Rows16<D>;
    constexpr int KS = D / 32, MD = D / 16, kRows = 16 * NT, kPart = kRows * (D + 2), kWave = 2 * R::kBytes;
    constexpr int kUnit = few_groups(NT), kFewRows = 64 * kUnit;                 // rows of a tile
    constexpr int kBytes = 4 * kWave > 12 * kPart ? 4 * kWave : 12 * kPart;      // staged rows, or the join of three waves
    __shared__ QuantLds<kBytes, 4, kRows> sh;

    const int run = slot_of_block();
    Share share;
    if (!share.take(parameters().t, run)) return;
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    char* staging = sh.rows + wave * kWave;

    while (share.pos < share.end) {
        const Item it = share.item(parameters().t);
        if (it.t0 == it.t1) return;                                      // a split behind the item's last tile
        const int64_t b = it.b;
        const int cached = (it.n + kFewRows - 1) / kFewRows;
        const int stop = max(it.t0, min(it.t1, cached));                 // tiles [t0, stop) of the cache
        __syncthreads();                                                 // the item before is done with LDS
        if (threadIdx.x == 0) sh.wild = 0;
        __syncthreads();
        // the wave's groups of 16 tiles from `base` on, one a lane; those past the last group again the last one
        const PoolView& z = parameters().z;
        GroupLoader<D> loader(z, b, it.h);
        const int last_row = (it.n - 1) & ~15;
        int base = it.t0;
        auto row_of = [&](int from) { return min((from + lane / kUnit) * kFewRows + (wave * kUnit + lane % kUnit) * 16, last_row); };
        if (it.t0 < stop) loader.places.ask(z, row_of(base));
        u32x4 qr[NT][KS];
        load_queries<KS, NT, true>(parameters().t, b, it.h, 0, qr);
        const float scale_log2 = parameters().t.scale_log2;

        Softmax<NT, kUnit, MD, F16> x;
        x.clear();

        struct Unit {
            Group<D> x[kUnit];
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
                    drop_scales<D>(unit.x[u].vs, left - 16 * u);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[nt][u][i] = 16 * u + 4 * grp + i < left ? s[nt][u][i] : kNegInf;
                }
            }
            x.move(s, scale_log2);
            u32x4 pb[kUnit / 2][NT];
            x.weigh(s, pb);
#pragma unroll
            for (int ss = 0; ss < kUnit / 2; ++ss) {
#pragma unroll
                for (int pr = 0; pr < MD / 2; ++pr) {
                    u32x2 lo[2], hi[2];
                    value_values<D, F16>(unit.x[2 * ss].v, unit.x[2 * ss].vs, pr, lo);
                    value_values<D, F16>(unit.x[2 * ss + 1].v, unit.x[2 * ss + 1].vs, pr, hi);
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            x.o[nt][2 * pr + i] = E::mma32(u32x4{lo[i].x, lo[i].y, hi[i].x, hi[i].y}, pb[ss][nt], x.o[nt][2 * pr + i]);
                }
            }
        };

        if (it.t0 < stop) {
            const GroupOffsets<D> off;
            loader.places.take(z, row_of(base));
            loader.places.ask(z, row_of(base + 64 / kUnit));
            auto load = [&](int t, Unit& unit) {
                if (t >= base + 64 / kUnit) {
                    base += 64 / kUnit;
                    loader.places.take(z, row_of(base));
                    loader.places.ask(z, row_of(base + 64 / kUnit));
                }
#pragma unroll
                for (int u = 0; u < kUnit; ++u) loader.template load<true>(off, (t - base) * kUnit + u, unit.x[u]);
            };
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

        const TreeParams& p = parameters().t;
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
                softmax_step<1, MD, F16>(s, scale_log2, x.m[nt], x.l[nt], x.o[nt]);
                const u32x2 pb = {E::pack(s[0][0], s[0][1]), E::pack(s[0][2], s[0][3])};
#pragma unroll
                for (int md = 0; md < MD; ++md)
                    x.o[nt][md] = E::mma16(value_operand<D>(staging + R::kBytes, md), pb, x.o[nt][md]);
            }
            wave_fence();
        }

        __syncthreads();
        join_keys<MD, NT, 4>(reinterpret_cast<float*>(sh.rows), kRows, 0, wave, x.m, x.l, x.o);
        if (wave == 0) {
            float* part = p.part + (2 * (int64_t)run + (it.t0 == 0)) * kPart;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int row = 16 * nt + col;
                if (sh.wild) add_unbounded<MD, F16>(p, b, it.h, 0, p.T, row, x.o[nt]);
                finish_rows<MD, F16>(p, b, it.h, row, row, kRows, it.t0 == 0 && it.t1 == it.tiles, part, x.m[nt], x.l[nt], x.o[nt]);
            }
        }
        share.done(it);
    }
}

// ---------------------------------------------------------------------------
// more than 32 query rows a KV head
// ---------------------------------------------------------------------------

// Four waves share tiles of 64 rows: RW of them side by side on the query rows, 32
// each, 4 / RW on a tile's keys.  Each wave turns one group of 16 rows into
// operands and leaves them in LDS in the order in which lanes take them (16 bytes a
// lane side by side: no bank is asked twice), two tiles side by side.
template <int D, bool F16, int RW>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) quant_many_kernel(QuantParams) {
    using R = Rows16<D>;
    using E = Elem<F16>;
    constexpr int NT = 2, KS = D / 32, MD = D / 16;
    constexpr int KW = 4 / RW, MT = 4 / KW;                // waves side by side on a tile's keys, 16-key groups of each
    constexpr int kRows = 16 * RW * NT, kPart = kRows * (D + 2);
    constexpr int kTile = 8 * R::kBytes, kApart = 4 * R::kBytes;
    constexpr int kJoin = KW > 1 ? 4 * (KW - 1) * kPart : 0;
    constexpr int kBytes = 2 * kTile > kJoin ? 2 * kTile : kJoin;
    __shared__ QuantLds<kBytes, 4, 16 * NT> sh;
    char* lds = sh.rows;

    const int slot = slot_of_block();
    Share share;
    {
        const TreeParams& p = parameters().t;
        if (!share.take(p, (uint32_t)slot / (uint32_t)p.row_blocks)) return;
    }
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int rw = wave % RW, kw = wave / RW;
    const int key0 = kw * 16 * MT;                        // the wave's first key in a tile

    while (share.pos < share.end) {
        const Item it = share.item(parameters().t);
        if (it.t0 == it.t1) return;                                      // a split behind the item's last tile
        const int64_t b = it.b;
        const int cached = (it.n + kKeys - 1) / kKeys;
        const int stop = max(it.t0, min(it.t1, cached));
        __syncthreads();                                   // the item before is done with LDS
        if (threadIdx.x == 0) sh.wild = 0;
        // the wave's groups of 64 tiles from `base` on, one a lane; those past the last group again the last one
        const PoolView& z = parameters().z;
        GroupLoader<D> loader(z, b, it.h);
        const int last_row = (it.n - 1) & ~15;
        int base = it.t0;
        auto row_of = [&](int from) { return min((from + lane) * kKeys + 16 * wave, last_row); };
        if (it.t0 < stop) loader.places.ask(z, row_of(base));
        int row0;                                          // the wave's first query row
        bool idle;                                         // past the last one: this wave makes operands only
        bool once;                                         // no other block of query rows reads the codes
        u32x4 qr[NT][KS];
        float scale_log2;
        {
            const TreeParams& p = parameters().t;
            row0 = (slot - (uint32_t)slot / (uint32_t)p.row_blocks * p.row_blocks) * kRows + rw * 16 * NT;
            idle = row0 >= p.M;
            once = p.row_blocks == 1;
            load_queries<KS, NT, true>(p, b, it.h, row0, qr);
            scale_log2 = p.scale_log2;
        }
        Softmax<NT, MT, MD, F16> x;
        x.clear();

        // scores, softmax and values of the wave's keys; the operands by key(mt, kk) and value(ss, md), unseen scores by
        // hide
        auto attend = [&](auto key, auto value, auto hide) {
            v4f s[NT][MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][mt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) {
                    const u32x4 a = key(mt, kk);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) s[nt][mt] = E::mma32(a, qr[nt][kk], s[nt][mt]);
                }
            }
            hide(s);
            x.move(s, scale_log2);
            u32x4 pb[MT / 2][NT];
            x.weigh(s, pb);
#pragma unroll
            for (int ss = 0; ss < MT / 2; ++ss)
#pragma unroll
                for (int md = 0; md < MD; ++md) {
                    const u32x4 a = value(ss, md);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) x.o[nt][md] = E::mma32(a, pb[ss][nt], x.o[nt][md]);
                }
        };

        if (it.t0 < stop) {
            const GroupOffsets<D> off;
            const int last = stop - 1;
            loader.places.take(z, row_of(base));
            loader.places.ask(z, row_of(base + 64));
            auto fetch = [&](int t, Group<D>& raw) {
                if (t >= base + 64) {
                    base += 64;
                    loader.places.take(z, row_of(base));
                    loader.places.ask(z, row_of(base + 64));
                }
                if (once) loader.template load<true>(off, t - base, raw);
                else loader.template load<false>(off, t - base, raw);
            };
            // pieces of the work of turning a group into operands
            auto put_key = [&](char* tile, const Group<D>& raw, int kk) {
                *reinterpret_cast<u32x4*>(tile + (wave * KS + kk) * 1024) = key_values<D, F16>(raw, kk);
            };
            auto put_values = [&](char* tile, const Group<D>& raw, int pr) {
                u32x2 v[2];
                value_values<D, F16>(raw.v, raw.vs, pr, v);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    *reinterpret_cast<u32x2*>(tile + kApart + ((wave >> 1) * MD + 2 * pr + i) * 1024 + 8 * (wave & 1)) = v[i];
            };
            auto put = [&](int t, Group<D>& raw) {
                char* tile = lds + (t & 1) * kTile + 16 * lane;
#pragma unroll
                for (int kk = 0; kk < KS; ++kk) put_key(tile, raw, kk);
#pragma unroll
                for (int pr = 0; pr < D / 32; ++pr) put_values(tile, raw, pr);
            };
            auto drop_behind = [&](int t, Group<D>& raw) {
                const int left = it.n - (t * kKeys + 16 * wave);
                if (left < 16) drop_scales<D>(raw.vs, left);
            };
            // Tile t, and beside it the operands of tile t + 1 (behind the last tile: nobody reads them).  A matrix product
            // leaves half of its time to other instructions of its wave, and waves hardly share a SIMD's time otherwise
            // (32 products and 128 other instructions a wave, one after the other, two waves: 1002 clocks each; mixed
            // by fours: 837): so each step has two products, a read for a product to come and a piece of other work.
            auto tile_step = [&](int t, Group<D>& raw) {
                char* to = lds + ((t + 1) & 1) * kTile + 16 * lane;
                const char* tile = lds + (t & 1) * kTile + 16 * lane;
                constexpr int kAhead = 4;
                u32x4 a[kAhead];
                // the softmax of one workgroup's wave goes before the scores of the other's, which wait for LDS and the
                // matrix cores more (26 tokens 261 us without, 254 with; 63 tokens 254 / 238)
                __builtin_amdgcn_s_setprio(0);
                v4f s[NT][MT];
                auto key = [&](int i) {
                    return *reinterpret_cast<const u32x4*>(tile + ((kw * MT + i / KS) * KS + i % KS) * 1024);
                };
                auto value = [&](int i) {
                    return *reinterpret_cast<const u32x4*>(tile + kApart + ((kw * (MT / 2) + i / MD) * MD + i % MD) * 1024);
                };
                constexpr int kScores = MT * KS, kValues = MT / 2 * MD;
                drop_behind(t + 1, raw);
#pragma unroll
                for (int i = 0; i < kAhead; ++i) a[i] = key(i);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < kScores; ++i) {
                    const int mt = i / KS, kk = i % KS;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        s[nt][mt] = E::mma32(a[i % kAhead], qr[nt][kk], kk == 0 ? v4f{0.f, 0.f, 0.f, 0.f} : s[nt][mt]);
                    if (i + kAhead < kScores) a[i % kAhead] = key(i + kAhead);
                    constexpr int kEach = kScores / (D / 32);
                    if (i % kEach == 0) put_values(to, raw, i / kEach);
                    if (i % 2) __builtin_amdgcn_sched_barrier(0);
                }
                __builtin_amdgcn_s_setprio(3);
                const int left = it.n - t * kKeys - key0;
                if (left < 16 * MT) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) s[nt][mt][i] = 16 * mt + 4 * grp + i < left ? s[nt][mt][i] : kNegInf;
                }
#pragma unroll
                for (int i = 0; i < kAhead; ++i) a[i] = value(i);
                x.move(s, scale_log2);
                u32x4 pb[MT / 2][NT];
                float sum[NT];
                // the weights of two groups of 16 keys, 4 NT pairs of them
                auto weigh = [&](int ss, int piece) {
                    const int nt = piece % NT, j = piece / NT;
                    pb[ss][nt][j] = x.weigh(nt, s[nt][2 * ss + j / 2][2 * (j & 1)], s[nt][2 * ss + j / 2][2 * (j & 1) + 1], sum[nt]);
                };
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) sum[nt] = 0.f;
#pragma unroll
                for (int piece = 0; piece < 4 * NT; ++piece) weigh(0, piece);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < kValues; ++i) {
                    const int ss = i / MD, md = i % MD;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) x.o[nt][md] = E::mma32(a[i % kAhead], pb[ss][nt], x.o[nt][md]);
                    if (i + kAhead < kValues) a[i % kAhead] = value(i + kAhead);
                    // the weights of the next groups beside the values of these, K's operands beside the last
                    if (ss + 1 < MT / 2) {
                        constexpr int kEach = 4 * NT / MD;
#pragma unroll
                        for (int e = 0; e < kEach; ++e) weigh(ss + 1, kEach * md + e);
                    } else if (md % 2 == 0 && md / 2 < KS) {
                        put_key(to, raw, md / 2);
                    }
                    if (i % 2) __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) x.l[nt] += sum[nt];
            };
            // a tile's codes are asked for three tiles before they are worked on and become operands one before
            Group<D> raw[2];
            fetch(it.t0, raw[0]);
            fetch(min(it.t0 + 1, last), raw[1]);
            drop_behind(it.t0, raw[0]);
            put(it.t0, raw[0]);
            fetch(min(it.t0 + 2, last), raw[0]);
            __syncthreads();
            if (idle) {
                for (int t = it.t0;;) {
                    drop_behind(t + 1, raw[1]);
                    put(t + 1, raw[1]);
                    fetch(min(t + 3, last), raw[1]);
                    __syncthreads();
                    if (++t >= stop) break;
                    drop_behind(t + 1, raw[0]);
                    put(t + 1, raw[0]);
                    fetch(min(t + 3, last), raw[0]);
                    __syncthreads();
                    if (++t >= stop) break;
                }
            } else {
                for (int t = it.t0;;) {
                    tile_step(t, raw[1]);
                    fetch(min(t + 3, last), raw[1]);
                    __syncthreads();
                    if (++t >= stop) break;
                    tile_step(t, raw[0]);
                    fetch(min(t + 3, last), raw[0]);
                    __syncthreads();
                    if (++t >= stop) break;
                }
            }
        }
        // the drafted tokens
        const TreeParams& p = parameters().t;
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
            if (!idle)
                attend([&](int mt, int kk) { return key_operand<D, true>(ks + mt * R::kBytes, kk); },
                       [&](int ss, int md) {
                           const u32x2 lo = value_operand<D>(ks + kApart + 2 * ss * R::kBytes, md);
                           const u32x2 hi = value_operand<D>(ks + kApart + (2 * ss + 1) * R::kBytes, md);
                           return u32x4{lo.x, lo.y, hi.x, hi.y};
                       },
                       [&](v4f(&s)[NT][MT]) {
                           const int from = min(row0, p.M - 1) / p.G;
#pragma unroll
                           for (int nt = 0; nt < NT; ++nt) {
                               const uint64_t word =
                                   sh.seen[wave][min(row0 + 16 * nt + col, p.M - 1) / p.G - from] >> (key0 + 4 * grp);
#pragma unroll
                               for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                                   for (int i = 0; i < 4; ++i) s[nt][mt][i] = word >> (16 * mt + i) & 1 ? s[nt][mt][i] : kNegInf;
                           }
                       });
        }
        __syncthreads();

        join_keys<MD, NT, KW>(reinterpret_cast<float*>(lds), kRows, rw * 16 * NT, kw, x.m, x.l, x.o);
        if (kw == 0) {
            float* part = p.part + (2 * (int64_t)slot + (it.t0 == 0)) * kPart;
            const int j0 = max(0, it.t0 - cached) * kKeys, j1 = min(p.T, max(0, it.t1 - cached) * kKeys);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int in = rw * 16 * NT + 16 * nt + col, row = row0 + 16 * nt + col;
                if (sh.wild) add_unbounded<MD, F16>(p, b, it.h, j0, j1, row, x.o[nt]);
                finish_rows<MD, F16>(p, b, it.h, row, in, kRows, it.t0 == 0 && it.t1 == it.tiles, part, x.m[nt], x.l[nt], x.o[nt]);
            }
        }
        share.done(it);
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

// How the tiles come to the workgroups.  Dealt over all items, every workgroup has the same number of them however
// ragged the batch is, but most work on two items, each with its own start and end.  Where an item's tiles are few
// it is cut into splits of its own instead: so many that two workgroups a CU have work, of at least two tiles, and
// where no split has more than 16; up to five tiles stay whole and need no merge.  Dealt / split, in a graph: one
// token of 16 sequences of 1024 rows 20.1 / 14.2 us (whole 12.4), 4096 28.8 / 22.4, 8192 38.9 / 32.3, of a quarter to
// all of 8192 30.7 / 28.9; of one sequence of 4096 13.6 / 11.2; 26 tokens of 4 sequences of 2048 37.5 / 31.2, 8192 50.1
// / 41.0; longer ones are equal.  Splits of one tile and of four: one sequence of 4096 9.9 and 13.2, 26 tokens over
// 512 rows of 4 sequences 25.4 and 19.0 against 17.7.
constexpr int kLeastTiles = 2, kMostTiles = 16, kWholeTiles = 5;

struct QuantPlan : TreePlan {
    int tile;                                      // cache rows of a tile
    int splits;                                    // of every item; 0: dealt
    bool merges() const { return splits ? splits > 1 : !whole(); }
    size_t bytes(int64_t D) const { return merges() ? (size_t)slots * 2 * rows() * (D + 2) * sizeof(float) : 0; }
};

QuantPlan plan_attention(const slimkv_quantized_attention_args* a) {
    QuantPlan t{};
    static_cast<TreePlan&>(t) = plan_tree(a->tokens * (a->heads / a->kv_heads));
    t.tile = t.rw == 1 ? 64 * few_groups(t.nt) : kKeys;
    const int64_t workgroups = a->batch * a->kv_heads * t.row_blocks, resident = 2 * device_cu_count();
    const int64_t tiles = (a->keys + t.tile - 1) / t.tile + (a->tokens + kKeys - 1) / kKeys;
    if (workgroups == 0 || workgroups > 65536) return t;
    const int64_t splits = tiles <= kWholeTiles ? 1 : std::max<int64_t>(1, std::min((tiles + kLeastTiles - 1) / kLeastTiles, resident / workgroups));
    if ((tiles + splits - 1) / splits > kMostTiles) return t;
    t.splits = (int)splits;
    t.runs = (int)(a->batch * a->kv_heads * splits);
    t.slots = workgroups * splits;
    return t;
}

template <int D, bool F16>
void launch_attention(const QuantParams& p, const QuantPlan& plan, hipStream_t st) {
    const dim3 grid((unsigned)((plan.slots + kXcdCount - 1) / kXcdCount * kXcdCount));
    void (*kernel)(QuantParams) = plan.rw == 4   ? quant_many_kernel<D, F16, 4>
                                  : plan.rw == 2 ? quant_many_kernel<D, F16, 2>
                                  : plan.nt == 2 ? quant_few_kernel<D, F16, 2>
                                                 : quant_few_kernel<D, F16, 1>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p);
    if (plan.merges()) launch_merge<D, F16>(p.t, plan, st);
}

}  // namespace

}  // namespace slimkv

using namespace slimkv;

extern "C" size_t slimkv_quantized_attention_workspace(const slimkv_quantized_attention_args* a) {
    if (check_attention(a) != SLIMKV_OK) return 0;
    return std::max<size_t>(plan_attention(a).bytes(a->head_dim), 16);
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
    const QuantPlan plan = plan_attention(a);
    if (plan.merges() &&
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
    // without drafted tokens a tile without work, so that a sequence without rows has a run that writes its output
    p.deal = Dealing{p.B, p.Hk, plan.tile, draft ? (p.T + kKeys - 1) / kKeys : 1, plan.runs, plan.splits};
    p.scale_log2 = (float)(a->scale * 1.4426950408889634);
    p.part = static_cast<float*>(workspace);
    if (B * Hk * p.M > 0x7fffffff || (plan.merges() && !launchable(B * Hk * plan_merge(plan, B * Hk, p.M, D).chunks, 256)) ||
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
