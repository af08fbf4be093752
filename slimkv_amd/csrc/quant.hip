// Rows of a cache held in 4 bits, written and read back
// (include/slimkv/quant_cache.h has the format).
//
// Both are moves, bound by HBM: 4 D bytes of a row's K and V against D + D / 16 of
// its codes and scales, and a few instructions an element (32749 rows of 8 heads of
// 128 written in 33 us, 5.2 TB/s, and read back in 27, the codes still in the last
// cache; 4 histories of 4-16K rows read in 58 us, 5.4 TB/s; a copy moves 5.2).  The
// rows are stored a half or a quarter of a cache line an instruction, which the L2
// joins: non-temporal stores, which it does not join, took 86 us for the histories
// instead of 65 (calls), non-temporal loads 81 for writing and reading instead of 72.

#include "quant.hpp"

namespace slimkv {

namespace {

struct RowsParams {
    PoolView c;
    char* k; int64_t k_sb, k_sn, k_sh;        // strides in bytes
    char* v; int64_t v_sb, v_sn, v_sh;
    const int32_t* starts;
    const int32_t* counts;
    int B, H, rows;
    FastDiv by_rows, by_heads;
};

__device__ __forceinline__ int count_of(const RowsParams& p, int b) {
    return p.counts ? max(0, min(p.counts[b], p.rows)) : p.rows;
}

__device__ __forceinline__ void report_bad_slot(int32_t* status) {
    if (status) *status = SLIMKV_STATUS_BAD_SLOT;
}

// Page of row `row` (inside the capacity) of sequence b, or -1 with a report.
__device__ __forceinline__ int64_t page_of(const PoolView& c, int b, int row) {
    if (!c.table) return b;
    const int64_t page = table_page(c.table[b * c.t_sb + quotient(row, c.block)], c.num_pages);
    if (page < 0) report_bad_page(c.status);
    return page;
}

template <int CTRL>
__device__ __forceinline__ uint32_t from_lane(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, true);
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e;      // quad_perm 1 0 3 2 and 2 3 0 1

// The bytes of lo and hi, chosen by the selector (0 .. 3 of lo, 4 .. 7 of hi).
__device__ __forceinline__ uint32_t bytes_of(uint32_t lo, uint32_t hi, uint32_t selector) {
    return __builtin_amdgcn_perm(hi, lo, selector);
}

// The scale byte of a block of 32 elements (16 dwords), its factor's bits for the
// conversion in *factor, and whether it holds an infinity or NaN.
template <bool F16>
__device__ __forceinline__ int block_scale(const u32x4 (&x)[4], bool* wild) {
    using C = Codes<F16>;
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 top = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, x[i][e] & 0x7fff7fffu));
    const uint32_t most = max((uint32_t)top.x, (uint32_t)top.y);
    *wild = most >= C::kInfinite;
    // a mantissa from 1.75 on carries into the exponent
    const int e = (int)((__float_as_uint(C::value(most)) + 0x200000u) >> 23) - 2;
    return *wild ? 255 : max(0, min(e, C::kTopScale));
}

// A thread holds one block of 32 elements of a row, D / 32 threads the row, and
// consecutive rows of one sequence and head lie in consecutive threads: codes and
// scales leave as whole pieces.  V's bytes hold elements 16 apart of one block,
// which the thread has; the row's threads then exchange dwords so that each holds
// whole units of D / 32 bytes.
template <int D, bool F16>
__global__ void __launch_bounds__(256) quantize_rows_kernel(RowsParams p) {
    using C = Codes<F16>;
    constexpr int kLanes = D / 32;
    const uint32_t at = blockIdx.x * 256u + threadIdx.x;
    const int unit = at / kLanes, part = threadIdx.x % kLanes;
    const int bh = quotient(unit, p.by_rows), i = unit - bh * p.rows;
    const int b = quotient(bh, p.by_heads), h = bh - b * p.H;
    if (b >= p.B || i >= count_of(p, b)) return;
    const int64_t to = (p.starts ? (int64_t)p.starts[b] : 0) + i;
    if (to < 0 || to >= p.c.capacity) return report_bad_slot(p.c.status);
    const int row = (int)to;
    const u32x4* ks = reinterpret_cast<const u32x4*>(p.k + b * p.k_sb + i * p.k_sn + h * p.k_sh) + 4 * part;
    const u32x4* vs = reinterpret_cast<const u32x4*>(p.v + b * p.v_sb + i * p.v_sn + h * p.v_sh) + 4 * part;
    u32x4 k[4], v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) k[e] = ks[e];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = vs[e];
    const int64_t page = page_of(p.c, b, row);
    if (page < 0) return;
    uint8_t* base = p.c.pages + page * p.c.p_sb + h * p.c.p_sh;
    const int64_t slot = p.c.table ? row - quotient(row, p.c.block) * (int)p.c.block.d : row;

    bool wild;
    const int k_scale = block_scale<F16>(k, &wild);
    uint32_t f = (uint32_t)k_scale << 23;
    u32x4 out;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint32_t w = C::template codes<0>(0u, k[c].x, f);
        w = C::template codes<1>(w, k[c].y, f);
        w = C::template codes<2>(w, k[c].z, f);
        w = C::template codes<3>(w, k[c].w, f);
        out[c] = wild ? 0u : w;
    }
    *reinterpret_cast<u32x4*>(base + slot * (D / 2) + 16 * part) = out;
    base[p.c.ks_at + slot * kLanes + part] = (uint8_t)k_scale;

    const int v_scale = block_scale<F16>(v, &wild);
    f = (uint32_t)v_scale << 23;
    uint32_t a[4];                                 // byte m of 16: elements m and 16 + m of the block
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint32_t x0 = v[c >> 1][2 * (c & 1)], x1 = v[c >> 1][2 * (c & 1) + 1];
        const uint32_t y0 = v[2 + (c >> 1)][2 * (c & 1)], y1 = v[2 + (c >> 1)][2 * (c & 1) + 1];
        uint32_t w = C::template codes<0>(0u, bytes_of(x0, y0, 0x05040100u), f);
        w = C::template codes<1>(w, bytes_of(x0, y0, 0x07060302u), f);
        w = C::template codes<2>(w, bytes_of(x1, y1, 0x05040100u), f);
        w = C::template codes<3>(w, bytes_of(x1, y1, 0x07060302u), f);
        a[c] = wild ? 0u : w;
    }
    base[p.c.vs_at + slot * kLanes + part] = (uint8_t)v_scale;
    const int r = (int)(slot & 15), g = r >> 2, j = r & 3;
    uint8_t* group = base + p.c.v_at + (slot & ~(int64_t)15) * (D / 2);
    if constexpr (D == 128) {
        // lane `part` of four gets dword `part` of each
        const bool odd = part & 1, high = part & 2;
#pragma unroll
        for (int x = 0; x < 4; x += 2) {
            const uint32_t got = from_lane<kXor1>(odd ? a[x] : a[x + 1]);
            if (odd) a[x] = got;
            else a[x + 1] = got;
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint32_t got = from_lane<kXor2>(high ? a[x] : a[x + 2]);
            if (high) a[x] = got;
            else a[x + 2] = got;
        }
        const uint32_t lo01 = bytes_of(a[0], a[1], 0x05010400u), hi01 = bytes_of(a[0], a[1], 0x07030602u);
        const uint32_t lo23 = bytes_of(a[2], a[3], 0x05010400u), hi23 = bytes_of(a[2], a[3], 0x07030602u);
        const uint32_t w[4] = {bytes_of(lo01, lo23, 0x05040100u), bytes_of(lo01, lo23, 0x07060302u),
                               bytes_of(hi01, hi23, 0x05040100u), bytes_of(hi01, hi23, 0x07060302u)};
#pragma unroll
        for (int m = 0; m < 4; ++m)
            *reinterpret_cast<uint32_t*>(group + ((16 * g + 4 * part + m) * 4 + j) * 4) = w[m];
    } else {
        const bool odd = part & 1;
        uint32_t w[4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint32_t got = from_lane<kXor1>(odd ? a[x] : a[2 + x]), own = odd ? a[2 + x] : a[x];
            const uint32_t first = odd ? got : own, second = odd ? own : got;
            w[2 * x] = bytes_of(first, second, 0x05010400u);
            w[2 * x + 1] = bytes_of(first, second, 0x07030602u);
        }
#pragma unroll
        for (int m = 0; m < 8; ++m)
            *reinterpret_cast<uint16_t*>(group + ((16 * g + 8 * part + m) * 4 + j) * 2) =
                (uint16_t)(w[m / 2] >> (16 * (m & 1)));
    }
}

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

// A wave holds 16 rows of one sequence and head that lie side by side in the
// cache.  K's codes are in the order of the elements; V's pass through LDS, whose
// transposing read gives a lane 16 consecutive elements of one row.
template <int D, bool F16>
__global__ void __launch_bounds__(256) dequantize_rows_kernel(RowsParams p, int groups, FastDiv by_groups) {
    constexpr int kLanes = D / 32, kBytes = 8 * D;             // bytes of 16 rows' codes
    __shared__ alignas(16) char lds[4][kBytes];
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    const int at = blockIdx.x * 4 + wave;
    const int bh = quotient(at, by_groups), b = quotient(bh, p.by_heads), h = bh - b * p.H;
    if (b >= p.B) return;
    const int64_t start = p.starts ? p.starts[b] : 0;
    const int64_t row0 = ((start >> 4) + (at - bh * groups)) << 4;
    const int64_t first = row0 - start;                        // output row of the group's first
    if (first >= p.rows) return;
    const int count = count_of(p, b);
    bool ok = max(first, (int64_t)0) < min(first + 16, (int64_t)count);        // any row to read
    if (ok && (row0 < 0 || row0 >= p.c.capacity)) {           // a group lies inside the capacity or outside
        report_bad_slot(p.c.status);
        ok = false;
    }
    const uint8_t* base = nullptr;
    int64_t slot = 0;
    if (ok) {
        const int64_t page = page_of(p.c, b, (int)row0);
        ok = page >= 0;
        slot = p.c.table ? (int)row0 - quotient((int)row0, p.c.block) * (int)p.c.block.d : (int)row0;
        base = p.c.pages + (ok ? page : 0) * p.c.p_sb + h * p.c.p_sh;
    }
    char* ko = p.k + b * p.k_sb + h * p.k_sh;
    char* vo = p.v + b * p.v_sb + h * p.v_sh;

    constexpr int kPieces = D / 8, kPass = 64 / kPieces;       // 8 elements a lane, rows a pass
    uint32_t codes[16 / kPass], scales[16 / kPass];
#pragma unroll
    for (int c = 0; c < 16 / kPass; ++c) {
        const int r = kPass * c + lane / kPieces, piece = lane % kPieces;
        codes[c] = scales[c] = 0;
        if (ok) {
            codes[c] = *reinterpret_cast<const uint32_t*>(base + (slot + r) * (D / 2) + 4 * piece);
            scales[c] = base[p.c.ks_at + (slot + r) * kLanes + piece / 4];
        }
    }
    typedef uint32_t vec __attribute__((ext_vector_type(D / 32)));
    vec vw = {};
    if (ok) vw = *reinterpret_cast<const vec*>(base + p.c.v_at + slot * (D / 2) + sizeof(vec) * lane);
    constexpr int kReads = D / 64;                             // transposing reads of 64 bits a lane
    const int g = lane >> 4, c16 = lane & 15, t = c16 % (D / 16);
    uint32_t v_scale[kReads];
#pragma unroll
    for (int x = 0; x < kReads; ++x) {
        const int r = 4 * g + (4 / kReads) * x + c16 / (D / 16);
        v_scale[x] = ok ? base[p.c.vs_at + (slot + r) * kLanes + t / 2] : 0;
    }
#pragma unroll
    for (int c = 0; c < 16 / kPass; ++c) {
        const int r = kPass * c + lane / kPieces, piece = lane % kPieces;
        const int64_t i = first + r;
        if (i < 0 || i >= p.rows) continue;
        const bool live = i < count;
        *reinterpret_cast<u32x4*>(ko + i * p.k_sn + 16 * piece) =
            eight_values<F16>(live ? codes[c] : 0u, live ? scales[c] << 23 : 0u);
    }
    *reinterpret_cast<vec*>(lds[wave] + sizeof(vec) * lane) = vw;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int x = 0; x < kReads; ++x) {
        const auto w = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
            (lds_i32x2*)(lds[wave] + sizeof(vec) * (lane & ~15) + sizeof(vec) * c16 + 8 * x));
        const int r = 4 * g + (4 / kReads) * x + c16 / (D / 16);
        const int64_t i = first + r;
        if (i < 0 || i >= p.rows) continue;
        const bool live = i < count;
        u32x4* to = reinterpret_cast<u32x4*>(vo + i * p.v_sn + 32 * t);
        const uint32_t f = live ? v_scale[x] << 23 : 0u;
        to[0] = eight_values<F16>(live ? (uint32_t)w[0] : 0u, f);
        to[1] = eight_values<F16>(live ? (uint32_t)w[1] : 0u, f);
    }
}

template <class A>
int check_rows(const A* a, const char* what, RowsParams* p) {
    const std::string w(what);
    if (!a) return fail(SLIMKV_EINVAL, w + ": null pointer");
    if (a->head_dim != 64 && a->head_dim != 128) return fail(SLIMKV_EUNSUP, w + ": head_dim must be 64 or 128");
    if (a->dtype != SLIMKV_DTYPE_BF16 && a->dtype != SLIMKV_DTYPE_F16)
        return fail(SLIMKV_EUNSUP, w + ": element type must be bf16 or fp16");
    if (a->batch < 0 || a->batch > 65535 || a->rows < 0 || a->rows > ((int64_t)1 << 30) || a->kv_heads <= 0 ||
        a->kv_heads > 4096)
        return fail(SLIMKV_EINVAL, w + ": invalid sizes");
    if (a->batch == 0 || a->rows == 0) return SLIMKV_OK;
    if (!a->k || !a->v) return fail(SLIMKV_EINVAL, w + ": null pointer");
    if (!rows_aligned(a->k, {{a->batch, a->k_sb}, {a->rows, a->k_sn}, {a->kv_heads, a->k_sh}}) ||
        !rows_aligned(a->v, {{a->batch, a->v_sb}, {a->rows, a->v_sn}, {a->kv_heads, a->v_sh}}))
        return fail(SLIMKV_EINVAL, w + ": rows must start on 16-byte boundaries (strides multiples of 8)");
    const int code = pool_view(a->cache, a->batch, a->kv_heads, a->head_dim, what, &p->c);
    if (code != SLIMKV_OK) return code;
    // threads, and the row numbers that they are divided by, in 31 bits
    if (a->batch * a->kv_heads * ((a->rows + 30) / 16 * 16) > 0x7fffffff / 4)
        return fail(SLIMKV_EINVAL, w + ": too many rows for one call");
    p->k = (char*)a->k; p->k_sb = 2 * a->k_sb; p->k_sn = 2 * a->k_sn; p->k_sh = 2 * a->k_sh;
    p->v = (char*)a->v; p->v_sb = 2 * a->v_sb; p->v_sn = 2 * a->v_sn; p->v_sh = 2 * a->v_sh;
    p->starts = a->starts; p->counts = a->counts;
    p->B = (int)a->batch; p->H = (int)a->kv_heads; p->rows = (int)a->rows;
    p->by_rows = fast_div(a->rows); p->by_heads = fast_div(a->kv_heads);
    return SLIMKV_OK;
}

}  // namespace

int pool_view(const slimkv_quant_pages& q, int64_t batch, int64_t kv_heads, int64_t head_dim, const char* what,
              PoolView* view) {
    const std::string w(what);
    if (!q.pages) return fail(SLIMKV_EINVAL, w + ": null page pool");
    if (q.block_size <= 0 || q.block_size % 16 || q.block_size > ((int64_t)1 << 30) || q.num_pages <= 0 ||
        q.num_pages > 0x7fffffff || (q.table ? q.t_cols <= 0 || q.t_cols > ((int64_t)1 << 30) : q.num_pages < batch) ||
        (q.table && batch > 1 && q.t_sb < q.t_cols && q.t_sb != 0))
        return fail(SLIMKV_EINVAL, w + ": invalid page layout (blocks are multiples of 16 rows; without a table a page "
                                       "a sequence)");
    const int64_t bytes = q.block_size * (head_dim + head_dim / 16);
    if ((reinterpret_cast<uintptr_t>(q.pages) & 15) || (q.num_pages > 1 && (q.p_sb % 16 || q.p_sb < 0)) ||
        (kv_heads > 1 && (q.p_sh % 16 || q.p_sh < bytes)))
        return fail(SLIMKV_EINVAL, w + ": pages must start on 16-byte boundaries and a page's heads lie apart");
    view->pages = q.pages; view->p_sb = q.p_sb; view->p_sh = q.p_sh;
    view->table = q.table; view->t_sb = q.t_sb; view->num_pages = q.num_pages;
    view->block = fast_div(q.block_size);
    view->capacity = (int)std::min<int64_t>((q.table ? q.t_cols : 1) * q.block_size, (int64_t)1 << 30);
    view->status = q.status;
    view->v_at = q.block_size * (head_dim / 2);
    view->ks_at = q.block_size * head_dim;
    view->vs_at = view->ks_at + q.block_size * (head_dim / 32);
    return SLIMKV_OK;
}

}  // namespace slimkv

using namespace slimkv;

extern "C" int slimkv_quant_abi_version(void) { return 1; }

extern "C" int slimkv_quantize_rows(const slimkv_quantize_rows_args* a, void* stream) {
    RowsParams p{};
    const int code = check_rows(a, "quantize rows", &p);
    if (code != SLIMKV_OK || p.B == 0) return code;
    const int64_t threads = a->batch * a->kv_heads * a->rows * (a->head_dim / 32);
    const dim3 grid((unsigned)((threads + 255) / 256));
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool f16 = a->dtype == SLIMKV_DTYPE_F16;
    auto kernel = a->head_dim == 128 ? (f16 ? quantize_rows_kernel<128, true> : quantize_rows_kernel<128, false>)
                                     : (f16 ? quantize_rows_kernel<64, true> : quantize_rows_kernel<64, false>);
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p);
    return check_hip(hipGetLastError(), "quantize rows launch");
}

extern "C" int slimkv_dequantize_rows(const slimkv_dequantize_rows_args* a, void* stream) {
    RowsParams p{};
    const int code = check_rows(a, "dequantize rows", &p);
    if (code != SLIMKV_OK || p.B == 0) return code;
    // groups of 16 cache rows that `rows` of them can touch
    const int64_t groups = (a->rows + 30) / 16;
    const dim3 grid((unsigned)((a->batch * a->kv_heads * groups + 3) / 4));
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool f16 = a->dtype == SLIMKV_DTYPE_F16;
    auto kernel = a->head_dim == 128 ? (f16 ? dequantize_rows_kernel<128, true> : dequantize_rows_kernel<128, false>)
                                     : (f16 ? dequantize_rows_kernel<64, true> : dequantize_rows_kernel<64, false>);
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p, (int)groups, fast_div(groups));
    return check_hip(hipGetLastError(), "dequantize rows launch");
}
