// Eviction from a cache: the rows to keep by weight, and their move.
//
// select: a radix selection over 11, 11 and 10 bits.  fp32 weights map to
// unsigned integers in their order (NaN to 0), the rows between the first
// `sink` and the last `recent` are ranked by them, and three histograms find
// the weight of the last row kept and how many rows of exactly that weight fit;
// a last pass counts and writes the kept rows in ascending order.  All counts
// are integers, so the result does not depend on the order of the LDS atomics.
// Up to 32768 rows one workgroup holds in registers.  More are cut into chunks: a
// launch makes each chunk's histogram, and every workgroup of the next one adds
// them up for itself, so no launch waits for another workgroup.
//
// compact: bytes moved.  Out of place a lane moves 16 bytes of K and V of one
// row; in place a workgroup takes some columns of one head's K or V and
// walks the kept rows in order.

#include "cache.hpp"

namespace slimkv {

namespace {

constexpr int kSelectThreads = 512, kSelectWaves = kSelectThreads / 64;
constexpr int kHeldThreads = 1024, kHeldWaves = kHeldThreads / 64, kMostHeld = 32;   // values a thread keeps
constexpr int kCopies = 4;        // of the first histogram, for lanes that meet in a bin
constexpr int kBins = 2048, kLastBins = 1024;
constexpr int kBatch = 8;         // loads a thread has open at once

struct SelectParams {
    const float* weights; int64_t w_sb, w_sh;
    const int32_t* lengths;
    int32_t* rows;
    int32_t* counts;
    int H, keys, keep, sink, recent;
    int chunks;
    uint32_t* ws;                 // a row's part: see SelectRow
};

// Order-preserving image of a weight: -0 as +0, NaN below everything.
__device__ __forceinline__ uint32_t rank_of(float w) {
    const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
    return w != w ? 0u : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

// Set bits of a wave's mask below this lane's.
__device__ __forceinline__ int lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// One (sequence, head): the ranked rows [first, last), of which `need` are
// taken, and this workgroup's chunk [from, to) of them.  Workspace of a row:
// histograms [chunks][2048], [chunks][2048], [chunks][1024], a count a chunk of
// the rows above the first and above the second prefix, and the state (prefix,
// rows left) after the first and the second level.
struct SelectRow {
    const float* w;
    int32_t* rows;
    uint32_t *h1, *h2, *h3, *above1, *above2;
    int n, first, last, need, chunk, from, to;
    bool trivial;                 // every row is kept, or none of the ranked ones

    __device__ __forceinline__ SelectRow(const SelectParams& p, int item, int chunk_) {
        const int64_t b = item / p.H, h = item % p.H;
        n = p.lengths ? max(0, min(p.lengths[b], p.keys)) : p.keys;
        w = p.weights + b * p.w_sb + h * p.w_sh;
        rows = p.rows + (int64_t)item * p.keep;
        need = p.keep - p.sink - p.recent;
        trivial = n <= p.keep || need == 0;
        first = p.sink;
        last = max(first, n - p.recent);
        chunk = chunk_;
        const int64_t span = last - first;
        from = first + (int)(span * chunk / p.chunks);
        to = first + (int)(span * (chunk + 1) / p.chunks);
        h1 = p.ws + (int64_t)item * (p.chunks * (2 * kBins + kLastBins + 2) + 4);
        h2 = h1 + p.chunks * kBins;
        h3 = h2 + p.chunks * kBins;
        above1 = h3 + p.chunks * kLastBins;
        above2 = above1 + p.chunks;
    }
    // What needs no ranking: the first and the recent rows, the padding, the count.
    __device__ __forceinline__ void write_given(const SelectParams& p, int item) const {
        const int count = min(n, p.keep), tid = threadIdx.x;
        if (item % p.H == 0 && tid == 0) p.counts[item / p.H] = count;
        const int threads = blockDim.x;
        for (int i = count + tid; i < p.keep; i += threads) rows[i] = -1;
        if (n <= p.keep) {
            for (int i = tid; i < n; i += threads) rows[i] = i;
            return;
        }
        for (int i = tid; i < p.sink; i += threads) rows[i] = i;
        for (int i = tid; i < p.recent; i += threads) rows[p.keep - p.recent + i] = n - p.recent + i;
    }
};

// What a workgroup shares: a histogram, the bin found, sums over its waves.
struct SelectLds {
    uint32_t hist[kBins];
    uint32_t bin, above;
    uint32_t wave[2][kHeldWaves];
};

// No row counted yet, once all threads are past what they read of s.
__device__ __forceinline__ void clear_bins(SelectLds& s) {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += blockDim.x) s.hist[i] = 0;
    __syncthreads();
}

// Sum of x over the workgroup's threads below this one, and over all of them.
template <int THREADS = kSelectThreads>
__device__ __forceinline__ uint32_t block_before(uint32_t x, SelectLds& s, uint32_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t upto = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(upto, d, 64);
        if (lane >= d) upto += y;
    }
    __syncthreads();
    if (lane == 63) s.wave[0][wave] = upto;
    __syncthreads();
    uint32_t below = 0, all = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) {
        below += i < wave ? s.wave[0][i] : 0u;
        all += s.wave[0][i];
    }
    *total = all;
    return below + upto - x;
}

// The bin, from the highest down, that holds row `left` (counted from 1):
// s.bin, and s.above rows in the bins above it.
template <int NB, int THREADS = kSelectThreads>
__device__ __forceinline__ void find_bin(SelectLds& s, uint32_t left) {
    constexpr int K = NB / THREADS;
    uint32_t c[K], sum = 0, all;
#pragma unroll
    for (int x = 0; x < K; ++x) sum += c[x] = s.hist[NB - 1 - (K * (int)threadIdx.x + x)];
    uint32_t before = block_before<THREADS>(sum, s, &all);
#pragma unroll
    for (int x = 0; x < K; ++x) {
        if (before < left && before + c[x] >= left) {
            s.bin = NB - 1 - (K * threadIdx.x + x);
            s.above = before;
        }
        before += c[x];
    }
    __syncthreads();
}

// The three levels of the ranking: bins of 11, 11 and 10 bits from the top.
template <int LEVEL>
struct Level {
    static constexpr int kN = LEVEL == 3 ? kLastBins : kBins;
    static constexpr int kShift = LEVEL == 1 ? 21 : LEVEL == 2 ? 10 : 0;
    static __device__ __forceinline__ bool matches(uint32_t u, uint32_t prefix) {
        return LEVEL == 1 || u >> (LEVEL == 2 ? 21 : 10) == prefix;
    }
};

// s.hist: the ranks in [from, to) that match the prefix, by this level's bits.
template <int LEVEL>
__device__ __forceinline__ void histogram(SelectLds& s, const SelectRow& r, uint32_t prefix) {
    using V = Level<LEVEL>;
    __syncthreads();
    for (int i = threadIdx.x; i < V::kN; i += kSelectThreads) s.hist[i] = 0;
    __syncthreads();
    for (int i0 = r.from; i0 < r.to; i0 += kBatch * kSelectThreads) {
        float x[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) x[k] = r.w[min(i0 + k * kSelectThreads + (int)threadIdx.x, r.to - 1)];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const uint32_t u = rank_of(x[k]);
            if (i0 + k * kSelectThreads + (int)threadIdx.x < r.to && V::matches(u, prefix))
                atomicAdd(&s.hist[u >> V::kShift & (V::kN - 1)], 1u);
        }
    }
    __syncthreads();
}

// s.hist: the chunks' histograms added up.
template <int N>
__device__ __forceinline__ void add_chunks(SelectLds& s, const uint32_t* h, int chunks) {
    constexpr int K = N / kSelectThreads;
    uint32_t sum[K] = {};
    for (int c0 = 0; c0 < chunks; c0 += kBatch) {
        uint32_t v[kBatch][K];
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
            for (int x = 0; x < K; ++x)
                v[k][x] = h[(int64_t)min(c0 + k, chunks - 1) * N + x * kSelectThreads + threadIdx.x];
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
            for (int x = 0; x < K; ++x) sum[x] += c0 + k < chunks ? v[k][x] : 0u;
    }
#pragma unroll
    for (int x = 0; x < K; ++x) s.hist[x * kSelectThreads + threadIdx.x] = sum[x];
    __syncthreads();
}

// Rows of one chunk's histogram in the bins above `bin`, on every thread.
template <int N>
__device__ __forceinline__ uint32_t rows_above(SelectLds& s, const uint32_t* h, uint32_t bin) {
    uint32_t sum = 0, all;
#pragma unroll
    for (int x = 0; x < N / kSelectThreads; ++x) {
        const uint32_t i = x * kSelectThreads + threadIdx.x;
        sum += i > bin ? h[i] : 0u;
    }
    block_before(sum, s, &all);
    return all;
}

// The chunk's rows above `least` and the first `left` equal to it (of the whole
// row: `same` equal ones lie in the chunks before), in order, from the row's
// position `at` on.  A wave owns a contiguous part.
__device__ __forceinline__ void write_taken(const SelectRow& r, SelectLds& s, uint32_t least, int left, int at, int same) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int part = ((r.to - r.from + kSelectWaves - 1) / kSelectWaves + 63) / 64 * 64;
    const int from = min(r.to, r.from + wave * part), to = min(r.to, from + part);
    int above = 0, equal = 0;
    for (int i0 = from; i0 < to; i0 += 64 * kBatch) {
        float x[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) x[k] = r.w[min(i0 + 64 * k + lane, to - 1)];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const uint32_t u = rank_of(x[k]);
            above += __popcll(__ballot(i0 + 64 * k + lane < to && u > least));
            equal += __popcll(__ballot(i0 + 64 * k + lane < to && u == least));
        }
    }
    if (lane == 0) {
        s.wave[0][wave] = above;
        s.wave[1][wave] = equal;
    }
    __syncthreads();
    for (int x = 0; x < wave; ++x) {
        at += (int)s.wave[0][x] + min((int)s.wave[1][x], max(0, left - same));
        same += (int)s.wave[1][x];
    }
    int32_t* dst = r.rows + at;
    for (int i0 = from; i0 < to; i0 += 64 * kBatch) {
        float x[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) x[k] = r.w[min(i0 + 64 * k + lane, to - 1)];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int i = i0 + 64 * k + lane;
            const uint32_t u = rank_of(x[k]);
            const uint64_t eq = __ballot(i < to && u == least);
            const bool take = i < to && (u > least || (u == least && same + lanes_below(eq) < left));
            const uint64_t all = __ballot(take);
            if (take) dst[lanes_below(all)] = i;
            dst += __popcll(all);
            same += __popcll(eq);
        }
    }
}

// A row whose values one workgroup holds, VALUES a thread: read once, ranked and
// written from registers.  A wave owns a contiguous part.  What lies behind the
// ranked rows has rank 0, the lowest, and the highest places: it is never taken.
// Bound by its instructions, some 85 for 64 values, and the LDS atomics.  Against
// chunks over four launches: 8 rows of 32768 values 18 us (26), 128 rows of 16384
// 12.5 (27.6) and of 32768 18 (37), 512 of 32768 41 (80).  Weights lie in few bins
// of the first level, zeros in one: rows of which half are zero take 29 us with
// one copy of its histogram, 20 with four, eight or sixteen.
template <int VALUES>
__global__ void __launch_bounds__(kHeldThreads) select_held_kernel(SelectParams p) {
    __shared__ SelectLds s;
    __shared__ uint32_t copies[kBins * kCopies];
    const SelectRow r(p, blockIdx.x, 0);
    r.write_given(p, blockIdx.x);
    if (r.trivial) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int first = r.first + 64 * VALUES * wave + lane;
    uint32_t u[VALUES], left = r.need;
    {
        float x[VALUES];
#pragma unroll
        for (int k = 0; k < VALUES; ++k) x[k] = r.w[min(first + 64 * k, r.last - 1)];
        for (int i = tid; i < kBins * kCopies; i += kHeldThreads) copies[i] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < VALUES; ++k) u[k] = first + 64 * k < r.last ? rank_of(x[k]) : 0u;
    }
#pragma unroll
    for (int k = 0; k < VALUES; ++k) atomicAdd(&copies[(u[k] >> 21) * kCopies + lane % kCopies], 1u);
    __syncthreads();
    for (int i = tid; i < kBins; i += kHeldThreads) {
        uint32_t sum = 0;
#pragma unroll
        for (int c = 0; c < kCopies; ++c) sum += copies[i * kCopies + c];
        s.hist[i] = sum;
    }
    __syncthreads();
    find_bin<kBins, kHeldThreads>(s, left);
    uint32_t prefix = s.bin << 21;
    left -= s.above;
    clear_bins(s);
#pragma unroll
    for (int k = 0; k < VALUES; ++k)
        if (u[k] - prefix < 1u << 21) atomicAdd(&s.hist[(u[k] - prefix) >> 10], 1u);
    __syncthreads();
    find_bin<kBins, kHeldThreads>(s, left);
    prefix |= s.bin << 10;
    left -= s.above;
    clear_bins(s);
#pragma unroll
    for (int k = 0; k < VALUES; ++k)
        if (u[k] - prefix < 1u << 10) atomicAdd(&s.hist[u[k] - prefix], 1u);
    __syncthreads();
    find_bin<kLastBins, kHeldThreads>(s, left);
    const uint32_t least = prefix | s.bin;
    const int wanted = (int)(left - s.above);
    int above = 0, equal = 0;
#pragma unroll
    for (int k = 0; k < VALUES; ++k) {
        above += __popcll(__ballot(u[k] > least));
        equal += __popcll(__ballot(u[k] == least));
    }
    __syncthreads();
    if (lane == 0) {
        s.wave[0][wave] = above;
        s.wave[1][wave] = equal;
    }
    __syncthreads();
    int at = p.sink, same = 0;
    for (int x = 0; x < wave; ++x) {
        at += (int)s.wave[0][x] + min((int)s.wave[1][x], max(0, wanted - same));
        same += (int)s.wave[1][x];
    }
    int32_t* dst = r.rows + uniform(at);
    same = uniform(same);
#pragma unroll
    for (int k = 0; k < VALUES; ++k) {
        asm volatile("" : "+v"(u[k]));                     // compared anew: the masks of the counting are too many to keep
        const uint64_t eq = __ballot(u[k] == least);
        uint64_t all = __ballot(u[k] > least);
        if (eq && same < wanted) {
            all |= __ballot(u[k] == least && same + lanes_below(eq) < wanted);
            same += __popcll(eq);
        }
        if (__builtin_amdgcn_inverse_ballot_w64(all)) dst[lanes_below(all)] = first + 64 * k;
        dst += __popcll(all);
    }
}

// A longer row in one workgroup, where rows are many.
__global__ void __launch_bounds__(kSelectThreads) select_kernel(SelectParams p) {
    __shared__ SelectLds s;
    const SelectRow r(p, blockIdx.x, 0);
    r.write_given(p, blockIdx.x);
    if (r.trivial) return;
    uint32_t left = r.need, prefix;
    histogram<1>(s, r, 0);
    find_bin<kBins>(s, left);
    prefix = s.bin;
    left -= s.above;
    histogram<2>(s, r, prefix);
    find_bin<kBins>(s, left);
    prefix = prefix << 11 | s.bin;
    left -= s.above;
    histogram<3>(s, r, prefix);
    find_bin<kLastBins>(s, left);
    prefix = prefix << 10 | s.bin;
    left -= s.above;
    __syncthreads();
    write_taken(r, s, prefix, (int)left, p.sink, 0);
}

// A row in chunks, one launch a level and one to write (LEVEL 4).
template <int LEVEL>
__global__ void __launch_bounds__(kSelectThreads) select_chunk_kernel(SelectParams p) {
    __shared__ SelectLds s;
    const int item = blockIdx.y, chunk = blockIdx.x;
    const SelectRow r(p, item, chunk);
    if (LEVEL == 1 && chunk == 0) r.write_given(p, item);
    if (r.trivial) return;
    // prefix and rows left after the first and the second level
    uint32_t* state = r.above2 + p.chunks;
    uint32_t prefix = 0, left = r.need;
    if constexpr (LEVEL >= 3) {
        prefix = state[2 * (LEVEL - 3)];
        left = state[2 * (LEVEL - 3) + 1];
    }
    if constexpr (LEVEL >= 2) {
        constexpr int N = LEVEL == 4 ? kLastBins : kBins;
        const uint32_t* h = LEVEL == 2 ? r.h1 : LEVEL == 3 ? r.h2 : r.h3;
        add_chunks<N>(s, h, p.chunks);
        find_bin<N>(s, left);
        const uint32_t bin = s.bin;
        left -= s.above;
        prefix = LEVEL == 2 ? bin : prefix << (LEVEL == 3 ? 11 : 10) | bin;
        if constexpr (LEVEL < 4) {
            const uint32_t above = rows_above<N>(s, h + (int64_t)chunk * N, bin);
            if (threadIdx.x == 0) {
                (LEVEL == 2 ? r.above1 : r.above2)[chunk] = above;
                if (chunk == 0) {
                    state[2 * (LEVEL - 2)] = prefix;
                    state[2 * (LEVEL - 2) + 1] = left;
                }
            }
        } else {
            // rows taken and equal ones in the chunks before
            uint32_t taken = 0, same = 0, unused;
            for (int c = threadIdx.x; c < chunk; c += kSelectThreads) {
                taken += r.above1[c] + r.above2[c];
                same += h[(int64_t)c * N + bin];
            }
            for (int c0 = 0; c0 < chunk; c0 += kBatch) {
                uint32_t v[kBatch][N / kSelectThreads];
#pragma unroll
                for (int k = 0; k < kBatch; ++k)
#pragma unroll
                    for (int x = 0; x < N / kSelectThreads; ++x)
                        v[k][x] = h[(int64_t)min(c0 + k, chunk - 1) * N + x * kSelectThreads + threadIdx.x];
#pragma unroll
                for (int k = 0; k < kBatch; ++k)
#pragma unroll
                    for (int x = 0; x < N / kSelectThreads; ++x)
                        taken += c0 + k < chunk && x * kSelectThreads + threadIdx.x > bin ? v[k][x] : 0u;
            }
            block_before(taken, s, &unused);
            const int before = (int)unused;
            block_before(same, s, &unused);
            const int equal = (int)unused;
            __syncthreads();
            write_taken(r, s, prefix, (int)left, p.sink + before + min(equal, (int)left), equal);
            return;
        }
    }
    if constexpr (LEVEL < 4) {
        histogram<LEVEL>(s, r, prefix);
        uint32_t* out = LEVEL == 1 ? r.h1 : LEVEL == 2 ? r.h2 : r.h3;
        constexpr int N = Level<LEVEL>::kN;
        for (int i = threadIdx.x; i < N; i += kSelectThreads) out[(int64_t)chunk * N + i] = s.hist[i];
    }
}

// Chunks of a row that no workgroup holds: of 8192 values, at most 32, and no more
// than give four workgroups a CU over all rows.
int select_chunks(const slimkv_select_rows_args* a) {
    if (a->keys <= kMostHeld * kHeldThreads) return 1;
    const int64_t rows = std::max<int64_t>(1, a->batch * a->heads), most = 4 * device_cu_count() / rows;
    return (int)std::max<int64_t>(1, std::min<int64_t>({(a->keys + 8191) / 8192, 32, most}));
}

size_t select_bytes(const slimkv_select_rows_args* a) {
    const int chunks = select_chunks(a);
    if (chunks == 1) return 16;
    return (size_t)(a->batch * a->heads) * ((size_t)chunks * (2 * kBins + kLastBins + 2) + 4) * sizeof(uint32_t);
}

struct CompactParams {
    CacheView c;
    const int32_t* rows; int64_t r_sb, r_sh;
    const int32_t* counts;
    uint16_t* ok; int64_t ok_sb, ok_sn, ok_sh;
    uint16_t* ov; int64_t ov_sb, ov_sn, ov_sh;
    float* weights; int64_t w_sb, w_sh;
    float* ow; int64_t ow_sb, ow_sh;
    int Hw, wkeys, Hk, D, keep;
    int move_blocks;                              // workgroups a sequence that move K and V rows
    int lanes_log;                                // in place: log2 of the 16-byte lanes of a part
};

__device__ __forceinline__ int kept_count(const CompactParams& p, int64_t b) {
    return max(0, min(p.counts[b], p.keep));
}

__device__ __forceinline__ void report_bad_row(int32_t* status) {
    if (status) *status = SLIMKV_STATUS_BAD_SLOT;
}

// blockIdx.y is the sequence; the first move_blocks workgroups move K and V,
// D / 8 lanes a (row, head), the others the weights.  APART: each head has rows
// of its own.
template <bool PAGED, bool APART>
__global__ void __launch_bounds__(256) compact_kernel(CompactParams p) {
    const int64_t b = blockIdx.y;
    const int count = kept_count(p, b);
    if ((int)blockIdx.x >= p.move_blocks) {
        const int64_t at = (int64_t)(blockIdx.x - p.move_blocks) * 256 + threadIdx.x;
        if (at >= (int64_t)p.Hw * p.keep) return;
        const int h = (int)(at / p.keep), i = (int)(at % p.keep);
        float x = 0.f;
        if (i < count) {
            const int row = p.rows[b * p.r_sb + h * p.r_sh + i];
            if (row >= 0 && row < p.wkeys) x = p.weights[b * p.w_sb + h * p.w_sh + row];
            else report_bad_row(p.c.status);
        }
        p.ow[b * p.ow_sb + h * p.ow_sh + i] = x;
        return;
    }
    const int lanes = p.D / 8, d = 8 * (threadIdx.x % lanes);
    const int64_t item = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
    if (item >= (int64_t)p.keep * p.Hk) return;
    const int i = (int)(item / p.Hk), h = (int)(item % p.Hk);
    u32x4 k = {0u, 0u, 0u, 0u}, v = {0u, 0u, 0u, 0u};
    if (i < count) {
        const int row = p.rows[b * p.r_sb + h * p.r_sh + i];
        if (row < 0 || row >= p.c.keys) {
            report_bad_row(p.c.status);
        } else {
            bool good = true;
            if constexpr (PAGED) {
                good = table_page(p.c.table[b * p.c.t_sb + quotient(row, p.c.block)], p.c.num_blocks) >= 0;
                if (!good) report_bad_page(p.c.status);
            }
            if (good) {
                const RowAt at = cache_row<PAGED>(p.c, b, row);
                const auto* ks = reinterpret_cast<const u32x4*>(p.c.k + at.k + h * p.c.k_sh + d);
                const auto* vs = reinterpret_cast<const u32x4*>(p.c.v + at.v + h * p.c.v_sh + d);
                // heads with rows of their own, whose 256-byte pieces lie apart: non-temporal (16 x 8 heads, 4096
                // paged rows each, 107 us without, 91 with); one choice for all heads, whole rows: not (16001 rows
                // 21.5 / 23.9 us)
                if constexpr (APART) {
                    k = __builtin_nontemporal_load(ks);
                    v = __builtin_nontemporal_load(vs);
                } else {
                    k = *ks;
                    v = *vs;
                }
            }
        }
    }
    *reinterpret_cast<u32x4*>(p.ok + b * p.ok_sb + i * p.ok_sn + h * p.ok_sh + d) = k;
    *reinterpret_cast<u32x4*>(p.ov + b * p.ov_sb + i * p.ov_sn + h * p.ov_sh + d) = v;
}

// In place: blockIdx = ((sequence, KV head), K or V, part of the columns), then the
// weights' workgroups.  A step reads the rows of kMoves places a thread, waits for
// all of them, and writes.  Row i comes from a row not below i and the choice
// ascends, so what a step reads lies past all that the steps before have written,
// and one barrier a step (reads done, then writes) is enough.  Bound by the chain
// of a step's dependent loads (row, block, data) where workgroups are few and by
// HBM where they are many.  A part is 64 columns, whole lines, if that gives every
// CU a workgroup, else 32: 16 sequences of 8 heads, 4096 rows kept of 32768, 136 us
// against 178; one sequence, 34 us against 23.  Parts of 16: 294 and 25.  Steps of
// 512 threads: 144 and 28.
constexpr int kMoveThreads = 1024, kMoves = 8;

// Whether place i of a choice may take row `row`, `prior` being the row before.
__device__ __forceinline__ bool may_move(int row, int prior, int i, int keys) {
    return row > prior && row >= i && row < keys;
}

// Every load above has reached its register, on all waves of the workgroup.
__device__ __forceinline__ void reads_done() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

template <bool PAGED>
__global__ void __launch_bounds__(kMoveThreads) compact_in_place_kernel(CompactParams p) {
    const int cols = p.D >> (p.lanes_log + 3), per_head = 2 * cols, tid = threadIdx.x;
    const int64_t b = blockIdx.y;
    const int count = kept_count(p, b);
    if ((int)blockIdx.x >= p.move_blocks) {
        const int h = (int)blockIdx.x - p.move_blocks;
        float* w = p.weights + b * p.w_sb + h * p.w_sh;
        const int32_t* rows = p.rows + b * p.r_sb + h * p.r_sh;
        for (int i0 = 0; i0 < count; i0 += kMoves * kMoveThreads) {
            int row[kMoves], prior[kMoves];
            float x[kMoves];
            bool good[kMoves];
#pragma unroll
            for (int y = 0; y < kMoves; ++y) {
                const int i = min(i0 + y * kMoveThreads + tid, count - 1);
                row[y] = rows[i];
                prior[y] = rows[max(i - 1, 0)];
            }
#pragma unroll
            for (int y = 0; y < kMoves; ++y) {
                const int i = i0 + y * kMoveThreads + tid;
                good[y] = i < count && may_move(row[y], i ? prior[y] : -1, i, p.wkeys);
                if (i < count && !good[y]) report_bad_row(p.c.status);
                if (good[y]) x[y] = w[row[y]];
            }
            reads_done();
#pragma unroll
            for (int y = 0; y < kMoves; ++y)
                if (good[y]) w[i0 + y * kMoveThreads + tid] = x[y];
        }
        __syncthreads();
        for (int i = count + tid; i < p.wkeys; i += kMoveThreads) w[i] = 0.f;
        return;
    }
    const int h = (int)blockIdx.x / per_head, rest = (int)blockIdx.x % per_head;
    const int lane = tid & ((1 << p.lanes_log) - 1), at = tid >> p.lanes_log;
    const int kind = rest / cols, d = ((rest % cols) << (p.lanes_log + 3)) + 8 * lane;
    const int32_t* rows = p.rows + b * p.r_sb + h * p.r_sh;
    uint16_t* base = const_cast<uint16_t*>(kind ? p.c.v + h * p.c.v_sh : p.c.k + h * p.c.k_sh) + d;
    const int64_t sb = kind ? p.c.v_sb : p.c.k_sb, sn = kind ? p.c.v_sn : p.c.k_sn;
    const int64_t* table = p.c.table + b * p.c.t_sb;
    const int step = kMoveThreads >> p.lanes_log;          // rows a thread's moves lie apart
    for (int i0 = 0; i0 < count; i0 += kMoves * step) {
        int row[kMoves], prior[kMoves];
        u32x4 x[kMoves];
        uint16_t* dst[kMoves];                             // null: nothing moves
#pragma unroll
        for (int y = 0; y < kMoves; ++y) {
            const int i = min(i0 + y * step + at, count - 1);
            row[y] = rows[i];
            prior[y] = rows[max(i - 1, 0)];
        }
        int64_t from[kMoves], to[kMoves];                  // blocks
#pragma unroll
        for (int y = 0; y < kMoves; ++y) {
            const int i = i0 + y * step + at;
            bool good = i < count && may_move(row[y], i ? prior[y] : -1, i, p.c.keys);
            if (i < count && !good) report_bad_row(p.c.status);
            if constexpr (PAGED) {
                from[y] = good ? table_page(table[quotient(row[y], p.c.block)], p.c.num_blocks) : 0;
                to[y] = good ? table_page(table[quotient(i, p.c.block)], p.c.num_blocks) : 0;
            }
            if (!good) row[y] = -1;
        }
#pragma unroll
        for (int y = 0; y < kMoves; ++y) {
            const int i = i0 + y * step + at;
            dst[y] = nullptr;
            const uint16_t* src = base;
            if (row[y] >= 0) {
                if constexpr (PAGED) {
                    if (from[y] < 0 || to[y] < 0) {
                        report_bad_page(p.c.status);
                    } else {
                        const int B = (int)p.c.block.d;
                        src = base + from[y] * sb + (row[y] - quotient(row[y], p.c.block) * B) * sn;
                        dst[y] = base + to[y] * sb + (i - quotient(i, p.c.block) * B) * sn;
                    }
                } else {
                    src = base + b * sb + row[y] * sn;
                    dst[y] = base + b * sb + i * sn;
                }
            }
            if (row[y] == i) dst[y] = nullptr;
            if (dst[y]) x[y] = *reinterpret_cast<const u32x4*>(src);
        }
        reads_done();
#pragma unroll
        for (int y = 0; y < kMoves; ++y)
            if (dst[y]) *reinterpret_cast<u32x4*>(dst[y]) = x[y];
    }
}

}  // namespace

}  // namespace slimkv

using namespace slimkv;

namespace {

int check_select(const slimkv_select_rows_args* a) {
    if (!a) return fail(SLIMKV_EINVAL, "select rows: null pointer");
    if (a->batch < 0 || a->batch > 0x7fffffff || a->heads <= 0 || a->heads > 0x7fffffff || a->batch * a->heads > 0x7fffffff ||
        a->keys < 0 || a->keys > ((int64_t)1 << 30) || a->keep <= 0 || a->keep > ((int64_t)1 << 30) || a->sink < 0 ||
        a->recent < 0)
        return fail(SLIMKV_EINVAL, "select rows: invalid sizes");
    if (a->sink > a->keep || a->recent > a->keep - a->sink)
        return fail(SLIMKV_EINVAL, "select rows: the first and the recent rows exceed the rows kept");
    return SLIMKV_OK;
}

}  // namespace

extern "C" size_t slimkv_select_rows_workspace(const slimkv_select_rows_args* a) {
    return check_select(a) == SLIMKV_OK ? select_bytes(a) : 0;
}

extern "C" int slimkv_select_rows(const slimkv_select_rows_args* a, void* workspace, size_t workspace_bytes,
                                  void* stream) {
    const int code = check_select(a);
    if (code != SLIMKV_OK) return code;
    if (a->batch == 0) return SLIMKV_OK;
    if ((!a->weights && a->keys > 0) || !a->rows || !a->counts) return fail(SLIMKV_EINVAL, "select rows: null pointer");
    SelectParams p{};
    p.weights = a->weights; p.w_sb = a->w_sb; p.w_sh = a->w_sh;
    p.lengths = a->lengths; p.rows = a->rows; p.counts = a->counts;
    p.H = (int)a->heads; p.keys = (int)a->keys; p.keep = (int)a->keep; p.sink = (int)a->sink; p.recent = (int)a->recent;
    p.chunks = select_chunks(a);
    p.ws = static_cast<uint32_t*>(workspace);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const unsigned rows = (unsigned)(a->batch * a->heads);
    const bool held = a->keys <= kMostHeld * kHeldThreads;
    if (!launchable(rows, held ? kHeldThreads : kSelectThreads))
        return fail(SLIMKV_EINVAL, "select rows: too many rows for one call");
    if (held) {
        void (*kernel)(SelectParams) = a->keys <= 4 * kHeldThreads    ? select_held_kernel<4>
                                       : a->keys <= 8 * kHeldThreads  ? select_held_kernel<8>
                                       : a->keys <= 16 * kHeldThreads ? select_held_kernel<16>
                                                                      : select_held_kernel<kMostHeld>;
        hipLaunchKernelGGL(kernel, dim3(rows), dim3(kHeldThreads), 0, st, p);
    } else if (p.chunks == 1) {
        hipLaunchKernelGGL(select_kernel, dim3(rows), dim3(kSelectThreads), 0, st, p);
    } else {
        if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3) || workspace_bytes < select_bytes(a))
            return fail(SLIMKV_EWORKSPACE, "select rows: workspace missing, misaligned or too small");
        const dim3 grid((unsigned)p.chunks, rows);
        hipLaunchKernelGGL(select_chunk_kernel<1>, grid, dim3(kSelectThreads), 0, st, p);
        hipLaunchKernelGGL(select_chunk_kernel<2>, grid, dim3(kSelectThreads), 0, st, p);
        hipLaunchKernelGGL(select_chunk_kernel<3>, grid, dim3(kSelectThreads), 0, st, p);
        hipLaunchKernelGGL(select_chunk_kernel<4>, grid, dim3(kSelectThreads), 0, st, p);
    }
    return check_hip(hipGetLastError(), "select rows launch");
}

extern "C" int slimkv_compact_rows(const slimkv_compact_rows_args* a, void* stream) {
    if (!a) return fail(SLIMKV_EINVAL, "compact rows: null pointer");
    if (a->head_dim != 64 && a->head_dim != 128)
        return fail(SLIMKV_EUNSUP, "compact rows: head_dim must be 64 or 128");
    if (a->dtype != SLIMKV_DTYPE_BF16 && a->dtype != SLIMKV_DTYPE_F16)
        return fail(SLIMKV_EUNSUP, "compact rows: element type must be bf16 or fp16");
    if (a->batch < 0 || a->batch > 65535 || a->kv_heads <= 0 || a->kv_heads > 4096 || a->keep < 0 ||
        a->keep > ((int64_t)1 << 30) || a->weight_keys < 0 || a->weight_keys > ((int64_t)1 << 30) ||
        (a->weight_heads != 0 && a->weight_heads != a->kv_heads && a->weight_heads != 1))
        return fail(SLIMKV_EINVAL, "compact rows: invalid sizes");
    if (a->batch == 0 || (a->keep == 0 && !a->in_place)) return SLIMKV_OK;
    if ((!a->rows && a->keep > 0) || !a->counts || (a->weight_heads && a->weight_keys && !a->weights) ||
        (!a->in_place && (!a->out_k || !a->out_v || (a->weight_heads && !a->out_weights))))
        return fail(SLIMKV_EINVAL, "compact rows: null pointer");
    CompactParams p{};
    const int view = cache_view(a->cache, a->batch, a->kv_heads, a->head_dim, true, "compact rows", &p.c);
    if (view != SLIMKV_OK) return view;
    if (a->in_place && a->cache.keys > 0) {
        const slimkv_cache_rows& c = a->cache;
        const bool many = a->batch > 1, pages = c.table != nullptr;
        if (c.k == c.v || (many && (pages ? c.t_sb == 0 : c.k_sb == 0 || c.v_sb == 0)) ||
            (a->kv_heads > 1 && (c.k_sh == 0 || c.v_sh == 0)) || (a->weight_heads > 1 && a->weight_keys > 0 && a->w_sh == 0) ||
            (many && a->weight_heads && a->weight_keys > 0 && a->w_sb == 0))
            return fail(SLIMKV_EINVAL, "compact rows: in place every sequence and head needs rows of its own");
    }
    if (!a->in_place && (!rows_aligned(a->out_k, {{a->batch, a->ok_sb}, {a->keep, a->ok_sn}, {a->kv_heads, a->ok_sh}}) ||
                         !rows_aligned(a->out_v, {{a->batch, a->ov_sb}, {a->keep, a->ov_sn}, {a->kv_heads, a->ov_sh}})))
        return fail(SLIMKV_EINVAL, "compact rows: output rows must start on 16-byte boundaries");
    p.rows = a->rows; p.r_sb = a->r_sb; p.r_sh = a->r_sh; p.counts = a->counts;
    p.ok = static_cast<uint16_t*>(a->out_k); p.ok_sb = a->ok_sb; p.ok_sn = a->ok_sn; p.ok_sh = a->ok_sh;
    p.ov = static_cast<uint16_t*>(a->out_v); p.ov_sb = a->ov_sb; p.ov_sn = a->ov_sn; p.ov_sh = a->ov_sh;
    p.weights = a->weights; p.w_sb = a->w_sb; p.w_sh = a->w_sh;
    p.ow = a->out_weights; p.ow_sb = a->ow_sb; p.ow_sh = a->ow_sh;
    p.Hw = (int)a->weight_heads; p.wkeys = (int)a->weight_keys;
    p.Hk = (int)a->kv_heads; p.D = (int)a->head_dim; p.keep = (int)a->keep;
    hipStream_t st = static_cast<hipStream_t>(stream);
    int64_t move, weights;
    if (a->in_place) {
        p.lanes_log = (int64_t)a->batch * a->kv_heads * 2 * (a->head_dim / 64) >= device_cu_count() ? 3 : 2;
        move = a->kv_heads * 2 * (a->head_dim >> (p.lanes_log + 3));
        weights = a->weight_heads;
    } else {
        const int64_t per = 256 / (a->head_dim / 8);
        move = (a->keep * a->kv_heads + per - 1) / per;
        weights = (a->weight_heads * a->keep + 255) / 256;
    }
    if (!launchable(move + weights, a->in_place ? kMoveThreads : 256))
        return fail(SLIMKV_EINVAL, "compact rows: too many rows for one call");
    p.move_blocks = (int)move;
    const dim3 grid((unsigned)(move + weights), (unsigned)a->batch);
    if (a->in_place) {
        if (p.c.table) hipLaunchKernelGGL(compact_in_place_kernel<true>, grid, dim3(kMoveThreads), 0, st, p);
        else hipLaunchKernelGGL(compact_in_place_kernel<false>, grid, dim3(kMoveThreads), 0, st, p);
    } else {
        void (*kernel)(CompactParams);
        if (p.r_sh) kernel = p.c.table ? compact_kernel<true, true> : compact_kernel<false, true>;
        else kernel = p.c.table ? compact_kernel<true, false> : compact_kernel<false, false>;
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p);
    }
    return check_hip(hipGetLastError(), "compact rows launch");
}
