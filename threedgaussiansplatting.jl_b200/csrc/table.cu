// table.cu — rows of SH coefficients shared through a table.
//   gs3d_table_lookup    out[i] = scale * table[indices[i]]
//   gs3d_table_gradient  table_grads[k] = scale * sum of grads[f] over the rows f with index k + 1,
//                        by the rows sorted by index (stable), so the order of every sum is fixed
#include <cooperative_groups.h>

#include <type_traits>
#include <utility>

#include "common.cuh"
#include "internal.h"
#include "rows.cuh"

namespace gs3d {
namespace {

// ---- lookup ----------------------------------------------------------------------------------
// out[i] = table[indices[i] - 1] * scale. Bound by the rows written (the table stays in L2). Threads side
// by side on a row's units of N elements, ROWS rows a thread, as many independent loads in flight. A unit
// is 16 bytes of the wider of table and output (two half types: of both), or less as the rows' lengths and
// starts allow (3M x 48 fp32 with 1 / 2 / 4 / 8 rows: 129 / 103 / 94 / 117 us; a write-only fill of as much: 79).
// Of units of one or two elements a thread takes COLS of a row, a share of the columns apart, for one
// index and one address (500K x 27 bf16: 17.1 us with one column, 15.0 with two, 19.8 with four; 1M x 54
// bf16 by pairs: 40.0, 35.9): bound by the instructions. Odd rows by the output's 32-bit words, whose halves
// come from two words of the table where the rows' parities differ, took 21 us.
constexpr int kLookupRows = 4, kLookupColumns = 2;

template <typename T, int N>
struct alignas(N * sizeof(T)) Pack {
    T e[N];
};

template <size_t BYTES>
using PackWord =
    typename std::conditional<BYTES == 16, uint4, typename std::conditional<BYTES == 8, uint2, uint32_t>::type>::type;

// A pack to memory that is not read again soon: streamed, so that it does not push
// the table out of L2 (104 us without, 94 with). Single elements go the ordinary way: L2 joins them.
template <typename T, int N>
__device__ __forceinline__ void store_streaming(T* p, const Pack<T, N>& v) {
    if constexpr (N == 1) {
        *p = v.e[0];
    } else {
        using W = PackWord<sizeof(v)>;
        __stcs(reinterpret_cast<W*>(p), *reinterpret_cast<const W*>(&v));
    }
}

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
    if constexpr (N == 1) {
        return Pack<T, N>{__ldg(p)};
    } else {
        using W = PackWord<sizeof(Pack<T, N>)>;
        const W w = __ldg(reinterpret_cast<const W*>(p));
        return *reinterpret_cast<const Pack<T, N>*>(&w);
    }
}

template <typename TI, typename TO, int N, int ROWS, int COLS>
__global__ void __launch_bounds__(256) k_table_lookup(const TI* __restrict__ table, int rows, int table_stride,
                                                      const int32_t* __restrict__ indices, float scale,
                                                      TO* __restrict__ out, int n, int64_t out_stride, int units,
                                                      int tile_units, int slots) {
    const int slot = threadIdx.x / tile_units;
    const int unit = blockIdx.y * (COLS * tile_units) + threadIdx.x - slot * tile_units;  // the first of COLS
    if (unit >= units) return;
    const int first = blockIdx.x * (slots * ROWS) + slot;
    const TI* column = table + unit * N;
    const int32_t* index = indices + first;
    TO* o = out + first * out_stride + unit * N;
    const int64_t step = slots * out_stride;
    const auto rows_of_thread = [&](auto full) {
        int k[ROWS];
#pragma unroll
        for (int q = 0; q < ROWS; ++q) k[q] = full || first + q * slots < n ? __ldg(index + q * slots) - 1 : -1;
        Pack<TI, N> v[ROWS][COLS];
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
            const TI* p = column + (int64_t)k[q] * table_stride;
#pragma unroll
            for (int j = 0; j < COLS; ++j) {
                v[q][j] = Pack<TI, N>{};
                if ((unsigned)k[q] < (unsigned)rows && (j == 0 || unit + j * tile_units < units))
                    v[q][j] = load_pack<TI, N>(p + j * tile_units * N);
            }
        }
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
            const float f = (unsigned)k[q] < (unsigned)rows ? scale : 0.0f;  // zeros whatever the scale
#pragma unroll
            for (int j = 0; j < COLS; ++j) {
                Pack<TO, N> p;
#pragma unroll
                for (int c = 0; c < N; ++c) p.e[c] = from_f32<TO>(to_f32(v[q][j].e[c]) * f);
                if ((full || first + q * slots < n) && (j == 0 || unit + j * tile_units < units))
                    store_streaming(o + j * tile_units * N, p);
            }
            o += step;
        }
    };
    if ((int)(blockIdx.x + 1) * (slots * ROWS) <= n) rows_of_thread(std::true_type{});
    else rows_of_thread(std::false_type{});
}

template <typename T>
bool packs(const gs3d_rows* r, int n) {
    return r->dim % n == 0 && r->row_stride % n == 0 && reinterpret_cast<uintptr_t>(r->data) % (n * sizeof(T)) == 0;
}

template <typename TI, typename TO, int N, int ROWS, int COLS>
int launch_lookup_units(const gs3d_rows* table, const int32_t* indices, float scale, const gs3d_rows* out,
                        cudaStream_t stream) {
    const int units = out->dim / N, tile_units = std::min((int)ceil_div(units, COLS), 256);
    const int slots = std::max(1, 256 / tile_units);
    const dim3 grid((unsigned)ceil_div(out->rows, (int64_t)slots * ROWS), (unsigned)ceil_div(units, COLS * tile_units));
    k_table_lookup<TI, TO, N, ROWS, COLS><<<grid, slots * tile_units, 0, stream>>>(
        static_cast<const TI*>(table->data), (int)table->rows, (int)table->row_stride, indices, scale,
        static_cast<TO*>(out->data), (int)out->rows, out->row_stride, units, tile_units, slots);
    GS3D_LAUNCHED("k_table_lookup");
    return GS3D_OK;
}

template <typename TI, typename TO>
int launch_lookup(const gs3d_rows* table, const int32_t* indices, float scale, const gs3d_rows* out,
                  cudaStream_t stream) {
    if constexpr (sizeof(TI) == 2 && sizeof(TO) == 2)
        if (packs<TI>(table, 8) && packs<TO>(out, 8))
            return launch_lookup_units<TI, TO, 8, kLookupRows, 1>(table, indices, scale, out, stream);
    if (packs<TI>(table, 4) && packs<TO>(out, 4))
        return launch_lookup_units<TI, TO, 4, kLookupRows, 1>(table, indices, scale, out, stream);
    if (packs<TI>(table, 2) && packs<TO>(out, 2))
        return launch_lookup_units<TI, TO, 2, kLookupRows, kLookupColumns>(table, indices, scale, out, stream);
    return launch_lookup_units<TI, TO, 1, kLookupRows, kLookupColumns>(table, indices, scale, out, stream);
}

// ---- gradient --------------------------------------------------------------------------------
// 1. Stable sort of the rows by table row (k_radix_*: tiles of 1024 to 4096 rows, digits of up to 10 bits,
//    three launches and one pass per 10 bits of the row number; up to 16384 rows k_sort_cluster, one cluster
//    in one launch; up to 1024 k_table_gradient_tiny does everything). Rows without a valid index drop
//    out of the first pass, which also zeroes the table's gradients.
// 2. k_table_segments: the sorted rows are cut into chunks of equal length, a block each, and a chunk
//    into one run of rows per slot (a slot: the threads side by side on a row's columns). A slot adds
//    its rows in order; a run of equal indices that crosses slots is added up in slot order through
//    shared memory, and what crosses a chunk's border is left as a partial sum.
// 3. k_table_join: the block in whose chunk such a run starts adds its partial sums in chunk order.
// The order of every sum follows from the sorted order and the sizes, whatever the number of rows that
// share an index: no atomics, and a row that half of the Gaussians use is spread over the GPU like any
// other. 3M x 48 fp32 into 65,536 rows, 194 us (the bytes alone: 93): sort 61 (count 8 to 15 a pass, bound
// by the gathers of the indices; spine 3; scatter 20, bound by ranking in shared memory: matched by
// ballots, 30 with match_any), sums 125 (the random 192-byte gather alone: 107 to 112), join 5.

// The kernels of one call follow one another with programmatic dependent launch: each starts while
// the one before it ends, and waits in `after_predecessor` (every thread, before anything else, so
// that the chain holds for all kernels before) until that one's writes are there. What a predecessor
// wrote is read with ordinary loads or through L2, not as read-only data.
__device__ __forceinline__ void after_predecessor() {
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <typename... P, typename... A>
int launch_after(const char* what, void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                 A&&... args) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    GS3D_CUDA(cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...), what);
    return GS3D_OK;
}

constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxDigitBits = 10;

// Row f's table row 0 .. rows - 1, or -1 where it takes no part.
struct KeySource {
    const int32_t* indices;
    const int32_t* f2g;
    const int32_t* counts;
    int64_t n_indices;
    int32_t n, rows;

    __device__ __forceinline__ int live() const { return counts ? min(max(counts[0], 0), n) : n; }
    // The keys of rows f0, f0 + 32, ...: all of a step's loads before the next step's.
    template <int R>
    __device__ __forceinline__ void keys(int f0, int (&key)[R]) const {
        const int last = live();
        int64_t i[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int f = f0 + 32 * r;
            i[r] = f >= last ? -1 : f2g ? (int64_t)__ldg(f2g + f) - 1 : f;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) key[r] = i[r] >= 0 && i[r] < n_indices ? __ldg(indices + i[r]) : 0;
#pragma unroll
        for (int r = 0; r < R; ++r) key[r] = key[r] >= 1 && key[r] <= rows ? key[r] - 1 : -1;
    }
};

// The zeroed table gradients (data NULL: accumulate, nothing to zero).
struct ZeroRows {
    float* data;
    int64_t stride;
    int32_t rows, dim;

    __device__ __forceinline__ void fill(int64_t thread, int64_t threads) const {
        if (!data) return;
        const int64_t total = (int64_t)rows * dim;
        if (stride == dim && (reinterpret_cast<uintptr_t>(data) & 15) == 0) {
            float4* d4 = reinterpret_cast<float4*>(data);
            for (int64_t i = thread; i < total / 4; i += threads) d4[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int64_t i = (total & ~(int64_t)3) + thread; i < total; i += threads) data[i] = 0.0f;
        } else {
            for (int64_t i = thread; i < total; i += threads) {
                const int64_t r = i / dim;
                data[r * stride + (i - r * dim)] = 0.0f;
            }
        }
    }
};

// An item: x the row's index - 1 in the table, y the row.
struct SortPass {
    int32_t* first_keys;  // the first pass: all rows' indices, -1 without one, written by its count kernel
    const int2* in;       // NULL: the first pass
    int2* out;
    int32_t* hist;    // [bin][tile]: counts, then their exclusive scan over the tiles
    int32_t* totals;  // [bin]
    int32_t* valid;   // number of rows with a valid index (written by the first pass)
    int32_t n, ntiles, shift, bits;
};

// A thread's place in a tile: its rows are place, place + 32, ..., warp after warp in row order.
template <int ROUNDS>
__device__ __forceinline__ int tile_place(int tile) {
    return tile * (kSortThreads * ROUNDS) + (threadIdx.x >> 5) * (ROUNDS * 32) + (threadIdx.x & 31);
}

template <int ROUNDS>
__global__ void __launch_bounds__(kSortThreads) k_radix_count(const SortPass p, const KeySource src,
                                                              const ZeroRows zero) {
    __shared__ int bins[1 << kMaxDigitBits];
    after_predecessor();
    const int fillers = gridDim.x - p.ntiles;  // blocks behind the tiles', which zero the table
    if ((int)blockIdx.x >= p.ntiles) {
        zero.fill((int64_t)(blockIdx.x - p.ntiles) * kSortThreads + threadIdx.x, (int64_t)fillers * kSortThreads);
        return;
    }
    const int nbins = 1 << p.bits, tile = blockIdx.x, place = tile_place<ROUNDS>(tile);
    for (int b = threadIdx.x; b < nbins; b += kSortThreads) bins[b] = 0;
    int key[ROUNDS];
    if (!p.in) {
        src.keys(place, key);
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (place + 32 * r < p.n) p.first_keys[place + 32 * r] = key[r];
    } else {
        const int m = *p.valid;
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) key[r] = place + 32 * r < m ? p.in[place + 32 * r].x : -1;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        if (key[r] >= 0) atomicAdd(&bins[(key[r] >> p.shift) & (nbins - 1)], 1);
    if (!p.in && fillers == 0) zero.fill((int64_t)tile * kSortThreads + threadIdx.x, (int64_t)p.ntiles * kSortThreads);
    __syncthreads();
    for (int b = threadIdx.x; b < nbins; b += kSortThreads) p.hist[(int64_t)b * p.ntiles + tile] = bins[b];
}

constexpr int kSpineThreads = 256;

// Block b: exclusive scan of bin b's counts over the tiles.
__global__ void __launch_bounds__(kSpineThreads) k_radix_spine(const SortPass p) {
    __shared__ int sm[33];
    after_predecessor();
    int32_t* row = p.hist + (int64_t)blockIdx.x * p.ntiles;
    int carry = 0, tot;
    for (int t0 = 0; t0 < p.ntiles; t0 += kSpineThreads) {
        const int t = t0 + threadIdx.x;
        const int ex = block_exclusive_scan(t < p.ntiles ? row[t] : 0, sm, &tot);
        if (t < p.ntiles) row[t] = carry + ex;
        carry += tot;
    }
    if (threadIdx.x == 0) p.totals[blockIdx.x] = carry;
}

size_t radix_scatter_smem(int rounds, int bits) {
    return (size_t)rounds * kSortThreads * 8 + (size_t)(1 << bits) * (4 + 2 * kSortWarps);
}

// Exclusive block scan of one 64-bit value per thread of kSortThreads.
__device__ __forceinline__ int64_t block_exclusive_scan64(int64_t v, int64_t* sm) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
    }
    if (lane == 31) sm[w] = inc;
    __syncthreads();
    if (w == 0) {
        int64_t t = lane < kSortWarps ? sm[lane] : 0;
#pragma unroll
        for (int o = 1; o < kSortWarps; o <<= 1) {
            const int64_t u = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += u;
        }
        if (lane < kSortWarps) sm[lane] = t;
    }
    __syncthreads();
    return inc - v + (w ? sm[w - 1] : 0);
}

template <int ROUNDS>
__global__ void __launch_bounds__(kSortThreads, 2) k_radix_scatter(const SortPass p) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int64_t sm[kSortWarps];
    constexpr int BINS = (1 << kMaxDigitBits) / kSortThreads;  // of a thread, at most
    after_predecessor();
    const int nbins = 1 << p.bits, tile = blockIdx.x;
    int2* items = reinterpret_cast<int2*>(smem);                   // the tile in digit order
    // a bin's place in the output, minus in the tile
    int32_t* dest = reinterpret_cast<int32_t*>(items + ROUNDS * kSortThreads);
    uint16_t* wcount = reinterpret_cast<uint16_t*>(dest + nbins);  // [warp][bin]
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int place = tile_place<ROUNDS>(tile), m = p.in ? *p.valid : p.n;
    int2 item[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int i = place + 32 * r;
        item[r] = make_int2(-1, i);
        if (i < m) {
            if (p.in) item[r] = p.in[i];
            else item[r].x = p.first_keys[i];
        }
    }
    // this thread's bins: totals over all tiles, and over the tiles before this one
    int total[BINS], before_tile[BINS];
    const int bins = max(1, nbins / kSortThreads), bin0 = threadIdx.x * bins;
#pragma unroll
    for (int b = 0; b < BINS; ++b) {
        const bool on = b < bins && bin0 + b < nbins;
        total[b] = on ? p.totals[bin0 + b] : 0;
        before_tile[b] = on ? p.hist[(int64_t)(bin0 + b) * p.ntiles + tile] : 0;
    }
    for (int i = threadIdx.x; i < nbins * kSortWarps / 2; i += kSortThreads) reinterpret_cast<uint32_t*>(wcount)[i] = 0;
    __syncthreads();
    // stable rank of every key among its warp's keys of the same digit: within its 32, then behind the 32s
    // before
    int rank[ROUNDS];
    const unsigned below = (1u << lane) - 1u;
    unsigned peers[ROUNDS];  // lanes with the same digit, bit by bit
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) peers[r] = __ballot_sync(0xffffffffu, item[r].x >= 0);
    for (int b = p.shift; b < p.shift + p.bits; ++b)
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const bool bit = (item[r].x >> b) & 1;
            const unsigned ones = __ballot_sync(0xffffffffu, bit);
            peers[r] &= bit ? ones : ~ones;
        }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) rank[r] = __popc(peers[r] & below) | __popc(peers[r]) << 8;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const bool on = item[r].x >= 0;
        uint16_t& c = wcount[w * nbins + (on ? (item[r].x >> p.shift) & (nbins - 1) : 0)];
        const int before = c, mine = rank[r] & 255, all = rank[r] >> 8;
        rank[r] = before + mine;
        __syncwarp();
        if (on && mine == 0) c = (uint16_t)(before + all);
        __syncwarp();
    }
    __syncthreads();
    // places of the bins in the tile (low words, over this tile's counts) and in the output (high words,
    // over all totals)
    int here[BINS];
    int64_t sum = 0;
#pragma unroll
    for (int b = 0; b < BINS; ++b) {
        here[b] = 0;
        if (b < bins && bin0 + b < nbins)
#pragma unroll
            for (int ww = 0; ww < kSortWarps; ++ww) here[b] += wcount[ww * nbins + bin0 + b];
        sum += ((int64_t)total[b] << 32) + here[b];
    }
    int64_t base = block_exclusive_scan64(sum, sm);
    const int64_t all = sm[kSortWarps - 1];
#pragma unroll
    for (int b = 0; b < BINS; ++b)
        if (b < bins && bin0 + b < nbins) {
            int at = (int)base;
            dest[bin0 + b] = (int)(base >> 32) + before_tile[b] - at;
#pragma unroll
            for (int ww = 0; ww < kSortWarps; ++ww) {
                uint16_t& c = wcount[ww * nbins + bin0 + b];
                const int count = c;
                c = (uint16_t)at;
                at += count;
            }
            base += ((int64_t)total[b] << 32) + here[b];
        }
    if (!p.in && tile == 0 && threadIdx.x == 0) *p.valid = (int32_t)(all >> 32);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        if (item[r].x >= 0) items[wcount[w * nbins + ((item[r].x >> p.shift) & (nbins - 1))] + rank[r]] = item[r];
    __syncthreads();
    const int count = (int)all;
    for (int i = threadIdx.x; i < count; i += kSortThreads) {
        const int2 it = items[i];
        p.out[dest[(it.x >> p.shift) & (nbins - 1)] + i] = it;
    }
}

// The rows with a valid index among the first THREADS * ROUNDS, sorted by one block in shared memory,
// 8 bits a pass; returns their number.
template <int THREADS, int ROUNDS>
__device__ __forceinline__ int sort_rows(const KeySource& src, int bits, int2* items, uint16_t (*wcount)[256],
                                         int* start, int* sm) {
    constexpr int WARPS = THREADS / 32;
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned below = (1u << lane) - 1u;
    const int place = w * (ROUNDS * 32) + lane;
    int count = 0;
    for (int shift = 0; shift < max(bits, 1); shift += 8) {
        int key[ROUNDS], row[ROUNDS], rank[ROUNDS];
        if (shift == 0) src.keys(place, key);
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int i = place + 32 * r;
            row[r] = i;
            if (shift) {
                const int2 it = items[i];
                key[r] = i < count ? it.x : -1;
                row[r] = it.y;
            }
        }
        for (int i = threadIdx.x; i < WARPS * 256; i += THREADS) (&wcount[0][0])[i] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int d = key[r] >= 0 ? (key[r] >> shift) & 255 : 256;
            const unsigned peers = __match_any_sync(0xffffffffu, d);
            const int before = d < 256 ? wcount[w][d] : 0;
            rank[r] = before + __popc(peers & below);
            __syncwarp();
            if (d < 256 && (peers & below) == 0) wcount[w][d] = (uint16_t)(before + __popc(peers));
            __syncwarp();
        }
        __syncthreads();
        int run = 0;
        if (threadIdx.x < 256)
#pragma unroll
            for (int ww = 0; ww < WARPS; ++ww) {
                const int c = wcount[ww][threadIdx.x];
                wcount[ww][threadIdx.x] = (uint16_t)run;
                run += c;
            }
        const int st = block_exclusive_scan(run, sm, &count);
        if (threadIdx.x < 256) start[threadIdx.x] = st;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (key[r] >= 0) {
                const int d = (key[r] >> shift) & 255;
                items[start[d] + wcount[w][d] + rank[r]] = make_int2(key[r], row[r]);
            }
        __syncthreads();
    }
    return count;
}

// Up to kClusterRows rows: one cluster sorts them, 8 bits a pass, the counts of its CTAs exchanged through
// distributed shared memory; the clusters behind it zero the table. One launch instead of three a pass,
// which for so few rows are bound by the host and by one another's latency: a whole gradient of 8,000 rows
// into 60,000 of 48 takes 18.5 us (27.7 by tiles), of 16,000 22.6 (27.7), of 32,000 it would take 30.2 (27.7).
constexpr int kClusterCtas = 8, kClusterThreads = 1024, kClusterRows = kClusterCtas * kClusterThreads * 2;

template <int ROUNDS>
__global__ void __cluster_dims__(kClusterCtas, 1, 1) __launch_bounds__(kClusterThreads)
    k_sort_cluster(const KeySource src, const ZeroRows zero, int bits, int2* __restrict__ out0,
                   int2* __restrict__ out1, int32_t* __restrict__ valid) {
    namespace cg = cooperative_groups;
    constexpr int WARPS = kClusterThreads / 32;
    __shared__ uint16_t wcount[WARPS][256];
    __shared__ int counts[256], start[256], sm[33];
    after_predecessor();
    if (blockIdx.x >= kClusterCtas) {
        zero.fill((int64_t)(blockIdx.x - kClusterCtas) * kClusterThreads + threadIdx.x,
                  (int64_t)(gridDim.x - kClusterCtas) * kClusterThreads);
        return;
    }
    cg::cluster_group cluster = cg::this_cluster();
    const int cta = blockIdx.x, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned below = (1u << lane) - 1u;
    const int place = cta * (kClusterThreads * ROUNDS) + w * (ROUNDS * 32) + lane;
    int count = 0;
    for (int shift = 0; shift < max(bits, 1); shift += 8) {
        const int2* in = shift & 8 ? out0 : out1;  // what the pass before wrote
        int2* out = shift & 8 ? out1 : out0;
        int key[ROUNDS], row[ROUNDS], rank[ROUNDS];
        if (shift == 0) src.keys(place, key);
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int i = place + 32 * r;
            row[r] = i;
            if (shift) {
                key[r] = -1;
                if (i < count) {
                    const int2 it = __ldcg(in + i);
                    key[r] = it.x;
                    row[r] = it.y;
                }
            }
        }
        for (int i = threadIdx.x; i < WARPS * 256 / 2; i += kClusterThreads)
            reinterpret_cast<uint32_t*>(&wcount[0][0])[i] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int d = key[r] >= 0 ? (key[r] >> shift) & 255 : 256;
            const unsigned peers = __match_any_sync(0xffffffffu, d);
            const int before = d < 256 ? wcount[w][d] : 0;
            rank[r] = before + __popc(peers & below);
            __syncwarp();
            if (d < 256 && (peers & below) == 0) wcount[w][d] = (uint16_t)(before + __popc(peers));
            __syncwarp();
        }
        __syncthreads();
        if (threadIdx.x < 256) {
            int run = 0;
#pragma unroll
            for (int ww = 0; ww < WARPS; ++ww) {
                const int c = wcount[ww][threadIdx.x];
                wcount[ww][threadIdx.x] = (uint16_t)run;
                run += c;
            }
            counts[threadIdx.x] = run;
        }
        cluster.sync();
        int total = 0, before_cta = 0;
        if (threadIdx.x < 256)
#pragma unroll
            for (int c = 0; c < kClusterCtas; ++c) {
                const int n = *cluster.map_shared_rank(counts + threadIdx.x, c);
                if (c < cta) before_cta += n;
                total += n;
            }
        const int st = block_exclusive_scan(total, sm, &count);
        if (threadIdx.x < 256) start[threadIdx.x] = st + before_cta;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (key[r] >= 0) {
                const int d = (key[r] >> shift) & 255;
                out[start[d] + wcount[w][d] + rank[r]] = make_int2(key[r], row[r]);
            }
        cluster.sync();  // every item is there, and every count was read
    }
    if (cta == 0 && threadIdx.x == 0) *valid = count;
}

// VB bytes of a row as VB / sizeof(T) floats.
template <typename T, int VB>
struct RowUnit {
    static constexpr int N = VB / (int)sizeof(T);
    alignas(VB) T e[N];
    __device__ __forceinline__ void load(const T* p) {
        // a row is read once, from a place of its own: nothing for L1, and 64 bytes a DRAM access
        // (a 3M x 192 B gather alone: 117 us plain, 107 us so)
        if constexpr (VB == 16) {
            uint4 v;
            asm("ld.global.nc.L1::no_allocate.L2::64B.v4.u32 {%0, %1, %2, %3}, [%4];"
                : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                : "l"(p));
            *reinterpret_cast<uint4*>(e) = v;
        } else if constexpr (VB == 8) {
            uint2 v;
            asm("ld.global.nc.L1::no_allocate.L2::64B.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
            *reinterpret_cast<uint2*>(e) = v;
        } else if constexpr (VB == 4 && sizeof(T) == 2) {
            *reinterpret_cast<uint32_t*>(e) = __ldg(reinterpret_cast<const uint32_t*>(p));
        } else {
            e[0] = __ldg(p);
        }
    }
};

// How a launch cuts the work: `units` units of VB bytes a row, in column tiles of at most 256; `slots`
// slots a block, each `run` sorted rows long.
struct SegmentPlan {
    int units, tile_units, slots, run, chunk, nchunks;
};

struct Segments {
    const int2* items;     // sorted
    const int32_t* valid;
    float* out;
    int64_t out_stride;
    float scale;
    int accumulate;
    int32_t* first_key;    // [chunk] index of its first row, -1: none
    int32_t* owned;        // [chunk] index whose run starts here and goes on in the next chunk, -1: none
    float* partial;        // [chunk][2][dim]: sums of a first run that began earlier, of the owned run
};

template <int N>
__device__ __forceinline__ void store_row(const Segments& g, int key, int col, const float (&s)[N]) {
    float* o = g.out + (int64_t)key * g.out_stride + col;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float v = g.scale * s[i];
        o[i] = g.accumulate ? o[i] + v : v;
    }
}

// The sums of one chunk: `count` items in shared memory, `run` after the other for each slot; every thread
// of the block calls it (those with slot >= pl.slots only wait). Where runs of equal indices cross from
// slot to slot the slot in which one starts adds the others' sums of it, from `part`, in slot order.
// open_left / open_right: the chunk's first / last run goes on in the chunk before / behind, and its sum
// goes to partial[0 ..] / partial[dim ..] (to the former if it is the same run).
template <typename T, int VB>
__device__ __forceinline__ void sum_chunk(const T* __restrict__ grads, int stride, int dim, const SegmentPlan& pl,
                                          int run, const Segments& g, const int2* items, int count, float* part,
                                          bool open_left, bool open_right, float* __restrict__ partial) {
    using Unit = RowUnit<T, VB>;
    // rows in flight a slot (1.2M x 119 bf16, an element a thread: 8 / 12 / 16 rows 53 / 46 / 41 us; 1M x 27
    // fp32: 54 / 55 / 58). In k_table_segments the half types then spill 12 to 44 bytes of their 48 or 64
    // registers a thread, fp32 none.
    constexpr int N = Unit::N, AHEAD = VB == 16 ? 6 : (VB < 8 && sizeof(T) == 2 ? 16 : 8);
    const int slot = threadIdx.x / pl.tile_units, lane = threadIdx.x - slot * pl.tile_units;
    const int unit = blockIdx.y * pl.tile_units + lane;
    const int col = unit * N;
    const bool on = unit < pl.units;
    const int width = pl.tile_units * N;
    const int j0 = slot * run, j1 = min(j0 + run, count);
    const bool some = slot < pl.slots && j0 < count;
    float acc[N];
    int cur = 0;
    bool from_left = false;  // the run in acc came from the slot before
    // a run that is complete, or goes on beyond the chunk
    const auto emit = [&](bool at_start, bool at_end) {
        if (!on) return;
        if (at_start && open_left || at_end && open_right) {
            float* p = partial + (at_start && open_left ? 0 : dim) + col;
#pragma unroll
            for (int i = 0; i < N; ++i) p[i] = acc[i];
        } else {
            store_row<N>(g, cur, col, acc);
        }
    };
    const auto hand_left = [&] {
#pragma unroll
        for (int i = 0; i < N; ++i) part[slot * width + lane * N + i] = acc[i];
    };
    bool first = true;
    if (some) {
        cur = items[j0].x;
        from_left = slot > 0 && items[j0 - 1].x == cur;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = 0.0f;
        const T* gc = grads + (on ? col : 0);
        for (int j = j0; j < j1; j += AHEAD) {
            Unit u[AHEAD];
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) u[q].load(gc + (int64_t)items[min(j + q, j1 - 1)].y * stride);
            if (j + AHEAD <= j1 && items[j + AHEAD - 1].x == cur) {  // sorted: all of them are
#pragma unroll
                for (int q = 0; q < AHEAD; ++q)
#pragma unroll
                    for (int i = 0; i < N; ++i) acc[i] += to_f32(u[q].e[i]);
                continue;
            }
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                if (j + q >= j1) break;
                const int key = items[j + q].x;
                if (key != cur) {
                    if (first && from_left) hand_left();
                    else emit(first && slot == 0, false);
                    first = false;
                    cur = key;
#pragma unroll
                    for (int i = 0; i < N; ++i) acc[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i] += to_f32(u[q].e[i]);
            }
        }
        if (first && from_left) hand_left();
    }
    __syncthreads();
    if (!some || (first && from_left)) return;
    int end = j1;
    for (int s = slot + 1; end < count && items[end].x == cur; ++s) {
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += part[s * width + lane * N + i];
        const int next = min(end + run, count);
        if (items[next - 1].x != cur) break;  // it ends inside that slot
        end = next;
    }
    emit(first && slot == 0, end == count);
}

template <typename T, int VB>
__global__ void __launch_bounds__(256, VB == 16 ? 4 : 5)
    k_table_segments(const T* __restrict__ grads, int stride, int dim, const SegmentPlan pl, const Segments g) {
    extern __shared__ __align__(16) unsigned char smem[];
    int2* items = reinterpret_cast<int2*>(smem);                // the chunk's
    float* part = reinterpret_cast<float*>(items + pl.chunk);   // [slot][tile_units * N]
    after_predecessor();
    const int m = *g.valid;
    const int begin = blockIdx.x * pl.chunk, count = min(pl.chunk, m - begin);
    const bool meta = threadIdx.x == 0 && blockIdx.y == 0;
    if (count <= 0) {
        if (meta) g.first_key[blockIdx.x] = g.owned[blockIdx.x] = -1;
        return;
    }
    __shared__ int outside[2];  // the keys before and behind the chunk
    for (int i = threadIdx.x; i < count; i += blockDim.x) items[i] = __ldcg(g.items + begin + i);
    if (threadIdx.x < 2) {
        const int at = threadIdx.x ? begin + count : begin - 1;
        outside[threadIdx.x] = at >= 0 && at < m ? __ldcg(g.items + at).x : -1;
    }
    __syncthreads();
    const int head = items[0].x, last = items[count - 1].x;
    const bool open_left = outside[0] == head, open_right = outside[1] == last;
    const bool earlier = open_left && head == last;
    if (meta) {
        g.first_key[blockIdx.x] = head;
        g.owned[blockIdx.x] = open_right && !earlier ? last : -1;
    }
    sum_chunk<T, VB>(grads, stride, dim, pl, pl.run, g, items, count, part, open_left, open_right,
                     g.partial + (int64_t)blockIdx.x * 2 * dim);
}

// Up to kTinyRows rows in one launch: every block sorts all of them in shared memory and takes the runs
// that start in its share of the sorted rows; nothing crosses a border, so nothing is left to join. It
// also zeroes, of its share of the table, the rows without gradients.
constexpr int kTinyRows = 1024, kTinyThreads = 256;

// Zeroes the rows first .. last - 1 of the table that no item names: marks those that are named, kZeroRows
// rows a turn, and leaves each row to 16 bytes (or an element) a thread of as many threads side by side
// (1,000 rows into 60,000 of 48: 12.4 us, 24.7 with a search and a thread a row).
constexpr int kZeroRows = 16384;

__device__ __forceinline__ void zero_unused(const ZeroRows& z, const int2* items, int count, int64_t first,
                                            int64_t last, uint32_t* used) {
    const bool wide = ((z.stride | z.dim) & 3) == 0 && (reinterpret_cast<uintptr_t>(z.data) & 15) == 0;
    const int units = wide ? z.dim / 4 : z.dim, side = min(32, 1 << (32 - __clz(units - 1 | 1)));
    const int lane = threadIdx.x & (side - 1);
    for (int64_t r = first; r < last; r += kZeroRows) {
        const int m = (int)min((int64_t)kZeroRows, last - r);
        for (int i = threadIdx.x; i < (m + 31) / 32; i += kTinyThreads) used[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < count; i += kTinyThreads) {
            const int64_t k = items[i].x - r;
            if (k >= 0 && k < m) atomicOr(used + (k >> 5), 1u << (k & 31));
        }
        __syncthreads();
        for (int k = threadIdx.x / side; k < m; k += kTinyThreads / side) {
            if ((used[k >> 5] >> (k & 31)) & 1u) continue;
            float* row = z.data + (r + k) * z.stride;
            for (int c = lane; c < units; c += side) {
                if (wide) reinterpret_cast<float4*>(row)[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                else row[c] = 0.0f;
            }
        }
        __syncthreads();
    }
}

__device__ __forceinline__ int first_above(const int2* items, int n, int key) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (items[mid].x <= key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <typename T, int VB>
__global__ void __launch_bounds__(kTinyThreads) k_table_gradient_tiny(const T* __restrict__ grads, int stride, int dim,
                                                                      const SegmentPlan pl, const Segments g,
                                                                      const KeySource src, const ZeroRows zero,
                                                                      int bits) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int2 items[kTinyRows];
    __shared__ uint16_t wcount[kTinyThreads / 32][256];
    __shared__ int start[256], sm[33];
    __shared__ uint32_t used[kZeroRows / 32];
    const int count = sort_rows<kTinyThreads, kTinyRows / kTinyThreads>(src, bits, items, wcount, start, sm);
    const int64_t b = blockIdx.x, blocks = gridDim.x;
    if (zero.data && blockIdx.y == 0)
        zero_unused(zero, items, count, b * zero.rows / blocks, (b + 1) * zero.rows / blocks, used);
    int p0 = (int)(b * count / blocks), p1 = (int)((b + 1) * count / blocks);
    if (p0 > 0) p0 = first_above(items, count, items[p0 - 1].x);
    if (p1 > 0) p1 = first_above(items, count, items[p1 - 1].x);
    if (p1 <= p0) return;
    sum_chunk<T, VB>(grads, stride, dim, pl, (p1 - p0 + pl.slots - 1) / pl.slots, g, items + p0, p1 - p0,
                     reinterpret_cast<float*>(smem), false, false, nullptr);
}

// A warp per chunk for the runs of up to 32 partial sums behind the first (nearly all: an average run is
// shorter than a chunk), 32 columns each; the whole block for a longer one, of which at most one starts in
// a block's chunks (the chunks that it covers own none), its warps 32 partial sums apart.
constexpr int kJoinWarps = 32;

__global__ void __launch_bounds__(32 * kJoinWarps) k_table_join(int dim, int nchunks, const Segments g) {
    __shared__ int long_run[2];  // its first chunk, its key
    __shared__ float part[kJoinWarps][32];
    after_predecessor();
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = blockIdx.x * kJoinWarps + w, col = blockIdx.y * 32 + lane;
    const bool on = col < dim;
    const int k = b < nchunks ? g.owned[b] : -1;
    const int next = b + 1 + lane;
    const unsigned same = __ballot_sync(0xffffffffu, k >= 0 && next < nchunks && g.first_key[next] == k);
    if (threadIdx.x == 0) long_run[0] = -1;
    __syncthreads();
    if (same == 0xffffffffu) {
        if (lane == 0) long_run[0] = b, long_run[1] = k;
    } else if (k >= 0 && on) {
        const int more = __ffs(~same) - 1;
        float s = g.partial[((int64_t)b * 2 + 1) * dim + col];
#pragma unroll 4
        for (int c = 1; c <= more; ++c) s += g.partial[(int64_t)(b + c) * 2 * dim + col];
        const float one[1] = {s};
        store_row<1>(g, k, col, one);
    }
    __syncthreads();
    const int lb = long_run[0], lk = long_run[1];
    if (lb < 0) return;
    int end = lb + 1;  // the run's last chunk is end - 1
    for (int more = 32 * kJoinWarps; more == 32 * kJoinWarps; end += more) {
        const int c = end + threadIdx.x;
        more = __syncthreads_count(c < nchunks && g.first_key[c] == lk);
    }
    float s = 0.0f;
    if (on) {
        if (w == 0) s = g.partial[((int64_t)lb * 2 + 1) * dim + col];
#pragma unroll 8
        for (int c = lb + 1 + w; c < end; c += kJoinWarps) s += g.partial[(int64_t)c * 2 * dim + col];
    }
    part[w][lane] = s;
    __syncthreads();
    if (w == 0 && on) {
#pragma unroll 8
        for (int t = 1; t < kJoinWarps; ++t) s += part[t][lane];
        const float one[1] = {s};
        store_row<1>(g, lk, col, one);
    }
}

struct GradLayout {
    size_t first_keys, items[2], hist, totals, valid, first_key, owned, partial, total;
    int ntiles, passes, bits, chunks_max;
};

// Rows a slot adds: enough blocks for few rows, few borders for many (500K x 27 bf16 of which 300K take part,
// 32 / 48 / 94 rows: 34.8 / 32.2 / 37.1 us a call), and more for many or long rows, of which a block has few
// slots, so that at most some 16 chunks an SM are left to join (1.2M x 119 bf16, 52 rows of which few are much
// used: 198 us in all with 48 rows a slot and a join of 256 columns a block, 67 so). 3M x 48 fp32 hardly
// depends on it: 61 rows by that rule 194.8 us a call, with 32 / 48 / 96 rows 194.0 / 192.1 / 193.4.
constexpr int kMinRun = 4, kMaxRun = 48, kMaxChunk = 2048;

// Bytes of a row that a thread reads at once: 16 where the rows allow it, else 8, 4 or an element.
template <typename T>
int unit_bytes(const gs3d_rows* r) {
    for (int b = 16; b > (int)sizeof(T); b /= 2)
        if (packs<T>(r, b / (int)sizeof(T))) return b;
    return (int)sizeof(T);
}

template <typename T, typename F>
int dispatch_unit(int bytes, F&& f) {
    switch (bytes) {
        case 16: return f(std::integral_constant<int, 16>{});
        case 8: return f(std::integral_constant<int, 8>{});
        case 4: return f(std::integral_constant<int, 4>{});
        default: return f(std::integral_constant<int, (int)sizeof(T)>{});
    }
}

int slots_for(int tile_units) { return std::max(1, std::min(32, 256 / tile_units)); }

SegmentPlan segment_plan(int64_t n, int units) {
    SegmentPlan p;
    p.units = units;
    p.tile_units = std::min(units, 256);
    p.slots = slots_for(p.tile_units);
    const int64_t want = ceil_div(n, (int64_t)p.slots * kSMs * 4), most = ceil_div(n, (int64_t)p.slots * kSMs * 16);
    const int64_t run = std::max(most, std::max<int64_t>(kMinRun, std::min<int64_t>(kMaxRun, want)));
    p.run = (int)std::min<int64_t>(run, kMaxChunk / p.slots);
    p.chunk = p.slots * p.run;
    p.nchunks = (int)std::max<int64_t>(1, ceil_div(n, p.chunk));
    return p;
}

// Rows a thread of the sort's tiles takes: small tiles for few rows, so that all SMs have some (300K rows into
// 60,000 of the table, 2 / 4 / 8 rows: 41 / 43 / 51 us in all; 450K: - / 49 / 56).
int sort_rounds(int64_t n) {
    return n <= 2 * kSMs * 2 * kSortThreads ? 2 : (n <= 2 * kSMs * 4 * kSortThreads ? 4 : 8);
}

// The most tiles that n rows or fewer are cut into.
int most_tiles(int64_t n) {
    int64_t most = 0;
    for (int rounds = 2; rounds <= 8; rounds *= 2) {
        const int64_t last = rounds < 8 ? std::min<int64_t>(n, 2 * kSMs * rounds * kSortThreads) : n;
        most = std::max(most, ceil_div(last, rounds * kSortThreads));
    }
    return (int)most;
}

template <typename F>
int dispatch_rounds(int rounds, F&& f) {
    switch (rounds) {
        case 2: return f(std::integral_constant<int, 2>{});
        case 4: return f(std::integral_constant<int, 4>{});
        default: return f(std::integral_constant<int, 8>{});
    }
}

// The most chunks that n rows or fewer are cut into.
int most_chunks(int64_t n, int units) {
    const int64_t s = slots_for(std::min(units, 256));
    const int64_t few = std::max<int64_t>(kSMs * 4, ceil_div(n, s * kMaxRun));
    return (int)std::max(std::min({ceil_div(n, s * kMinRun), few, (int64_t)kSMs * 16}), ceil_div(n, s * (kMaxChunk / s)));
}

int bits_of(int64_t v) {
    int b = 0;
    while (v >> b) ++b;
    return b;
}

GradLayout grad_layout(int64_t n, int64_t rows, int dim) {
    GradLayout L;
    L.ntiles = (int)ceil_div(n, sort_rounds(n) * kSortThreads);
    L.bits = bits_of(std::max<int64_t>(rows, 1) - 1);
    L.passes = std::max(1, (L.bits + kMaxDigitBits - 1) / kMaxDigitBits);
    const int digit = (L.bits + L.passes - 1) / L.passes;
    // the launch picks its unit from the gradients' alignment, and fewer rows other tiles and chunks: room for all
    L.chunks_max = 1;
    for (int units = dim; units >= 1; units = units % 2 == 0 ? units / 2 : 0)
        L.chunks_max = std::max(L.chunks_max, most_chunks(n, units));
    size_t off = 0;
    L.first_keys = off; off += align256((size_t)n * 4);
    for (int i = 0; i < 2; ++i) {
        L.items[i] = off; off += i == 0 || L.bits > 8 ? align256((size_t)n * 8) : 0;
    }
    L.hist = off; off += align256((size_t)most_tiles(n) * ((size_t)1 << digit) * 4);
    L.totals = off; off += align256(((size_t)1 << kMaxDigitBits) * 4);
    L.valid = off; off += 256;
    L.first_key = off; off += align256((size_t)L.chunks_max * 4);
    L.owned = off; off += align256((size_t)L.chunks_max * 4);
    L.partial = off; off += align256((size_t)L.chunks_max * 2 * dim * 4);
    L.total = off;
    return L;
}

}  // namespace
}  // namespace gs3d

using namespace gs3d;

extern "C" {

GS3D_API int gs3d_table_lookup(const gs3d_rows* table, const int32_t* indices, float scale, const gs3d_rows* out,
                               gs3d_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    GS3D_RETURN_IF(check_rows(table, "table"));
    GS3D_RETURN_IF(check_rows(out, "lookup output"));
    if (table->dim != out->dim) return invalid("table dim %d, output dim %d", table->dim, out->dim);
    if (out->rows == 0) return GS3D_OK;
    if (!indices) return invalid("NULL indices");
    GS3D_RETURN_IF(check_words(indices, "indices"));
    ProfScope prof("table_lookup", stream);
    return dispatch_type(table->type, [&](auto ti) {
        using TI = typename decltype(ti)::T;
        return dispatch_type(out->type, [&](auto to) {
            using TO = typename decltype(to)::T;
            return launch_lookup<TI, TO>(table, indices, scale, out, stream);
        });
    });
}

GS3D_API int gs3d_table_gradient_workspace_size(int64_t grad_rows, int64_t table_rows, int32_t dim, size_t* bytes) {
    if (!bytes) return invalid("bytes is NULL");
    if (grad_rows < 0 || grad_rows > kMaxRows || table_rows < 0 || table_rows > kMaxRows || dim < 1 ||
        dim > kMaxRowDim)
        return invalid("%lld rows, table of %lld rows, dim %d", (long long)grad_rows, (long long)table_rows, dim);
    *bytes = grad_rows <= kTinyRows ? 0 : grad_layout(grad_rows, table_rows, dim).total;
    return GS3D_OK;
}

GS3D_API int gs3d_table_gradient(const gs3d_rows* grads, const int32_t* indices, int64_t n_indices,
                                 const int32_t* fgidx_to_gidx, const int32_t* device_counts, float scale,
                                 const gs3d_rows* table_grads, uint32_t flags, void* workspace,
                                 size_t workspace_bytes, gs3d_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    GS3D_RETURN_IF(check_rows(grads, "gradients"));
    GS3D_RETURN_IF(check_rows(table_grads, "table gradients"));
    if (grads->dim != table_grads->dim)
        return invalid("gradient dim %d, table dim %d", grads->dim, table_grads->dim);
    if (table_grads->type != GS3D_F32) return invalid("table gradients are GS3D_F32");
    if (flags & ~GS3D_TABLE_ACCUMULATE) return invalid("flags %u", flags);
    if (n_indices < 0 || (!fgidx_to_gidx && n_indices < grads->rows))
        return invalid("%lld indices for %lld rows", (long long)n_indices, (long long)grads->rows);
    if (grads->rows > 0 && !indices && n_indices > 0) return invalid("NULL indices");
    GS3D_RETURN_IF(check_words(indices, "indices"));
    GS3D_RETURN_IF(check_words(fgidx_to_gidx, "fgidx_to_gidx"));
    GS3D_RETURN_IF(check_words(device_counts, "device_counts"));
    if (table_grads->rows == 0) return GS3D_OK;
    const int64_t n = grads->rows;
    const bool tiny = n <= kTinyRows;
    const GradLayout L = grad_layout(std::max<int64_t>(n, 1), table_grads->rows, grads->dim);
    if (!tiny && (!workspace || workspace_bytes < L.total))
        return set_error("table gradient workspace %zu bytes < %zu", workspace_bytes, L.total), GS3D_ERR_WORKSPACE;
    if (!tiny && (reinterpret_cast<uintptr_t>(workspace) & 255)) return invalid("workspace not 256-byte aligned");
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    const auto at = [&](size_t off) { return reinterpret_cast<int32_t*>(ws + off); };
    const auto items = [&](int i) { return reinterpret_cast<int2*>(ws + L.items[i]); };
    const bool accumulate = (flags & GS3D_TABLE_ACCUMULATE) != 0;
    float* out = static_cast<float*>(table_grads->data);
    const KeySource src{indices, fgidx_to_gidx, device_counts, n_indices, (int32_t)n, (int32_t)table_grads->rows};
    const ZeroRows zero{accumulate ? nullptr : out, table_grads->row_stride, (int32_t)table_grads->rows,
                        table_grads->dim};
    if (n == 0 && accumulate) return GS3D_OK;
    ProfScope prof("table_grad", stream);
    if (tiny)
        return dispatch_type(grads->type, [&](auto t) {
            using T = typename decltype(t)::T;
            const T* g = static_cast<const T*>(grads->data);
            const int bytes = unit_bytes<T>(grads), per = bytes / (int)sizeof(T);
            const SegmentPlan pl = segment_plan(n, grads->dim / per);
            const Segments seg{nullptr, nullptr, out, table_grads->row_stride, scale, accumulate ? 1 : 0, nullptr,
                               nullptr, nullptr};
            const size_t smem = (size_t)pl.slots * pl.tile_units * per * 4;
            // a block for 32 rows, or for 64 KB of table to zero up to one an SM and for 1 MB up to four (60,000 rows of
            // 48: 10.9 us by 148 blocks, 12.9 by 176)
            const int64_t zeroed = accumulate ? 0 : table_grads->rows * table_grads->dim;
            const int blocks = (int)std::max({ceil_div(n, 32), std::min<int64_t>(ceil_div(zeroed, 1 << 14), kSMs),
                                              std::min<int64_t>(ceil_div(zeroed, 1 << 18), 4 * kSMs)});
            const dim3 grid(blocks, (unsigned)ceil_div(pl.units, pl.tile_units));
            return dispatch_unit<T>(bytes, [&](auto vb) {
                k_table_gradient_tiny<T, decltype(vb)::value><<<grid, kTinyThreads, smem, stream>>>(
                    g, (int)grads->row_stride, grads->dim, pl, seg, src, zero, L.bits);
                GS3D_LAUNCHED("k_table_gradient_tiny");
                return GS3D_OK;
            });
        });
    int sorted = 0;
    if (n <= kClusterRows) {
        const int64_t words = accumulate ? 0 : table_grads->rows * table_grads->dim;
        const int fillers = (int)std::min<int64_t>(ceil_div(words, kClusterCtas * kClusterThreads * 8), kSMs / 4);
        const dim3 grid((unsigned)(kClusterCtas * (1 + fillers)));
        const auto kernel = n <= kClusterRows / 2 ? k_sort_cluster<1> : k_sort_cluster<2>;
        kernel<<<grid, kClusterThreads, 0, stream>>>(src, zero, L.bits, items(0), items(1), at(L.valid));
        GS3D_LAUNCHED("k_sort_cluster");
        sorted = (std::max(L.bits, 1) - 1) / 8 & 1;
    } else {
        SortPass p{at(L.first_keys), nullptr, nullptr, at(L.hist), at(L.totals), at(L.valid), (int32_t)n, L.ntiles, 0, 0};
        const int digit = (L.bits + L.passes - 1) / L.passes;
        GS3D_RETURN_IF(dispatch_rounds(sort_rounds(n), [&](auto rounds) {
            constexpr int R = decltype(rounds)::value;
            const size_t smem = radix_scatter_smem(R, digit);
            if (smem > (48u << 10))
                GS3D_CUDA(cudaFuncSetAttribute(k_radix_scatter<R>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)radix_scatter_smem(R, kMaxDigitBits)),
                          "scatter smem attribute");
            // few tiles leave SMs that zero the table: a block for 16 KB of it
            const int64_t zeroed = accumulate ? 0 : table_grads->rows * table_grads->dim;
            const int fillers = (int)std::min<int64_t>(ceil_div(zeroed, 1 << 12), std::max(0, 4 * kSMs - L.ntiles));
            for (int i = 0; i < L.passes; ++i) {
                p.shift = i * digit;
                p.bits = digit;
                p.out = items(i & 1);
                if (i == 0) {  // behind whatever wrote the inputs
                    k_radix_count<R><<<L.ntiles + fillers, kSortThreads, 0, stream>>>(p, src, zero);
                    GS3D_LAUNCHED("k_radix_count");
                } else {
                    GS3D_RETURN_IF(launch_after("k_radix_count", k_radix_count<R>, dim3(L.ntiles), kSortThreads, 0,
                                                stream, p, src, zero));
                }
                GS3D_RETURN_IF(
                    launch_after("k_radix_spine", k_radix_spine, dim3(1 << digit), kSpineThreads, 0, stream, p));
                GS3D_RETURN_IF(launch_after("k_radix_scatter", k_radix_scatter<R>, dim3(L.ntiles), kSortThreads, smem,
                                            stream, p));
                p.in = p.out;
                sorted = i & 1;
            }
            return GS3D_OK;
        }));
    }
    const Segments seg{items(sorted), at(L.valid), out, table_grads->row_stride, scale,
                       accumulate ? 1 : 0, at(L.first_key), at(L.owned), reinterpret_cast<float*>(ws + L.partial)};
    return dispatch_type(grads->type, [&](auto t) {
        using T = typename decltype(t)::T;
        const T* g = static_cast<const T*>(grads->data);
        const int bytes = unit_bytes<T>(grads), per = bytes / (int)sizeof(T);
        const SegmentPlan pl = segment_plan(n, grads->dim / per);
        const size_t smem = (size_t)pl.chunk * 8 + (size_t)pl.slots * pl.tile_units * per * 4;
        const dim3 grid(pl.nchunks, (unsigned)ceil_div(pl.units, pl.tile_units));
        const int threads = pl.slots * pl.tile_units;
        const int stride = (int)grads->row_stride;
        GS3D_RETURN_IF(dispatch_unit<T>(bytes, [&](auto vb) {
            return launch_after("k_table_segments", k_table_segments<T, decltype(vb)::value>, grid, threads, smem, stream, g,
                                stride, grads->dim, pl, seg);
        }));
        GS3D_RETURN_IF(launch_after("k_table_join", k_table_join,
                                    dim3((unsigned)ceil_div(pl.nchunks, kJoinWarps), (unsigned)ceil_div(grads->dim, 32)),
                                    32 * kJoinWarps, 0, stream, (int)grads->dim, pl.nchunks, seg));
        return GS3D_OK;
    });
}

}  // extern "C"
