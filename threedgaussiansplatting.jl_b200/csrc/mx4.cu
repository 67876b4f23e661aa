// mx4.cu — microscaled 4-bit rows: quantisation, dequantisation, and the colours of Gaussians whose
// SH coefficients are held in them.
//   gs3d_mx4_tensor_scale   largest magnitude of all rows -> NVFP4 tensor scale
//   gs3d_mx4_quantise       rows -> e2m1 codes and block scales
//   gs3d_mx4_dequantise     and back
//   gs3d_mx4_colours        product of the 4-bit blocks with the SH basis of a view direction
//
// Rounding. An element is the exact quotient q = |x| / (s g) (s block scale, g tensor scale, 1 for
// MXFP4) rounded to the e2m1 grid.
//   MXFP4: s is a power of two, so x (1 / s) is exact and one conversion decides.
//   NVFP4: x (1 / (s g)) is not exact. Products with the reciprocal moved down and up by 2^-21 (more
//     than the errors of s g, its reciprocal and the product) enclose q, and rounding is monotone: where
//     both convert to the same code, q does. Else one border b lies between them, and q is held against it:
//     q passes b iff |x| > b s g (>= where the tie goes up). b s is exact in fp32 (at most 7 significant
//     bits); b s g is not, but no fp32 lies between it and its neighbours RD(b s g) <= b s g <= RU(b s g),
//     so |x| > b s g iff |x| > RD(b s g) and |x| >= b s g iff |x| >= RU(b s g): exact with one directed
//     product. Such borders are common where x has few bits: of 16-bit x and its own tensor scale, q is a
//     ratio of small numbers. The block scale is decided in the same way.
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "mx4.cuh"
#include "mx4_colour.cuh"
#include "rows.cuh"

namespace gs3d {
namespace {

// Rows that consist of packs of BYTES bytes.
template <typename T, int BYTES>
bool packs_of(const gs3d_rows* r) {
    constexpr int n = BYTES / (int)sizeof(T);
    return r->dim % n == 0 && r->row_stride % n == 0 && reinterpret_cast<uintptr_t>(r->data) % BYTES == 0;
}

int grid_for(int64_t items, int threads, int per_sm) {
    const int64_t b = std::min<int64_t>(ceil_div(items, threads), (int64_t)device_sm_count() * per_sm);
    return (int)std::max<int64_t>(b, 1);
}

template <typename T, int N>
struct alignas(N * sizeof(T)) Pack {
    T e[N];
};

// Quotients of numbers below 2^31 by a divisor that the host knows (Granlund and Montgomery 1994).
struct FastDiv {
    uint32_t d, m;
    int s;
    explicit FastDiv(uint32_t divisor) : d(divisor), s(0) {
        while (((uint64_t)1 << s) < d) ++s;
        m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << s) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};

// ---- tensor scale ----------------------------------------------------------------------------
__device__ __forceinline__ void take_finite_abs(uint32_t& m, float v) {
    const uint32_t b = f2u(v) & 0x7fffffffu;  // magnitudes order like unsigned integers
    if (b < 0x7f800000u) m = max(m, b);
}

// The largest magnitude among packs, NaN left out: a word of it for each word of the packs.
__device__ __forceinline__ float abs_max(float m, float v) { return fmaxf(m, fabsf(v)); }
__device__ __forceinline__ __half2 abs_max(__half2 m, __half2 v) { return __hmax2(m, __habs2(v)); }
__device__ __forceinline__ __nv_bfloat162 abs_max(__nv_bfloat162 m, __nv_bfloat162 v) { return __hmax2(m, __habs2(v)); }
__device__ __forceinline__ float larger(float m) { return m; }
__device__ __forceinline__ float larger(__half2 m) { return fmaxf(__low2float(m), __high2float(m)); }
__device__ __forceinline__ float larger(__nv_bfloat162 m) { return fmaxf(__low2float(m), __high2float(m)); }
template <typename T>
using Word = typename std::conditional<
    sizeof(T) == 4, float,
    typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type>::type;

// Every block turns its largest magnitude into the scale it asks for (monotone, positive: fp32 bits
// order like unsigned integers) and the largest one stays; a lone block stores it. A maximum does not
// depend on the order, so the atomics give equal bits.
// WIDE: rows of 16-byte packs, back to back, eight loads a thread in flight, of 16-bit elements two a
// comparison. Bound by reading x: 3M x 48 fp32 95 us (6.0 TB/s), 1.5M x 48 bf16 29 (39 with the elements one by
// one in fp32). All but the last 96 MB are read as data that L2 need not keep, so that what k_mx4_quantise_blocks
// begins with is there: with its own loads so marked too the two and the dequantisation behind them take
// 281 us at 3M x 48 fp32, 298 with plain loads.
// Else an element at a time, with a division for its row: 1M x 48 fp32 in rows 64 apart 186 us (33 back to back).
constexpr int64_t kScaleKept = (int64_t)96 << 20;
constexpr int kScaleThreads = 512;

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kScaleThreads) k_mx4_tensor_scale(const T* __restrict__ x, int64_t rows,
                                                                    int64_t stride, int dim,
                                                                    uint32_t* __restrict__ tensor_scale) {
    constexpr int N = 16 / (int)sizeof(T);
    __shared__ uint32_t warp_max[kScaleThreads / 32];
    uint32_t m = 0;
    const int64_t total = rows * dim, threads = (int64_t)gridDim.x * blockDim.x;
    const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (WIDE) {
        using W = Word<T>;
        const int64_t packs = total / N;
        const uint4* p = reinterpret_cast<const uint4*>(x);
        W top{};
        constexpr int AHEAD = 8;
        const int64_t streamed = packs - max(kScaleKept / 16, AHEAD * threads);
        const auto batch = [&](int64_t i, auto full) {
            uint4 v[AHEAD];
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                v[q] = make_uint4(0u, 0u, 0u, 0u);
                if (i < streamed) v[q] = __ldcs(p + i + q * threads);
                else if (full || i + q * threads < packs) v[q] = __ldg(p + i + q * threads);
            }
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                top = abs_max(top, *reinterpret_cast<const W*>(&v[q].x));
                top = abs_max(top, *reinterpret_cast<const W*>(&v[q].y));
                top = abs_max(top, *reinterpret_cast<const W*>(&v[q].z));
                top = abs_max(top, *reinterpret_cast<const W*>(&v[q].w));
            }
        };
        int64_t i = t;
        for (; i + (AHEAD - 1) * threads < packs; i += AHEAD * threads) batch(i, std::true_type{});
        if (i < packs) batch(i, std::false_type{});
        const float a = larger(top);
        if (f2u(a) < 0x7f800000u) {
            m = f2u(a);
        } else {  // infinities do not count: once more without them
            for (int64_t i = t; i < packs; i += threads) {
                const Pack<T, N> v = reinterpret_cast<const Pack<T, N>*>(x)[i];
#pragma unroll
                for (int c = 0; c < N; ++c) take_finite_abs(m, to_f32(v.e[c]));
            }
        }
        const int64_t tail = total / N * N + t;
        if (tail < total) take_finite_abs(m, to_f32(x[tail]));
    } else {
        for (int64_t i = t; i < total; i += threads) {
            const int64_t r = i / dim;
            take_finite_abs(m, to_f32(x[r * stride + (i - r * dim)]));
        }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kScaleThreads / 32; ++w) m = max(m, warp_max[w]);
        const uint32_t scale = f2u(fmaxf(u2f(m) * (1.0f / 2688.0f), 0x1p-100f));
        if (gridDim.x == 1) *tensor_scale = scale;
        else atomicMax(tensor_scale, scale);
    }
}

// ---- quantise --------------------------------------------------------------------------------
// a / (6 g) to the nearest e4m3 value, ties to even, at most 448 (0x7e): an estimate (within a step),
// corrected against the exact borders around it.
__device__ __noinline__ uint32_t nvfp4_scale_byte_exact(float a, float g, float inv6g) {
    const float est = fminf(a * inv6g, 448.0f);
    uint32_t u = __nv_cvt_float_to_fp8(est, __NV_SATFINITE, __NV_E4M3) & 0x7fu;
    const float v = e4m3_value(u);
    if (u < 0x7eu) {
        const float border = 3.0f * (v + e4m3_value(u + 1));  // 6 x midpoint, exact
        if ((u & 1u) ? a >= __fmul_ru(border, g) : a > __fmul_rd(border, g)) return u + 1;
    }
    if (u > 0) {
        const float border = 3.0f * (v + e4m3_value(u - 1));
        if ((u & 1u) ? a <= __fmul_rd(border, g) : a < __fmul_ru(border, g)) return u - 1;
    }
    return u;
}

// The same: enclosed, where both ends convert to the same value (0x7f for a NaN).
__device__ __forceinline__ uint32_t nvfp4_scale_byte(float a, float g, float inv6g) {
    const uint32_t both = __nv_cvt_float2_to_fp8x2(
        make_float2(a * (inv6g * (1.0f - 0x1p-21f)), a * (inv6g * (1.0f + 0x1p-21f))), __NV_SATFINITE, __NV_E4M3);
    const uint32_t lo = both & 0xffu;
    return lo == both >> 8 ? lo : nvfp4_scale_byte_exact(a, g, inv6g);
}

// 2^(floor(log2 a) - 2) as its e8m0 byte.
__device__ __forceinline__ uint32_t mxfp4_scale_byte(float a) { return (uint32_t)max((int)(f2u(a) >> 23) - 2, 0); }

// The codes of eight elements, each x[k] * f rounded to the grid (ties to even, magnitudes above 6 to 6).
__device__ __forceinline__ uint32_t e2m1_word(const float* x, float f) {
    uint32_t w;
    asm("{ .reg .b8 a, b, c, d;\n"
        "  cvt.rn.satfinite.e2m1x2.f32 a, %2, %1; cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        "  cvt.rn.satfinite.e2m1x2.f32 c, %6, %5; cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        "  mov.b32 %0, {a, b, c, d}; }"
        : "=r"(w)
        : "f"(x[0] * f), "f"(x[1] * f), "f"(x[2] * f), "f"(x[3] * f), "f"(x[4] * f), "f"(x[5] * f), "f"(x[6] * f),
          "f"(x[7] * f));
    return w;
}

// Whether a magnitude lies beyond the border between codes c and c + 1, ties to the even code.
__device__ __forceinline__ bool beyond_border(float a, uint32_t c, float s, float g) {
    const float2 e = __half22float2(e2m1_pair_half(c | (c + 1) << 4));
    const float bs = (e.x + e.y) * 0x1p13f * s;  // border * s, exact
    return (c & 1u) ? a >= __fmul_ru(bs, g) : a > __fmul_rd(bs, g);
}

// 1 / v within one unit in the last place, for v and 1 / v within the normal numbers.
__device__ __forceinline__ float reciprocal(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// The larger magnitude, NaN if one is.
__device__ __forceinline__ float max_abs(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}

struct TensorScale {
    float g, inv6g;
    template <int FMT>
    static __device__ __forceinline__ TensorScale load(const float* p) {
        TensorScale t{1.0f, 0.0f};
        if (FMT == GS3D_NVFP4) {
            t.g = __ldg(p);
            t.inv6g = reciprocal(6.0f * t.g);
        }
        return t;
    }
};

// A block's scale byte and the codes of its first EL elements v (zeros behind the row's end), two a byte,
// in words of eight. EL < block size: rows of at most EL elements.
template <int FMT, int EL>
__device__ __forceinline__ uint32_t quantise_block(const float (&v)[EL], const TensorScale& t,
                                                   uint32_t (&words)[EL / 8]) {
    float a = fabsf(v[0]);
#pragma unroll
    for (int k = 1; k < EL; ++k) a = max_abs(a, v[k]);
    const bool nan = a != a;
    if (FMT == GS3D_MXFP4) {
        const uint32_t byte = mxfp4_scale_byte(a);
        const float inv = u2f((254u - byte) << 23);  // 2^(127 - byte), byte <= 253
#pragma unroll
        for (int w = 0; w < EL / 8; ++w) words[w] = e2m1_word(v + 8 * w, inv);
        return nan ? 0xffu : byte;
    }
    const uint32_t byte = nvfp4_scale_byte(a, t.g, t.inv6g);
    const float s = e4m3_value(byte);
    const float inv = s > 0.0f ? reciprocal(s * t.g) : 0.0f;
    const float lo = inv * (1.0f - 0x1p-21f), hi = inv * (1.0f + 0x1p-21f);
    uint32_t differ = 0, upper[EL / 8];
#pragma unroll
    for (int w = 0; w < EL / 8; ++w) {
        words[w] = e2m1_word(v + 8 * w, lo);
        upper[w] = e2m1_word(v + 8 * w, hi) ^ words[w];
        differ |= upper[w];
    }
    if (differ)
#pragma unroll
        for (int k = 0; k < EL; ++k) {
            const uint32_t d = (upper[k / 8] >> (4 * (k % 8))) & 15u, c = (words[k / 8] >> (4 * (k % 8))) & 7u;
            if (d && beyond_border(fabsf(v[k]), c, s, t.g)) words[k / 8] ^= d << (4 * (k % 8));
        }
    return nan ? 0x7fu : byte;
}

// Rows in packs of N elements (16 bytes, or four): a block a thread, whose elements, scale and codes stay
// in its registers; from the last row to the first, so that what a tensor-scale pass just before has left
// in L2 is read from there. Bound by memory with fp32 (3M x 48 in NVFP4 87 us behind that pass; 657 MB, 100 us
// at the rate of a plain copy; 2.6M x 48 in MXFP4, whose last block is half, 98 us, through shared memory
// 339), by the instructions with 16-bit elements in NVFP4 (1.5M x 48 bf16 40 us, 26 for the bytes; 78 with all
// elements of a block held against all borders where one might lie between two codes). The tensor scale
// is known before x is read again: one kernel for both would need all of x on the chip.
// WHOLE: rows of whole blocks, the codes stored a block at a time; else in words, or in halves of them.
template <typename T, int FMT, int EL, int N, bool WHOLE>
__global__ void __launch_bounds__(256)
    k_mx4_quantise_blocks(const T* __restrict__ x, int64_t blocks, int64_t stride, int dim, const FastDiv nb, bool flat,
                          uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                          const float* __restrict__ tensor_scale) {
    constexpr int BS = Mx4Block<FMT>::size;
    const int64_t i = (int64_t)(gridDim.x - 1 - blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= blocks) return;
    const TensorScale t = TensorScale::load<FMT>(tensor_scale);
    const T* xb = x + i * BS;
    int64_t r = 0;
    int b = 0, len = BS;
    if (!WHOLE || !flat) {
        r = i < INT_MAX ? (int64_t)nb.quotient((uint32_t)i) : i / nb.d;
        b = (int)(i - r * nb.d);
        xb = x + r * stride + b * BS;
        if (!WHOLE) len = min(BS, dim - b * BS);
    }
    float v[EL];
#pragma unroll
    for (int k = 0; k < EL; k += N) {
        Pack<T, N> p{};
        if (WHOLE || k < len) {
            using W = typename std::conditional<sizeof(p) == 16, uint4, uint2>::type;
            const W w = __ldcs(reinterpret_cast<const W*>(xb + k));
            p = *reinterpret_cast<const Pack<T, N>*>(&w);
        }
#pragma unroll
        for (int c = 0; c < N; ++c) v[k + c] = to_f32(p.e[c]);
    }
    uint32_t words[EL / 8];
    scales[i] = (uint8_t)quantise_block<FMT>(v, t, words);
    if constexpr (WHOLE) {
        Pack<uint32_t, BS / 8> o;
#pragma unroll
        for (int w = 0; w < BS / 8; ++w) o.e[w] = words[w];
        *reinterpret_cast<Pack<uint32_t, BS / 8>*>(codes + i * (BS / 2)) = o;
    } else {
        uint8_t* c = codes + r * (dim / 2) + b * (BS / 2);
        if (dim % 8 == 0) {
#pragma unroll
            for (int w = 0; w < EL / 8; ++w)
                if (8 * w < len) reinterpret_cast<uint32_t*>(c)[w] = words[w];
        } else {  // 4 more than a multiple of 8
#pragma unroll
            for (int h = 0; h < EL / 4; ++h)
                if (4 * h < len) reinterpret_cast<uint16_t*>(c)[h] = (uint16_t)(words[h / 2] >> (16 * (h & 1)));
        }
    }
}

// Rows of any length (they may end inside a block): a CTA takes `per` (a power of two) rows, which lie back
// to back, as one range of bytes through shared memory (asynchronous copies: 2.1M x 27 fp32 in MXFP4 49 us, 82
// with a load and a store a turn), and hands the codes back the same way. The threads of a warp take one
// block of neighbouring rows, so that what they read lies an odd number of elements or pairs apart (rows
// of four-element packs do not come here) and meets few bank conflicts. 500K x 27 bf16 10.5 us (5.4 for the
// bytes): a CTA reads, computes and writes in turn. Reading the elements as shifted 32-bit words was slower.
// Most rows a CTA: short ones want many (2.9M x 3 fp16, 128 / 256 / 512 rows: 24 / 18 / 15.5 us; more were
// not tried).
constexpr int kRowsThreads = 128, kRowsMost = 512;

template <typename T, int FMT, int EL>
__global__ void __launch_bounds__(kRowsThreads)
    k_mx4_quantise_rows(const T* __restrict__ x, int64_t rows, int dim, int log_per, uint8_t* __restrict__ codes,
                        uint8_t* __restrict__ scales, const float* __restrict__ tensor_scale) {
    constexpr int BS = Mx4Block<FMT>::size;
    extern __shared__ __align__(16) unsigned char smem[];
    const int nb = (dim + BS - 1) / BS, cb = (dim + 1) / 2, per = 1 << log_per;
    const int64_t r0 = (int64_t)blockIdx.x << log_per;
    const int mine = (int)min((int64_t)per, rows - r0);
    const unsigned char* gx = reinterpret_cast<const unsigned char*>(x + r0 * dim);
    uint8_t* gc = codes + r0 * cb;
    unsigned char* sc = smem + ((16 + (size_t)per * dim * sizeof(T) + 15) & ~(size_t)15) + head_of(gc);
    copy_in(smem, gx, mine * dim * (int)sizeof(T));
    __syncthreads();
    const T* sx = reinterpret_cast<const T*>(smem + head_of(gx));
    const TensorScale t = TensorScale::load<FMT>(tensor_scale);
    for (int i = threadIdx.x; i < nb << log_per; i += kRowsThreads) {
        const int r = i & (per - 1), b = i >> log_per;
        if (r >= mine) continue;
        const int len = min(BS, dim - b * BS);
        float v[EL];
#pragma unroll
        for (int k = 0; k < EL; ++k) v[k] = k < len ? to_f32(sx[r * dim + b * BS + k]) : 0.0f;
        uint32_t words[EL / 8];
        scales[(r0 + r) * nb + b] = (uint8_t)quantise_block<FMT>(v, t, words);
        unsigned char* o = sc + r * cb + b * (BS / 2);
#pragma unroll
        for (int k = 0; k < EL / 2; ++k)
            if (2 * k < len) o[k] = (unsigned char)(words[k / 4] >> (8 * (k % 4)));
    }
    __syncthreads();
    copy_out(gc, sc - head_of(gc), mine * cb);
}

// Rows apart and not of packs, or long: a block a thread, element by element (1M x 48 fp32 in rows 49 apart 60
// us, back to back by packs 34).
template <typename T, int FMT>
__global__ void __launch_bounds__(256) k_mx4_quantise(const T* __restrict__ x, int64_t rows, int64_t stride,
                                                      int dim, uint8_t* __restrict__ codes,
                                                      uint8_t* __restrict__ scales,
                                                      const float* __restrict__ tensor_scale) {
    constexpr int BS = Mx4Block<FMT>::size;
    const int nb = (dim + BS - 1) / BS, cb = (dim + 1) / 2;
    const TensorScale t = TensorScale::load<FMT>(tensor_scale);
    const int64_t total = rows * nb;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
         i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / nb;
        const int b = (int)(i - r * nb);
        const int len = min(BS, dim - b * BS);
        const T* xr = x + r * stride + b * BS;
        float v[BS];
#pragma unroll
        for (int k = 0; k < BS; ++k) v[k] = k < len ? to_f32(xr[k]) : 0.0f;
        uint32_t words[BS / 8];
        scales[i] = (uint8_t)quantise_block<FMT>(v, t, words);
        uint8_t* cr = codes + r * cb + b * (BS / 2);
#pragma unroll
        for (int k = 0; k < BS / 2; ++k)
            if (2 * k < len) cr[k] = (uint8_t)(words[k / 4] >> (8 * (k % 4)));
    }
}

// ---- dequantise ------------------------------------------------------------------------------
// Rows of packs of N elements (16 bytes, or four), back to back: the codes and values of all rows are one
// run each. A thread fills kDequantisePacks packs of output, next to its neighbours' each time. WHOLE: rows
// of whole blocks, whose scales are one run too. Bound by memory: 3M x 48 fp32 97 us (657 MB, 6.7 TB/s); 139
// with one pack a thread, 152 with the packs of a thread side by side.
constexpr int kDequantisePacks = 4;

template <typename T, int FMT, int N, bool WHOLE>
__global__ void __launch_bounds__(256)
    k_mx4_dequantise_blocks(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                            const float* __restrict__ tensor_scale, int64_t packs, const FastDiv row_packs, int nb,
                            T* __restrict__ out) {
    constexpr int BS = Mx4Block<FMT>::size, R = kDequantisePacks;
    // a pack's codes; in whole blocks a word that two packs of four share, faster (97 us, 103 by halves) but
    // beyond the last row where the rows hold an odd number of packs
    constexpr int SHARE = WHOLE && N == 4 ? 2 : 1;
    using Codes = typename std::conditional<N * SHARE == 8, uint32_t, uint16_t>::type;
    const float g = FMT == GS3D_NVFP4 ? __ldg(tensor_scale) : 1.0f;
    const int64_t first = (int64_t)blockIdx.x * (256 * R) + threadIdx.x;
    uint32_t word[R], scale[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
        const int64_t i = min(first + 256 * q, packs - 1);
        word[q] = __ldg(reinterpret_cast<const Codes*>(codes) + i / SHARE);
        int64_t block = i * N / BS;
        if (!WHOLE) {
            const uint32_t r = row_packs.quotient((uint32_t)i);
            block = (int64_t)r * nb + (int)((uint32_t)i - r * row_packs.d) * N / BS;
        }
        scale[q] = __ldg(scales + block);
    }
#pragma unroll
    for (int q = 0; q < R; ++q) {
        const int64_t i = first + 256 * q;
        const Mx4Decode<FMT> d(scale[q], g);
        Pack<T, N> o;
        if constexpr (N == 8) {
            __half2 e[4];
            e2m1_word_half(word[q], e);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 v = mx4_value(d, e[k]);
                o.e[k] = from_f32<T>(v.x);
                o.e[k + 4] = from_f32<T>(v.y);
            }
        } else {
            if (SHARE == 2 && (threadIdx.x & 1)) word[q] >>= 16;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float2 v = mx4_value(d, e2m1_pair_half(word[q] >> (8 * k)));
                o.e[2 * k] = from_f32<T>(v.x);
                o.e[2 * k + 1] = from_f32<T>(v.y);
            }
        }
        using W = typename std::conditional<sizeof(o) == 16, uint4, uint2>::type;
        if (i < packs) __stcs(reinterpret_cast<W*>(out) + i, *reinterpret_cast<const W*>(&o));
    }
}

// A word from shared memory at any byte address (reads up to 3 bytes before it and 7 behind).
__device__ __forceinline__ uint32_t word_at(const unsigned char* p) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(a & ~(uintptr_t)3);
    return __funnelshift_r(w[0], w[1], 8 * (int)(a & 3));
}

// Rows of any length, back to back: a CTA takes `per` rows' codes through shared memory, a block of a
// row a thread, and hands the values back as one range of bytes. 500K x 27 bf16: 10.0 us (5.4 for the
// bytes), for the same reason as k_mx4_quantise_rows.
template <typename T, int FMT>
__global__ void __launch_bounds__(kRowsThreads)
    k_mx4_dequantise_rows(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                          const float* __restrict__ tensor_scale, int64_t rows, int dim, int log_per,
                          T* __restrict__ out) {
    constexpr int BS = Mx4Block<FMT>::size;
    extern __shared__ __align__(16) unsigned char smem[];
    const int nb = (dim + BS - 1) / BS, cb = (dim + 1) / 2, per = 1 << log_per;
    const float g = FMT == GS3D_NVFP4 ? __ldg(tensor_scale) : 1.0f;
    const int64_t r0 = (int64_t)blockIdx.x << log_per;
    const int mine = (int)min((int64_t)per, rows - r0);
    const uint8_t* gc = codes + r0 * cb;
    unsigned char* go = reinterpret_cast<unsigned char*>(out + r0 * dim);
    unsigned char* so = smem + ((16 + (size_t)per * cb + 15) & ~(size_t)15);
    copy_in(smem, gc, mine * cb);
    __syncthreads();
    const unsigned char* sc = smem + head_of(gc);
    T* sv = reinterpret_cast<T*>(so + head_of(go));
    for (int i = threadIdx.x; i < nb << log_per; i += kRowsThreads) {
        const int r = i & (per - 1), b = i >> log_per;
        if (r >= mine) continue;
        const int len = min(BS, dim - b * BS);
        const Mx4Decode<FMT> d(__ldg(scales + (r0 + r) * nb + b), g);
        const unsigned char* c = sc + r * cb + b * (BS / 2);
        T* o = sv + r * dim + b * BS;
#pragma unroll
        for (int k = 0; k < BS; k += 8)
            if (k < len) {
                __half2 e[4];
                e2m1_word_half(word_at(c + k / 2), e);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 v = mx4_value(d, e[j]);
                    if (k + j < len) o[k + j] = from_f32<T>(v.x);
                    if (k + j + 4 < len) o[k + j + 4] = from_f32<T>(v.y);
                }
            }
    }
    __syncthreads();
    copy_out(go, so, mine * dim * (int)sizeof(T));
}

// Rows apart or long: an element a thread, with a division for its row (1M x 48 fp32 into rows 64 apart 160 us,
// back to back 37).
template <typename T, int FMT>
__global__ void __launch_bounds__(256) k_mx4_dequantise(const uint8_t* __restrict__ codes,
                                                        const uint8_t* __restrict__ scales,
                                                        const float* __restrict__ tensor_scale, int64_t rows,
                                                        int64_t stride, int dim, T* __restrict__ out) {
    constexpr int BS = Mx4Block<FMT>::size;
    const int nb = (dim + BS - 1) / BS, cb = (dim + 1) / 2;
    const float g = FMT == GS3D_NVFP4 ? __ldg(tensor_scale) : 1.0f;
    const int64_t total = rows * dim;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
         i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / dim;
        const int k = (int)(i - r * dim);
        const Mx4Decode<FMT> d(scales[r * nb + k / BS], g);
        const float2 two = mx4_value(d, e2m1_pair_half(codes[r * cb + k / 2]));
        out[r * stride + k] = from_f32<T>(k & 1 ? two.y : two.x);
    }
}

// Rows a CTA of the *_rows kernels takes (log2): what fits, as far as it gives each of its threads few blocks.
int log_rows_per_cta(int row_bytes) {
    int l = 0;
    while (2 << l <= kRowsMost && row_bytes * (2 << l) <= kRowsBytes) ++l;
    return l;
}

template <typename T, int FMT, int EL>
int launch_quantise_elements(const gs3d_rows* x, const gs3d_mx4_rows* out, cudaStream_t stream) {
    constexpr int BS = Mx4Block<FMT>::size, N = 16 / (int)sizeof(T);
    const T* in = static_cast<const T*>(x->data);
    const int dim = x->dim, nb = mx4_blocks(dim, FMT);
    const int64_t blocks = x->rows * nb;
    const bool flat = x->row_stride == dim;
    if (packs_of<T, 4 * (int)sizeof(T)>(x) && blocks / 256 < INT_MAX &&
        reinterpret_cast<uintptr_t>(out->codes) % (dim % BS ? 4 : BS / 2) == 0) {
        auto kernel = k_mx4_quantise_blocks<T, FMT, EL, 4, false>;
        if (packs_of<T, 16>(x)) {
            kernel = k_mx4_quantise_blocks<T, FMT, EL, N, false>;
            if constexpr (EL == BS)
                if (dim % BS == 0) kernel = k_mx4_quantise_blocks<T, FMT, EL, N, true>;
        }
        kernel<<<(unsigned)ceil_div(blocks, 256), 256, 0, stream>>>(in, blocks, x->row_stride, dim, FastDiv(nb), flat,
                                                                    out->codes, out->scales, out->tensor_scale);
    } else if (flat && dim * (int)sizeof(T) <= kRowsBytes) {
        const int l = log_rows_per_cta(dim * (int)sizeof(T));
        const size_t smem = ((16 + ((size_t)dim * sizeof(T) << l) + 15) & ~(size_t)15) + 16 +
                            ((size_t)mx4_code_bytes(dim) << l) + 16;
        k_mx4_quantise_rows<T, FMT, EL><<<(unsigned)ceil_div(x->rows, (int64_t)1 << l), kRowsThreads, smem, stream>>>(
            in, x->rows, dim, l, out->codes, out->scales, out->tensor_scale);
    } else {
        k_mx4_quantise<T, FMT><<<grid_for(blocks, 256, 8), 256, 0, stream>>>(
            in, x->rows, x->row_stride, dim, out->codes, out->scales, out->tensor_scale);
    }
    GS3D_LAUNCHED("k_mx4_quantise");
    return GS3D_OK;
}

// Rows shorter than a block need not pay for all of it.
template <typename T, int FMT>
int launch_quantise(const gs3d_rows* x, const gs3d_mx4_rows* out, cudaStream_t stream) {
    if (x->dim <= 8) return launch_quantise_elements<T, FMT, 8>(x, out, stream);
    if (x->dim <= 16) return launch_quantise_elements<T, FMT, 16>(x, out, stream);
    return launch_quantise_elements<T, FMT, Mx4Block<FMT>::size>(x, out, stream);
}

template <typename T, int FMT>
int launch_dequantise(const gs3d_mx4_rows* x, const gs3d_rows* out, cudaStream_t stream) {
    constexpr int BS = Mx4Block<FMT>::size;
    T* o = static_cast<T*>(out->data);
    const int dim = x->dim, nb = mx4_blocks(dim, FMT);
    const int n = packs_of<T, 16>(out) ? 16 / (int)sizeof(T) : 4;
    const int64_t packs = x->rows * dim / n;
    const bool flat = out->row_stride == dim, whole = n * sizeof(T) == 16 && dim % BS == 0;
    if (flat && packs_of<T, 4 * (int)sizeof(T)>(out) && reinterpret_cast<uintptr_t>(x->codes) % 4 == 0 &&
        (whole ? packs / 256 : packs) < INT_MAX) {
        auto kernel = k_mx4_dequantise_blocks<T, FMT, 4, false>;
        if (n * sizeof(T) == 16) kernel = k_mx4_dequantise_blocks<T, FMT, 16 / (int)sizeof(T), false>;
        if (whole) kernel = k_mx4_dequantise_blocks<T, FMT, 16 / (int)sizeof(T), true>;
        kernel<<<(unsigned)ceil_div(packs, 256 * kDequantisePacks), 256, 0, stream>>>(
            x->codes, x->scales, x->tensor_scale, packs, FastDiv(dim / n), nb, o);
    } else if (flat && dim * (int)sizeof(T) <= kRowsBytes) {
        const int l = log_rows_per_cta(dim * (int)sizeof(T));
        const size_t smem = ((16 + ((size_t)mx4_code_bytes(dim) << l) + 15) & ~(size_t)15) + 16 +
                            ((size_t)dim * sizeof(T) << l) + 16 + 16;  // and what word_at reads behind the codes
        k_mx4_dequantise_rows<T, FMT><<<(unsigned)ceil_div(x->rows, (int64_t)1 << l), kRowsThreads, smem, stream>>>(
            x->codes, x->scales, x->tensor_scale, x->rows, dim, l, o);
    } else {
        k_mx4_dequantise<T, FMT><<<grid_for(x->rows * dim, 256, 8), 256, 0, stream>>>(
            x->codes, x->scales, x->tensor_scale, x->rows, out->row_stride, dim, o);
    }
    GS3D_LAUNCHED("k_mx4_dequantise");
    return GS3D_OK;
}

template <typename T>
int launch_tensor_scale(const gs3d_rows* x, float* tensor_scale, cudaStream_t stream) {
    constexpr int N = 16 / (int)sizeof(T);
    const T* in = static_cast<const T*>(x->data);
    const int64_t total = x->rows * x->dim;
    const bool wide = x->row_stride == x->dim && reinterpret_cast<uintptr_t>(in) % 16 == 0;
    uint32_t* out = reinterpret_cast<uint32_t*>(tensor_scale);
    // up to 128 elements a thread one block is as fast as several, which need a zeroed result first
    const int grid = total <= 128 * kScaleThreads ? 1 : grid_for(ceil_div(total, N * 8), kScaleThreads, 4);
    if (grid > 1) GS3D_CUDA(cudaMemsetAsync(tensor_scale, 0, sizeof(float), stream), "memset tensor scale");
    if (wide) k_mx4_tensor_scale<T, true><<<grid, kScaleThreads, 0, stream>>>(in, x->rows, x->row_stride, x->dim, out);
    else k_mx4_tensor_scale<T, false><<<grid, kScaleThreads, 0, stream>>>(in, x->rows, x->row_stride, x->dim, out);
    GS3D_LAUNCHED("k_mx4_tensor_scale");
    return GS3D_OK;
}

// ---- colours ---------------------------------------------------------------------------------
struct Positions {
    float p[GS3D_MAX_FACTORED_VIEWS][3];
};

// Gaussians i and i + 32 of a warp's 64 a thread (neighbouring lanes load and store neighbouring rows),
// their operations in packed pairs. ONE: a single view; else `views` of them a block, with the elements
// decoded once.
// Bound by instruction issue with one view (3M at degree 3: 33 us, 27 for the bytes; 74 % of the issue slots
// used, of some 520 instructions a pair 180 decode), by the stores with several (500K at degree 2, 8 views:
// 17 us, 11.5 for the bytes).
// Blocks an SM: a single view in whole rows holds one channel at a time, 72 registers and 7 blocks (33.4 us;
// 35.5 left to the compiler); several views hold all elements of both Gaussians (degree 3 with 2 / 3 / 4 / 5
// blocks: 479K and 7 views 21.8 / 18.4 / 21.3 / 34.6 us, 916K and 4 views 26.5 / 26.4 / 24.8 / 35.2).
template <int DEG, bool WHOLE, bool ONE>
constexpr int colour_blocks() { return ONE && WHOLE ? 7 : (DEG == 3 ? 3 : 5); }

template <int DEG, int FMT, bool WHOLE, bool ONE>
__global__ void __launch_bounds__(128, colour_blocks<DEG, WHOLE, ONE>())
    k_mx4_colours(const Mx4Sh a, int order, const float4* __restrict__ mo4, int n, const Positions cv, int nv, int views,
                  float4* __restrict__ out, int64_t view_stride) {
    constexpr int NC = (DEG + 1) * (DEG + 1);
    const int64_t i = (int64_t)blockIdx.x * 256 + (threadIdx.x >> 5) * 64 + (threadIdx.x & 31);
    if (i >= n) return;
    const bool two = i + 32 < n;
    const float g = FMT == GS3D_NVFP4 ? __ldg(a.tensor_scale) : 1.0f;
    const int64_t r0 = sh_row(a, i), r1 = two ? sh_row(a, i + 32) : -1;
    const float4 m0 = __ldg(mo4 + i), m1 = __ldg(mo4 + (two ? i + 32 : i));
    const int64_t r[2] = {r0, r1};
    const Float2 mx(m0.x, m1.x), my(m0.y, m1.y), mz(m0.z, m1.z);
    if constexpr (ONE) {
        Float2 c[3];
        mx4_colour<Float2, DEG, FMT, WHOLE>(a, order, r, g, cv.p[0], mx, my, mz, c);
        __stcs(out + i, make_float4(c[0].x, c[1].x, c[2].x, 0.0f));
        if (two) __stcs(out + i + 32, make_float4(c[0].y, c[1].y, c[2].y, 0.0f));
    } else {
        Float2 h[(3 * NC + 7) / 8 * 8], factor[ShRow<DEG, FMT>::NB];
        load_sh<Float2, DEG, FMT, WHOLE>(a, order, r, g, h, factor);
        const int last = min(nv, ((int)blockIdx.y + 1) * views);
        for (int v = blockIdx.y * views; v < last; ++v) {
            Float2 basis[NC], c[3];
            sh_basis_fused<DEG>(cv.p[v], mx, my, mz, basis);
#pragma unroll
            for (int ch = 0; ch < 3; ++ch) c[ch] = mx4_channel<Float2, DEG, FMT, WHOLE>(ch, h + ch * NC, factor, basis);
            float4* o = out + (size_t)v * view_stride + i;
            __stcs(o, make_float4(c[0].x, c[1].x, c[2].x, 0.0f));
            if (two) __stcs(o + 32, make_float4(c[0].y, c[1].y, c[2].y, 0.0f));
        }
    }
}

int check_mx4(const gs3d_mx4_rows* q, const char* what) {
    if (!q) return invalid("NULL %s", what);
    if (q->rows < 0 || q->rows > kMaxRows) return invalid("%s: %lld rows", what, (long long)q->rows);
    if (q->dim < 1 || q->dim > kMaxRowDim) return invalid("%s: dim = %d (1 .. %d)", what, q->dim, kMaxRowDim);
    if (q->format != GS3D_NVFP4 && q->format != GS3D_MXFP4) return invalid("%s: format %d", what, q->format);
    if (q->rows > 0 && (!q->codes || !q->scales)) return invalid("%s: NULL codes or scales", what);
    if (q->format == GS3D_NVFP4 && !q->tensor_scale) return invalid("%s: NULL tensor scale", what);
    if (q->format == GS3D_NVFP4) GS3D_RETURN_IF(check_words(q->tensor_scale, "tensor scale"));
    return GS3D_OK;
}

int check_pair(const gs3d_rows* x, const gs3d_mx4_rows* q) {
    GS3D_RETURN_IF(check_rows(x, "rows"));
    GS3D_RETURN_IF(check_mx4(q, "4-bit rows"));
    if (x->rows != q->rows || x->dim != q->dim)
        return invalid("%lld rows of %d elements and %lld 4-bit rows of %d", (long long)x->rows, x->dim,
                       (long long)q->rows, q->dim);
    return GS3D_OK;
}

// f.run<degree, format, whole rows>()
template <int DEG, typename F>
int dispatch_format(int format, bool whole, F&& f) {
    if (format == GS3D_NVFP4)
        return whole ? f.template run<DEG, GS3D_NVFP4, true>() : f.template run<DEG, GS3D_NVFP4, false>();
    return whole ? f.template run<DEG, GS3D_MXFP4, true>() : f.template run<DEG, GS3D_MXFP4, false>();
}

template <typename F>
int dispatch_colours(const gs3d_mx4_rows* sh, int degree, F&& f) {
    const bool whole = mx4_sh_whole(sh, degree);
    switch (degree) {
        case 0: return dispatch_format<0>(sh->format, whole, f);
        case 1: return dispatch_format<1>(sh->format, whole, f);
        case 2: return dispatch_format<2>(sh->format, whole, f);
        default: return dispatch_format<3>(sh->format, whole, f);
    }
}

struct ColoursLaunch {
    Mx4Sh a;
    int order;
    const float4* mo4;
    int n;
    Positions cv;
    int nv;
    float4* out;
    int64_t view_stride;
    cudaStream_t stream;
    template <int DEG, int FMT, bool WHOLE>
    int run() const {
        const unsigned grid = (unsigned)ceil_div(n, 256);
        if (nv == 1) {
            k_mx4_colours<DEG, FMT, WHOLE, true><<<grid, 128, 0, stream>>>(a, order, mo4, n, cv, nv, 1, out, view_stride);
        } else {
            // all views a block, unless that leaves SMs without: then as many shares of them as fill two waves
            const int64_t waves = 2 * 6 * (int64_t)device_sm_count();
            const int shares = (int)std::min<int64_t>(nv, std::max<int64_t>(1, waves / grid));
            const int views = (int)ceil_div(nv, shares);
            k_mx4_colours<DEG, FMT, WHOLE, false><<<dim3(grid, (unsigned)ceil_div(nv, views)), 128, 0, stream>>>(
                a, order, mo4, n, cv, nv, views, out, view_stride);
        }
        GS3D_LAUNCHED("k_mx4_colours");
        return GS3D_OK;
    }
};

}  // namespace

int check_mx4_sh(const gs3d_mx4_rows* sh, const int32_t* indices, int64_t n, int sh_degree) {
    GS3D_RETURN_IF(check_mx4(sh, "4-bit SH rows"));
    int degree = -1;
    for (int d = 0; d <= 3; ++d)
        if (sh->dim == 3 * (d + 1) * (d + 1)) degree = d;
    if (degree < 0) return invalid("4-bit SH rows: dim = %d is not 3 (d+1)^2 with d <= 3", sh->dim);
    if (sh_degree < 0 || sh_degree > degree)
        return invalid("SH degree %d (storage %d)", sh_degree, degree);
    if (!indices && sh->rows < n)
        return invalid("%lld 4-bit SH rows for %lld Gaussians", (long long)sh->rows, (long long)n);
    GS3D_RETURN_IF(check_words(indices, "indices"));
    return GS3D_OK;
}

}  // namespace gs3d

using namespace gs3d;

extern "C" {

GS3D_API int gs3d_mx4_tensor_scale(const gs3d_rows* x, float* tensor_scale, gs3d_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    GS3D_RETURN_IF(check_rows(x, "rows"));
    if (!tensor_scale) return invalid("NULL tensor scale");
    GS3D_RETURN_IF(check_words(tensor_scale, "tensor scale"));
    ProfScope prof("mx4_quantise", stream);
    return dispatch_type(x->type, [&](auto t) {
        return launch_tensor_scale<typename decltype(t)::T>(x, tensor_scale, stream);
    });
}

GS3D_API int gs3d_mx4_quantise(const gs3d_rows* x, const gs3d_mx4_rows* out, gs3d_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    GS3D_RETURN_IF(check_pair(x, out));
    if (x->rows == 0) return GS3D_OK;
    ProfScope prof("mx4_quantise", stream);
    return dispatch_type(x->type, [&](auto t) {
        using T = typename decltype(t)::T;
        return out->format == GS3D_NVFP4 ? launch_quantise<T, GS3D_NVFP4>(x, out, stream)
                                         : launch_quantise<T, GS3D_MXFP4>(x, out, stream);
    });
}

GS3D_API int gs3d_mx4_dequantise(const gs3d_mx4_rows* x, const gs3d_rows* out, gs3d_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    GS3D_RETURN_IF(check_pair(out, x));
    if (x->rows == 0) return GS3D_OK;
    ProfScope prof("mx4_quantise", stream);
    return dispatch_type(out->type, [&](auto t) {
        using T = typename decltype(t)::T;
        return x->format == GS3D_NVFP4 ? launch_dequantise<T, GS3D_NVFP4>(x, out, stream)
                                       : launch_dequantise<T, GS3D_MXFP4>(x, out, stream);
    });
}

GS3D_API int gs3d_mx4_colours(const gs3d_mx4_rows* sh, int32_t sh_degree, const int32_t* indices,
                              const float* means4, int32_t n, const float* view_positions, int32_t n_views,
                              float* colours, int64_t view_stride, gs3d_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    if (n < 0) return invalid("negative Gaussian count %d", n);
    GS3D_RETURN_IF(check_mx4_sh(sh, indices, n, sh_degree));
    if (!view_positions || (n > 0 && (!means4 || !colours))) return invalid("NULL argument");
    if (n_views < 1 || n_views > GS3D_MAX_FACTORED_VIEWS)
        return invalid("%d views (1 .. %d)", n_views, GS3D_MAX_FACTORED_VIEWS);
    if (view_stride < n) return invalid("view stride %lld < %d", (long long)view_stride, n);
    if ((reinterpret_cast<uintptr_t>(means4) & 15) || (reinterpret_cast<uintptr_t>(colours) & 15))
        return invalid("means or colours not 16-byte aligned");
    if (n == 0) return GS3D_OK;
    ColoursLaunch L{mx4_sh_source(sh, indices), sh->dim / 3, reinterpret_cast<const float4*>(means4), n, {}, n_views,
                    reinterpret_cast<float4*>(colours), view_stride, stream};
    for (int v = 0; v < n_views; ++v)
        for (int k = 0; k < 3; ++k) L.cv.p[v][k] = view_positions[3 * v + k];
    ProfScope prof("mx4_colours", stream);
    return dispatch_colours(sh, sh_degree, L);
}

}  // extern "C"
