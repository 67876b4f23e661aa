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
//     both convert to the same code, q does. Else a border lies between them, and the block is decided
//     against the borders themselves: q passes a border b iff |x| > b s g (>= where the tie goes up).
//     b s is exact in fp32 (at most 7 significant bits); b s g is not, but no fp32 lies between it and
//     its neighbours RD(b s g) <= b s g <= RU(b s g), so |x| > b s g iff |x| > RD(b s g) and
//     |x| >= b s g iff |x| >= RU(b s g): exact with one directed product per border.
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "mx4.cuh"
#include "rows.cuh"
#include "sh_colour.cuh"

namespace gs3d {
namespace {

int grid_for(int64_t items, int threads, int per_sm) {
    const int64_t b = std::min<int64_t>(ceil_div(items, threads), (int64_t)device_sm_count() * per_sm);
    return (int)std::max<int64_t>(b, 1);
}

template <typename T, int N>
struct alignas(N * sizeof(T)) Pack {
    T e[N];
};

// ---- tensor scale ----------------------------------------------------------------------------
__device__ __forceinline__ void take_finite_abs(uint32_t& m, float v) {
    const uint32_t b = f2u(v) & 0x7fffffffu;  // magnitudes order like unsigned integers
    if (b < 0x7f800000u) m = max(m, b);
}

// Every block turns its largest magnitude into the scale it asks for (monotone, positive: fp32 bits
// order like unsigned integers) and the largest one stays; a lone block stores it. WIDE: rows of
// 16-byte packs, back to back.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) k_mx4_tensor_scale(const T* __restrict__ x, int64_t rows, int64_t stride,
                                                          int dim, uint32_t* __restrict__ tensor_scale) {
    constexpr int N = 16 / (int)sizeof(T);
    __shared__ uint32_t warp_max[8];
    uint32_t m = 0;
    const int64_t total = rows * dim, threads = (int64_t)gridDim.x * blockDim.x;
    const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (WIDE) {
        const Pack<T, N>* p = reinterpret_cast<const Pack<T, N>*>(x);
#pragma unroll 8
        for (int64_t i = t; i < total / N; i += threads) {
            const Pack<T, N> v = p[i];
#pragma unroll
            for (int c = 0; c < N; ++c) take_finite_abs(m, to_f32(v.e[c]));
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
        for (int w = 1; w < 8; ++w) m = max(m, warp_max[w]);
        const uint32_t scale = f2u(fmaxf(u2f(m) / 2688.0f, 0x1p-100f));
        if (gridDim.x == 1) *tensor_scale = scale;
        else atomicMax(tensor_scale, scale);
    }
}

// ---- quantise --------------------------------------------------------------------------------
// a / (6 g) to the nearest e4m3 value, ties to even, at most 448 (0x7e): an estimate (within a step),
// corrected against the exact borders around it.
__device__ __forceinline__ uint32_t nvfp4_scale_byte(float a, float g, float inv6g) {
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

// The code of x against the borders themselves.
__device__ __noinline__ uint32_t e2m1_code_exact(float x, float s, float g) {
    const float b[7] = {0.25f, 0.75f, 1.25f, 1.75f, 2.5f, 3.5f, 5.0f};
    const float a = fabsf(x);
    uint32_t c = 0;
#pragma unroll
    for (int j = 0; j < 7; ++j) {
        const float bs = b[j] * s;
        c += ((j & 1) ? a >= __fmul_ru(bs, g) : a > __fmul_rd(bs, g)) ? 1u : 0u;
    }
    return c | ((f2u(x) >> 28) & 8u);
}

struct TensorScale {
    float g, inv6g;
    template <int FMT>
    static __device__ __forceinline__ TensorScale load(const float* p) {
        TensorScale t{1.0f, 0.0f};
        if (FMT == GS3D_NVFP4) {
            t.g = __ldg(p);
            t.inv6g = 1.0f / (6.0f * t.g);
        }
        return t;
    }
};

// A block's scale byte and the codes of its elements v (zeros behind the row's end), two a byte,
// in words of eight.
template <int FMT>
__device__ __forceinline__ uint32_t quantise_block(const float (&v)[Mx4Block<FMT>::size], const TensorScale& t,
                                                   uint32_t (&words)[Mx4Block<FMT>::size / 8]) {
    constexpr int BS = Mx4Block<FMT>::size;
    float a = 0.0f;
    bool nan = false;
#pragma unroll
    for (int k = 0; k < BS; ++k) {
        a = fmaxf(a, fabsf(v[k]));
        nan |= v[k] != v[k];
    }
    if (FMT == GS3D_MXFP4) {
        const uint32_t byte = mxfp4_scale_byte(a);
        const float inv = u2f((254u - byte) << 23);  // 2^(127 - byte), byte <= 253
#pragma unroll
        for (int w = 0; w < BS / 8; ++w) words[w] = e2m1_word(v + 8 * w, inv);
        return nan ? 0xffu : byte;
    }
    const uint32_t byte = nvfp4_scale_byte(a, t.g, t.inv6g);
    const float s = e4m3_value(byte);
    const float inv = s > 0.0f ? 1.0f / (s * t.g) : 0.0f;
    const float lo = inv * (1.0f - 0x1p-21f), hi = inv * (1.0f + 0x1p-21f);
    uint32_t differ = 0;
#pragma unroll
    for (int w = 0; w < BS / 8; ++w) {
        words[w] = e2m1_word(v + 8 * w, lo);
        differ |= words[w] ^ e2m1_word(v + 8 * w, hi);
    }
    if (differ && s > 0.0f) {
#pragma unroll
        for (int w = 0; w < BS / 8; ++w) {
            words[w] = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) words[w] |= e2m1_code_exact(v[8 * w + k], s, t.g) << (4 * k);
        }
    }
    return nan ? 0x7fu : byte;
}

// Rows of whole blocks in 16-byte packs: a block a thread, from the last row to the first, so that
// what a tensor-scale pass just before has left in L2 is read from there.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) k_mx4_quantise_blocks(const T* __restrict__ x, int64_t blocks, int64_t stride,
                                                             int nb, bool flat, uint8_t* __restrict__ codes,
                                                             uint8_t* __restrict__ scales,
                                                             const float* __restrict__ tensor_scale) {
    constexpr int BS = Mx4Block<FMT>::size, N = 16 / (int)sizeof(T);
    const int64_t i = (int64_t)(gridDim.x - 1 - blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= blocks) return;
    const TensorScale t = TensorScale::load<FMT>(tensor_scale);
    const T* xb = x + i * BS;
    if (!flat) {
        const int64_t r = i / nb;
        xb = x + r * stride + (i - r * nb) * BS;
    }
    float v[BS];
#pragma unroll
    for (int k = 0; k < BS; k += N) {
        const Pack<T, N> p = *reinterpret_cast<const Pack<T, N>*>(xb + k);
#pragma unroll
        for (int c = 0; c < N; ++c) v[k + c] = to_f32(p.e[c]);
    }
    uint32_t words[BS / 8];
    scales[i] = (uint8_t)quantise_block<FMT>(v, t, words);
    Pack<uint32_t, BS / 8> o;
#pragma unroll
    for (int w = 0; w < BS / 8; ++w) o.e[w] = words[w];
    *reinterpret_cast<Pack<uint32_t, BS / 8>*>(codes + i * (BS / 2)) = o;
}

// `bytes` bytes between global and shared memory, 16 at a time where the global side allows it (its
// first `skip` bytes come before a 16-byte border; the shared side starts at its own offset `skip`
// behind a border, so that both sides' packs are aligned).
__device__ __forceinline__ int head_of(const void* p) { return (int)(reinterpret_cast<uintptr_t>(p) & 15); }

__device__ __forceinline__ void copy_in(unsigned char* sh, const unsigned char* gl, int64_t bytes) {
    // sh + head_of(gl) is where the first byte goes
    const int h = head_of(gl);
    const int64_t end = h + bytes;
    const unsigned char* g0 = gl - h;
    const int64_t first = h ? 16 : 0, last = end & ~(int64_t)15;
    for (int64_t i = h + threadIdx.x; i < min(first, end); i += blockDim.x) sh[i] = g0[i];
    for (int64_t i = first + 16 * (int64_t)threadIdx.x; i < last; i += 16 * (int64_t)blockDim.x)
        *reinterpret_cast<uint4*>(sh + i) = *reinterpret_cast<const uint4*>(g0 + i);
    for (int64_t i = max(first, last) + threadIdx.x; i < end; i += blockDim.x) sh[i] = g0[i];
}

__device__ __forceinline__ void copy_out(unsigned char* gl, const unsigned char* sh, int64_t bytes) {
    const int h = head_of(gl);
    const int64_t end = h + bytes;
    unsigned char* g0 = gl - h;
    const int64_t first = h ? 16 : 0, last = end & ~(int64_t)15;
    for (int64_t i = h + threadIdx.x; i < min(first, end); i += blockDim.x) g0[i] = sh[i];
    for (int64_t i = first + 16 * (int64_t)threadIdx.x; i < last; i += 16 * (int64_t)blockDim.x)
        *reinterpret_cast<uint4*>(g0 + i) = *reinterpret_cast<const uint4*>(sh + i);
    for (int64_t i = max(first, last) + threadIdx.x; i < end; i += blockDim.x) g0[i] = sh[i];
}

// Rows of any length (they may end inside a block): a CTA takes `per` rows, which lie back to back, as
// one range of bytes through shared memory, and hands the codes back the same way.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) k_mx4_quantise_rows(const T* __restrict__ x, int64_t rows, int dim, int per,
                                                           uint8_t* __restrict__ codes,
                                                           uint8_t* __restrict__ scales,
                                                           const float* __restrict__ tensor_scale) {
    constexpr int BS = Mx4Block<FMT>::size;
    extern __shared__ __align__(16) unsigned char smem[];
    const int nb = (dim + BS - 1) / BS, cb = (dim + 1) / 2;
    const int64_t r0 = (int64_t)blockIdx.x * per;
    const int mine = (int)min((int64_t)per, rows - r0);
    const unsigned char* gx = reinterpret_cast<const unsigned char*>(x + r0 * dim);
    uint8_t* gc = codes + r0 * cb;
    unsigned char* sc = smem + ((16 + (size_t)per * dim * sizeof(T) + 15) & ~(size_t)15) + head_of(gc);
    copy_in(smem, gx, (int64_t)mine * dim * sizeof(T));
    __syncthreads();
    const T* sx = reinterpret_cast<const T*>(smem + head_of(gx));
    const TensorScale t = TensorScale::load<FMT>(tensor_scale);
    for (int i = threadIdx.x; i < mine * nb; i += blockDim.x) {
        const int r = i / nb, b = i - r * nb;
        const int len = min(BS, dim - b * BS);
        float v[BS];
#pragma unroll
        for (int k = 0; k < BS; ++k) v[k] = k < len ? to_f32(sx[r * dim + b * BS + k]) : 0.0f;
        uint32_t words[BS / 8];
        scales[r0 * nb + i] = (uint8_t)quantise_block<FMT>(v, t, words);
        unsigned char* o = sc + r * cb + b * (BS / 2);
#pragma unroll
        for (int k = 0; k < BS / 2; ++k)
            if (2 * k < len) o[k] = (unsigned char)(words[k / 4] >> (8 * (k % 4)));
    }
    __syncthreads();
    copy_out(gc, sc - head_of(gc), (int64_t)mine * cb);
}

// Rows apart or long: a block a thread, element by element.
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
// Rows of whole blocks, back to back: the codes, scales and values of all rows are one run each. Eight
// elements (a word of codes) a thread.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) k_mx4_dequantise_blocks(const uint32_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales,
                                                               const float* __restrict__ tensor_scale,
                                                               int64_t words, T* __restrict__ out) {
    constexpr int BS = Mx4Block<FMT>::size, N = 16 / (int)sizeof(T);
    const float g = FMT == GS3D_NVFP4 ? __ldg(tensor_scale) : 1.0f;
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= words) return;
    __half2 e[4];
    e2m1_word_half(__ldg(codes + i), e);
    const Mx4Decode<FMT> d(scales[i / (BS / 8)], g);
    Pack<T, N> o[8 / N];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 v = d.value(e[k]);
        o[2 * k / N].e[2 * k % N] = from_f32<T>(v.x);
        o[2 * k / N].e[2 * k % N + 1] = from_f32<T>(v.y);
    }
#pragma unroll
    for (int k = 0; k < 8 / N; ++k) reinterpret_cast<Pack<T, N>*>(out + i * 8)[k] = o[k];
}

// Rows of any length, back to back: a CTA takes `per` rows' codes and scales through shared memory,
// and its threads fill the output's 16-byte packs across the rows' ends.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) k_mx4_dequantise_rows(const uint8_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ scales,
                                                             const float* __restrict__ tensor_scale, int64_t rows,
                                                             int dim, int per, T* __restrict__ out) {
    constexpr int BS = Mx4Block<FMT>::size, N = 16 / (int)sizeof(T);
    extern __shared__ __align__(16) unsigned char smem[];
    const int nb = (dim + BS - 1) / BS, cb = (dim + 1) / 2;
    const float g = FMT == GS3D_NVFP4 ? __ldg(tensor_scale) : 1.0f;
    const int64_t r0 = (int64_t)blockIdx.x * per;
    const int mine = (int)min((int64_t)per, rows - r0);
    const uint8_t* gc = codes + r0 * cb;
    const uint8_t* gs = scales + r0 * nb;
    unsigned char* ss = smem + ((16 + (size_t)per * cb + 15) & ~(size_t)15);
    copy_in(smem, gc, (int64_t)mine * cb);
    copy_in(ss, gs, (int64_t)mine * nb);
    __syncthreads();
    const unsigned char* sc = smem + head_of(gc);
    ss += head_of(gs);
    const int head = head_of(out + r0 * dim) / (int)sizeof(T);  // elements behind a 16-byte border
    T* o0 = out + r0 * dim - head;
    const int end = head + mine * dim;
    for (int p = threadIdx.x; p * N < end; p += blockDim.x) {
        Pack<T, N> o;
        int e = p * N - head;
        int r = e > 0 ? e / dim : 0, c = max(e, 0) - r * dim;
#pragma unroll
        for (int k = 0; k < N; ++k, ++e) {
            float v = 0.0f;
            if (e >= 0 && r < mine) {
                const Mx4Decode<FMT> d(ss[r * nb + c / BS], g);
                const float2 two = d.value(e2m1_pair_half(sc[r * cb + c / 2]));
                v = c & 1 ? two.y : two.x;
                if (++c == dim) c = 0, ++r;
            }
            o.e[k] = from_f32<T>(v);
        }
        if (p * N >= head && (p + 1) * N <= end) {
            *reinterpret_cast<Pack<T, N>*>(o0 + p * N) = o;
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (p * N + k >= head && p * N + k < end) o0[p * N + k] = o.e[k];
        }
    }
}

// Rows apart or long: an element a thread.
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
        const float2 two = d.value(e2m1_pair_half(codes[r * cb + k / 2]));
        out[r * stride + k] = from_f32<T>(k & 1 ? two.y : two.x);
    }
}

constexpr int kRowsBytes = 16 << 10;  // of a CTA's rows in shared memory (three CTAs' worth of 256 threads fit)

// Rows a CTA of the *_rows kernels takes: about kRowsBytes of them, fewer where that leaves SMs without.
int rows_per_cta(int64_t rows, int row_bytes) {
    const int64_t fit = std::max(1, kRowsBytes / row_bytes);
    return (int)std::max<int64_t>(1, std::min<int64_t>(fit, ceil_div(rows, 4 * (int64_t)device_sm_count())));
}

template <typename T, int FMT>
int launch_quantise(const gs3d_rows* x, const gs3d_mx4_rows* out, cudaStream_t stream) {
    constexpr int BS = Mx4Block<FMT>::size, N = 16 / (int)sizeof(T);
    const T* in = static_cast<const T*>(x->data);
    const int dim = x->dim, nb = mx4_blocks(dim, FMT);
    const int64_t blocks = x->rows * nb;
    const bool flat = x->row_stride == dim;
    if (dim % BS == 0 && x->row_stride % N == 0 && reinterpret_cast<uintptr_t>(in) % 16 == 0 &&
        reinterpret_cast<uintptr_t>(out->codes) % (BS / 2) == 0 && blocks / 256 < INT_MAX) {
        k_mx4_quantise_blocks<T, FMT><<<(unsigned)ceil_div(blocks, 256), 256, 0, stream>>>(
            in, blocks, x->row_stride, nb, flat, out->codes, out->scales, out->tensor_scale);
    } else if (flat && dim * (int)sizeof(T) <= kRowsBytes) {
        const int per = rows_per_cta(x->rows, dim * (int)sizeof(T));
        const size_t smem = ((16 + (size_t)per * dim * sizeof(T) + 15) & ~(size_t)15) + 16 +
                            (size_t)per * mx4_code_bytes(dim) + 16;
        k_mx4_quantise_rows<T, FMT><<<(unsigned)ceil_div(x->rows, per), 256, smem, stream>>>(
            in, x->rows, dim, per, out->codes, out->scales, out->tensor_scale);
    } else {
        k_mx4_quantise<T, FMT><<<grid_for(blocks, 256, 8), 256, 0, stream>>>(
            in, x->rows, x->row_stride, dim, out->codes, out->scales, out->tensor_scale);
    }
    GS3D_LAUNCHED("k_mx4_quantise");
    return GS3D_OK;
}

template <typename T, int FMT>
int launch_dequantise(const gs3d_mx4_rows* x, const gs3d_rows* out, cudaStream_t stream) {
    constexpr int BS = Mx4Block<FMT>::size;
    T* o = static_cast<T*>(out->data);
    const int dim = x->dim;
    const int64_t words = x->rows * dim / 8;
    const bool flat = out->row_stride == dim;
    if (flat && dim % BS == 0 && reinterpret_cast<uintptr_t>(o) % 16 == 0 &&
        reinterpret_cast<uintptr_t>(x->codes) % 4 == 0 && words / 256 < INT_MAX) {
        k_mx4_dequantise_blocks<T, FMT><<<(unsigned)ceil_div(words, 256), 256, 0, stream>>>(
            reinterpret_cast<const uint32_t*>(x->codes), x->scales, x->tensor_scale, words, o);
    } else if (flat && dim * (int)sizeof(T) <= kRowsBytes) {
        const int per = rows_per_cta(x->rows, dim * (int)sizeof(T));
        const size_t smem = ((16 + (size_t)per * mx4_code_bytes(dim) + 15) & ~(size_t)15) + 16 +
                            (size_t)per * mx4_blocks(dim, FMT) + 16;
        k_mx4_dequantise_rows<T, FMT><<<(unsigned)ceil_div(x->rows, per), 256, smem, stream>>>(
            x->codes, x->scales, x->tensor_scale, x->rows, dim, per, o);
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
    // up to 64 elements a thread one block is as fast as several and needs no zeroed result before it
    const int grid = total <= 64 * 256 ? 1 : grid_for(ceil_div(total, N * 8), 256, 8);
    if (grid > 1) GS3D_CUDA(cudaMemsetAsync(tensor_scale, 0, sizeof(float), stream), "memset tensor scale");
    if (wide) k_mx4_tensor_scale<T, true><<<grid, 256, 0, stream>>>(in, x->rows, x->row_stride, x->dim, out);
    else k_mx4_tensor_scale<T, false><<<grid, 256, 0, stream>>>(in, x->rows, x->row_stride, x->dim, out);
    GS3D_LAUNCHED("k_mx4_tensor_scale");
    return GS3D_OK;
}

// ---- colours ---------------------------------------------------------------------------------
// The coefficients of Gaussian i. WHOLE: rows of exactly the rendered degree, their codes aligned to
// 8 bytes at degree 3 (24 bytes a row) and to 2 below (2, 6 and 14 bytes): wide loads, and every
// element's byte and block known at compile time. Else element by element.
template <int DEG, int FMT, bool WHOLE>
__device__ __forceinline__ void load_mx4_sh(const Mx4Sh& a, int order, int64_t i, float g,
                                            float (&hc)[3][(DEG + 1) * (DEG + 1)]) {
    constexpr int NC = (DEG + 1) * (DEG + 1), DIM = 3 * NC;
    constexpr int BS = Mx4Block<FMT>::size, NB = (DIM + BS - 1) / BS, CB = (DIM + 1) / 2;
    int64_t r = i;
    if (a.indices) {
        r = (int64_t)__ldg(a.indices + i) - 1;
        if (r < 0 || r >= a.rows) {
#pragma unroll
            for (int e = 0; e < DIM; ++e) (&hc[0][0])[e] = 0.0f;
            return;
        }
    }
    if (WHOLE) {
        using W = typename std::conditional<DEG == 3, uint2, uint16_t>::type;
        constexpr int NW = CB / (int)sizeof(W);
        W w[NW];
        const W* p = reinterpret_cast<const W*>(a.codes + r * CB);
#pragma unroll
        for (int k = 0; k < NW; ++k) w[k] = __ldg(p + k);
        const uint8_t* s = a.scales + r * NB;
        uint32_t sb[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) sb[b] = __ldg(s + b);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const Mx4Decode<FMT> d(sb[b], g);
#pragma unroll
            for (int e0 = b * BS; e0 < (b + 1) * BS && e0 < DIM; e0 += 8) {
                uint32_t word;
                if constexpr (DEG == 3) {
                    word = (e0 / 8) & 1 ? w[e0 / 16].y : w[e0 / 16].x;
                } else {
                    // the row's last word may be half: what is doubled then lies behind its end
                    word = w[e0 / 4] | (uint32_t)w[e0 / 4 + 1 < NW ? e0 / 4 + 1 : e0 / 4] << 16;
                }
                __half2 h[4];
                e2m1_word_half(word, h);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 v = d.value(h[k]);
                    if (e0 + 2 * k < DIM) (&hc[0][0])[e0 + 2 * k] = v.x;
                    if (e0 + 2 * k + 1 < DIM) (&hc[0][0])[e0 + 2 * k + 1] = v.y;
                }
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < 3; ++c)
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                const int e = c * order + k;
                const Mx4Decode<FMT> d(a.scales[r * a.blocks + e / BS], g);
                const float2 v = d.value(e2m1_pair_half(a.codes[r * a.code_bytes + e / 2]));
                hc[c][k] = e & 1 ? v.y : v.x;
            }
    }
}

struct Positions {
    float p[GS3D_MAX_FACTORED_VIEWS][3];
};

template <int DEG, int FMT, bool WHOLE>
__global__ void __launch_bounds__(128) k_mx4_colours(const Mx4Sh a, int order, const float4* __restrict__ mo4,
                                                     int n, const Positions cv, int nv,
                                                     float4* __restrict__ out, int64_t view_stride) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const float g = FMT == GS3D_NVFP4 ? __ldg(a.tensor_scale) : 1.0f;
    float hc[3][(DEG + 1) * (DEG + 1)];
    load_mx4_sh<DEG, FMT, WHOLE>(a, order, i, g, hc);
    const float4 mo = mo4[i];
    for (int v = 0; v < nv; ++v) {
        const float3 c = colour_from_sh<DEG>(hc, cv.p[v], mo.x, mo.y, mo.z);
        out[(size_t)v * view_stride + i] = make_float4(c.x, c.y, c.z, 0.0f);
    }
}

// Floats 6..8 of the filtered Gaussians' 2D records.
template <int DEG, int FMT, bool WHOLE>
__global__ void __launch_bounds__(128) k_mx4_render_colours(const Mx4Sh a, int order,
                                                            const float4* __restrict__ mo4,
                                                            const int32_t* __restrict__ f2g,
                                                            const int32_t* __restrict__ counts,
                                                            const gs3d_camera cam, float* __restrict__ f2d) {
    const int F = counts[0];
    const float g = FMT == GS3D_NVFP4 ? __ldg(a.tensor_scale) : 1.0f;
    for (int f = blockIdx.x * blockDim.x + threadIdx.x; f < F; f += gridDim.x * blockDim.x) {
        const int gi = f2g[f] - 1;
        float hc[3][(DEG + 1) * (DEG + 1)];
        load_mx4_sh<DEG, FMT, WHOLE>(a, order, gi, g, hc);
        const float4 mo = mo4[gi];
        const float3 c = colour_from_sh<DEG>(hc, cam.position, mo.x, mo.y, mo.z);
        float* rr = f2d + 9 * (size_t)f;
        rr[6] = c.x; rr[7] = c.y; rr[8] = c.z;
    }
}

int check_mx4(const gs3d_mx4_rows* q, const char* what) {
    if (!q) return invalid("NULL %s", what);
    if (q->rows < 0 || q->rows > kMaxRows) return invalid("%s: %lld rows", what, (long long)q->rows);
    if (q->dim < 1 || q->dim > kMaxRowDim) return invalid("%s: dim = %d (1 .. %d)", what, q->dim, kMaxRowDim);
    if (q->format != GS3D_NVFP4 && q->format != GS3D_MXFP4) return invalid("%s: format %d", what, q->format);
    if (q->rows > 0 && (!q->codes || !q->scales)) return invalid("%s: NULL codes or scales", what);
    if (q->format == GS3D_NVFP4 && !q->tensor_scale) return invalid("%s: NULL tensor scale", what);
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
    const bool whole = sh->dim == 3 * (degree + 1) * (degree + 1) &&
                       reinterpret_cast<uintptr_t>(sh->codes) % (degree == 3 ? 8 : 2) == 0;
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
        k_mx4_colours<DEG, FMT, WHOLE><<<(unsigned)ceil_div(n, 128), 128, 0, stream>>>(a, order, mo4, n, cv, nv, out,
                                                                             view_stride);
        GS3D_LAUNCHED("k_mx4_colours");
        return GS3D_OK;
    }
};

struct RenderColoursLaunch {
    Mx4Sh a;
    int order;
    const float4* mo4;
    int n;
    const gs3d_render_buffers* buf;
    const gs3d_camera* cam;
    cudaStream_t stream;
    template <int DEG, int FMT, bool WHOLE>
    int run() const {
        k_mx4_render_colours<DEG, FMT, WHOLE><<<grid_for(n, 128, 16), 128, 0, stream>>>(
            a, order, mo4, buf->fgidx_to_gidx, buf->device_counts, *cam,
            buf->means2d_opacities_inverse_covariances_colors);
        GS3D_LAUNCHED("k_mx4_render_colours");
        return GS3D_OK;
    }
};

Mx4Sh sh_source(const gs3d_mx4_rows* sh, const int32_t* indices) {
    return Mx4Sh{sh->codes, sh->scales, sh->tensor_scale, indices, sh->rows, mx4_code_bytes(sh->dim),
                 mx4_blocks(sh->dim, sh->format)};
}

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
    return GS3D_OK;
}

int launch_mx4_render_colours(const gs3d_mx4_rows* sh, const int32_t* indices, const float* means4, int n,
                              const gs3d_camera* cam, int sh_degree, const gs3d_render_buffers* buf,
                              cudaStream_t stream) {
    if (n == 0) return GS3D_OK;
    ProfScope prof("mx4_colours", stream);
    const RenderColoursLaunch L{sh_source(sh, indices), sh->dim / 3, reinterpret_cast<const float4*>(means4), n,
                                buf, cam, stream};
    return dispatch_colours(sh, sh_degree, L);
}

}  // namespace gs3d

using namespace gs3d;

extern "C" {

GS3D_API int gs3d_mx4_tensor_scale(const gs3d_rows* x, float* tensor_scale, gs3d_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    GS3D_RETURN_IF(check_rows(x, "rows"));
    if (!tensor_scale) return invalid("NULL tensor scale");
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
    ColoursLaunch L{sh_source(sh, indices), sh->dim / 3, reinterpret_cast<const float4*>(means4), n, {}, n_views,
                    reinterpret_cast<float4*>(colours), view_stride, stream};
    for (int v = 0; v < n_views; ++v)
        for (int k = 0; k < 3; ++k) L.cv.p[v][k] = view_positions[3 * v + k];
    ProfScope prof("mx4_colours", stream);
    return dispatch_colours(sh, sh_degree, L);
}

}  // extern "C"
