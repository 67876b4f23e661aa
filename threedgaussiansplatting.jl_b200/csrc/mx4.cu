// mx4.cu — microscaled 4-bit rows: quantisation, dequantisation, and the colours of Gaussians whose
// SH coefficients are held in them.
//   gs3d_mx4_tensor_scale   largest magnitude of all rows -> NVFP4 tensor scale
//   gs3d_mx4_quantise       rows -> e2m1 codes and block scales
//   gs3d_mx4_dequantise     and back
//   gs3d_mx4_colours        product of the 4-bit blocks with the SH basis of a view direction
//
// Rounding. An element is the exact quotient |x| / (s g) (s block scale, g tensor scale, 1 for MXFP4)
// rounded to the e2m1 grid, so a value passes the border b between two grid values iff |x| > b s g
// (>= where the tie goes up). b s is exact in fp32 (at most 7 significant bits); b s g is not, but no
// fp32 lies between it and its neighbours RD(b s g) <= b s g <= RU(b s g), so |x| > b s g iff
// |x| > RD(b s g) and |x| >= b s g iff |x| >= RU(b s g): the decision is exact with one directed
// product per border and block.
#include <cfloat>

#include <cuda_fp8.h>

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

// ---- tensor scale ----------------------------------------------------------------------------
// The largest finite |x| as its fp32 bits, which order like unsigned integers.
template <typename T>
__global__ void __launch_bounds__(256) k_mx4_amax(const T* __restrict__ x, int64_t rows, int64_t stride,
                                                  int dim, uint32_t* __restrict__ amax) {
    uint32_t m = 0;
    const int64_t total = rows * dim;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
         i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / dim;
        const uint32_t b = f2u(to_f32(x[r * stride + (i - r * dim)])) & 0x7fffffffu;
        if (b < 0x7f800000u) m = max(m, b);
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0 && m) atomicMax(amax, m);
}

__global__ void k_mx4_amax_to_scale(float* tensor_scale) {
    tensor_scale[0] = fmaxf(tensor_scale[0] / 2688.0f, 0x1p-100f);
}

// ---- quantise --------------------------------------------------------------------------------
// a / (6 g) to the nearest e4m3 value, ties to even, at most 448 (0x7e): an estimate, corrected
// against the exact borders around it.
__device__ __forceinline__ uint32_t nvfp4_scale_byte(float a, float g) {
    const float est = fminf(a / (6.0f * g), 448.0f);
    uint32_t u = __nv_cvt_float_to_fp8(est, __NV_SATFINITE, __NV_E4M3) & 0x7fu;
    if (u < 0x7eu) {
        const float border = 3.0f * (e4m3_value(u) + e4m3_value(u + 1));  // 6 x midpoint, exact
        if ((u & 1u) ? a >= __fmul_ru(border, g) : a > __fmul_rd(border, g)) return u + 1;
    }
    if (u > 0) {
        const float border = 3.0f * (e4m3_value(u) + e4m3_value(u - 1));
        if ((u & 1u) ? a <= __fmul_rd(border, g) : a < __fmul_ru(border, g)) return u - 1;
    }
    return u;
}

// 2^(floor(log2 a) - 2) as its e8m0 byte.
__device__ __forceinline__ uint32_t mxfp4_scale_byte(float a) {
    const int e = (int)(f2u(a) >> 23);
    return (uint32_t)max(e - 2, 0);
}

struct Borders {
    float t[7];  // up iff |x| > t[j] (even j) or |x| >= t[j] (odd j)
};

template <int FMT>
__device__ __forceinline__ Borders mx4_borders(float s, float g) {
    const float b[7] = {0.25f, 0.75f, 1.25f, 1.75f, 2.5f, 3.5f, 5.0f};
    Borders B;
#pragma unroll
    for (int j = 0; j < 7; ++j) {
        const float bs = b[j] * s;
        // an infinity's scale 2^126 takes the last border out of fp32: only infinities pass FLT_MAX
        B.t[j] = FMT == GS3D_MXFP4 ? fminf(bs, FLT_MAX) : ((j & 1) ? __fmul_ru(bs, g) : __fmul_rd(bs, g));
    }
    return B;
}

__device__ __forceinline__ uint32_t e2m1_code(float x, const Borders& B) {
    const float a = fabsf(x);
    uint32_t c = (f2u(x) >> 28) & 8u;
#pragma unroll
    for (int j = 0; j < 7; ++j) c += ((j & 1) ? a >= B.t[j] : a > B.t[j]) ? 1u : 0u;
    return c;
}

// One thread per block of a row.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) k_mx4_quantise(const T* __restrict__ x, int64_t rows, int64_t stride,
                                                      int dim, uint8_t* __restrict__ codes,
                                                      uint8_t* __restrict__ scales,
                                                      const float* __restrict__ tensor_scale) {
    constexpr int BS = Mx4Block<FMT>::size;
    const int nb = (dim + BS - 1) / BS, cb = (dim + 1) / 2;
    const float g = FMT == GS3D_NVFP4 ? __ldg(tensor_scale) : 1.0f;
    const int64_t total = rows * nb;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
         i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / nb;
        const int b = (int)(i - r * nb);
        const int len = min(BS, dim - b * BS);
        const T* xr = x + r * stride + b * BS;
        float v[BS];
        float a = 0.0f;
        bool nan = false;
#pragma unroll
        for (int k = 0; k < BS; ++k) {
            v[k] = k < len ? to_f32(xr[k]) : 0.0f;
            a = fmaxf(a, fabsf(v[k]));
            nan |= v[k] != v[k];
        }
        const uint32_t byte = nan ? (FMT == GS3D_NVFP4 ? 0x7fu : 0xffu)
                                  : (FMT == GS3D_NVFP4 ? nvfp4_scale_byte(a, g) : mxfp4_scale_byte(a));
        scales[i] = (uint8_t)byte;
        const float s = mx4_scale<FMT>(byte);
        const Borders B = mx4_borders<FMT>(s, g);
        uint8_t* cr = codes + r * cb + b * (BS / 2);
#pragma unroll
        for (int k = 0; k < BS; k += 2)
            if (k < len) {
                uint32_t lo = e2m1_code(v[k], B), hi = k + 1 < len ? e2m1_code(v[k + 1], B) : 0u;
                if (s == 0.0f) lo &= 8u, hi &= 8u;
                cr[k / 2] = (uint8_t)(lo | (hi << 4));
            }
    }
}

// ---- dequantise ------------------------------------------------------------------------------
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
        const uint32_t code = (codes[r * cb + k / 2] >> (4 * (k & 1))) & 15u;
        const float s = mx4_scale<FMT>(scales[r * nb + k / BS]);
        out[r * stride + k] = from_f32<T>(mx4_value<FMT>(code, s, g));
    }
}

// ---- colours ---------------------------------------------------------------------------------
template <int DEG, int FMT>
__device__ __forceinline__ void load_mx4_sh(const Mx4Sh& a, int order, int64_t i, float g,
                                            float (&hc)[3][(DEG + 1) * (DEG + 1)]) {
    constexpr int NC = (DEG + 1) * (DEG + 1);
    constexpr int BS = Mx4Block<FMT>::size;
    int64_t r = i;
    bool ok = true;
    if (a.indices) {
        r = (int64_t)a.indices[i] - 1;
        ok = r >= 0 && r < a.rows;
    }
#pragma unroll
    for (int c = 0; c < 3; ++c)
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            const int e = c * order + k;
            hc[c][k] = 0.0f;
            if (ok) {
                const uint32_t code = (a.codes[r * a.code_bytes + e / 2] >> (4 * (e & 1))) & 15u;
                hc[c][k] = mx4_value<FMT>(code, mx4_scale<FMT>(a.scales[r * a.blocks + e / BS]), g);
            }
        }
}

struct Positions {
    float p[GS3D_MAX_FACTORED_VIEWS][3];
};

template <int DEG, int FMT>
__global__ void __launch_bounds__(128) k_mx4_colours(const Mx4Sh a, int order, const float4* __restrict__ mo4,
                                                     int n, const Positions cv, int nv,
                                                     float4* __restrict__ out, int64_t view_stride) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const float g = FMT == GS3D_NVFP4 ? __ldg(a.tensor_scale) : 1.0f;
    float hc[3][(DEG + 1) * (DEG + 1)];
    load_mx4_sh<DEG, FMT>(a, order, i, g, hc);
    const float4 mo = mo4[i];
    for (int v = 0; v < nv; ++v) {
        const float3 c = colour_from_sh<DEG>(hc, cv.p[v], mo.x, mo.y, mo.z);
        out[(size_t)v * view_stride + i] = make_float4(c.x, c.y, c.z, 0.0f);
    }
}

// Floats 6..8 of the filtered Gaussians' 2D records.
template <int DEG, int FMT>
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
        load_mx4_sh<DEG, FMT>(a, order, gi, g, hc);
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

template <typename F>
int dispatch_degree_format(int degree, int format, F&& f) {
#define GS3D_MX4_CASE(D) \
    case D: return format == GS3D_NVFP4 ? f.template run<D, GS3D_NVFP4>() : f.template run<D, GS3D_MXFP4>();
    switch (degree) {
        GS3D_MX4_CASE(0)
        GS3D_MX4_CASE(1)
        GS3D_MX4_CASE(2)
        default: GS3D_MX4_CASE(3)
    }
#undef GS3D_MX4_CASE
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
    template <int DEG, int FMT>
    int run() const {
        k_mx4_colours<DEG, FMT><<<(unsigned)ceil_div(n, 128), 128, 0, stream>>>(a, order, mo4, n, cv, nv, out,
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
    template <int DEG, int FMT>
    int run() const {
        k_mx4_render_colours<DEG, FMT><<<grid_for(n, 128, 16), 128, 0, stream>>>(
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
    return dispatch_degree_format(sh_degree, sh->format, L);
}

}  // namespace gs3d

using namespace gs3d;

extern "C" {

GS3D_API int gs3d_mx4_tensor_scale(const gs3d_rows* x, float* tensor_scale, gs3d_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    GS3D_RETURN_IF(check_rows(x, "rows"));
    if (!tensor_scale) return invalid("NULL tensor scale");
    ProfScope prof("mx4_quantise", stream);
    GS3D_CUDA(cudaMemsetAsync(tensor_scale, 0, sizeof(float), stream), "memset tensor scale");
    if (x->rows > 0)
        GS3D_RETURN_IF(dispatch_type(x->type, [&](auto t) {
            using T = typename decltype(t)::T;
            k_mx4_amax<T><<<grid_for(x->rows * x->dim, 256, 8), 256, 0, stream>>>(
                static_cast<const T*>(x->data), x->rows, x->row_stride, x->dim,
                reinterpret_cast<uint32_t*>(tensor_scale));
            GS3D_LAUNCHED("k_mx4_amax");
            return GS3D_OK;
        }));
    k_mx4_amax_to_scale<<<1, 1, 0, stream>>>(tensor_scale);
    GS3D_LAUNCHED("k_mx4_amax_to_scale");
    return GS3D_OK;
}

GS3D_API int gs3d_mx4_quantise(const gs3d_rows* x, const gs3d_mx4_rows* out, gs3d_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    GS3D_RETURN_IF(check_pair(x, out));
    if (x->rows == 0) return GS3D_OK;
    ProfScope prof("mx4_quantise", stream);
    return dispatch_type(x->type, [&](auto t) {
        using T = typename decltype(t)::T;
        const int grid = grid_for(x->rows * mx4_blocks(x->dim, out->format), 256, 8);
        const T* in = static_cast<const T*>(x->data);
        if (out->format == GS3D_NVFP4)
            k_mx4_quantise<T, GS3D_NVFP4><<<grid, 256, 0, stream>>>(in, x->rows, x->row_stride, x->dim, out->codes,
                                                                    out->scales, out->tensor_scale);
        else
            k_mx4_quantise<T, GS3D_MXFP4><<<grid, 256, 0, stream>>>(in, x->rows, x->row_stride, x->dim, out->codes,
                                                                    out->scales, out->tensor_scale);
        GS3D_LAUNCHED("k_mx4_quantise");
        return GS3D_OK;
    });
}

GS3D_API int gs3d_mx4_dequantise(const gs3d_mx4_rows* x, const gs3d_rows* out, gs3d_stream_t stream_) {
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
    GS3D_RETURN_IF(check_pair(out, x));
    if (x->rows == 0) return GS3D_OK;
    ProfScope prof("mx4_quantise", stream);
    return dispatch_type(out->type, [&](auto t) {
        using T = typename decltype(t)::T;
        const int grid = grid_for(x->rows * x->dim, 256, 8);
        T* o = static_cast<T*>(out->data);
        if (x->format == GS3D_NVFP4)
            k_mx4_dequantise<T, GS3D_NVFP4><<<grid, 256, 0, stream>>>(x->codes, x->scales, x->tensor_scale, x->rows,
                                                                      out->row_stride, x->dim, o);
        else
            k_mx4_dequantise<T, GS3D_MXFP4><<<grid, 256, 0, stream>>>(x->codes, x->scales, x->tensor_scale, x->rows,
                                                                      out->row_stride, x->dim, o);
        GS3D_LAUNCHED("k_mx4_dequantise");
        return GS3D_OK;
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
    return dispatch_degree_format(sh_degree, sh->format, L);
}

}  // extern "C"
