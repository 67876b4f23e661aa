// rows.cuh — gs3d_rows on the device and its checks on the host (table.cu, mx4.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace gs3d {

template <int TYPE>
struct RowElem;
template <>
struct RowElem<GS3D_F32> { using T = float; };
template <>
struct RowElem<GS3D_F16> { using T = __half; };
template <>
struct RowElem<GS3D_BF16> { using T = __nv_bfloat16; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

inline int row_elem_bytes(int type) { return type == GS3D_F32 ? 4 : 2; }

constexpr int64_t kMaxRows = (int64_t)1 << 30;  // row counts and indices stay within int32
constexpr int kMaxRowDim = 1 << 16;

// int32 and fp32 arrays: aligned to their elements.
inline int check_words(const void* p, const char* what) {
    if (reinterpret_cast<uintptr_t>(p) & 3) return invalid("%s not 4-byte aligned", what);
    return GS3D_OK;
}

inline int check_rows(const gs3d_rows* r, const char* what) {
    if (!r) return invalid("NULL %s", what);
    if (r->rows < 0 || r->rows > kMaxRows) return invalid("%s: %lld rows", what, (long long)r->rows);
    if (r->dim < 1 || r->dim > kMaxRowDim) return invalid("%s: dim = %d (1 .. %d)", what, r->dim, kMaxRowDim);
    if (r->row_stride < r->dim || r->row_stride > INT_MAX)
        return invalid("%s: row stride %lld with dim %d", what, (long long)r->row_stride, r->dim);
    if (r->type != GS3D_F32 && r->type != GS3D_F16 && r->type != GS3D_BF16)
        return invalid("%s: element type %d", what, r->type);
    if (r->rows > 0 && !r->data) return invalid("%s: NULL data", what);
    if (reinterpret_cast<uintptr_t>(r->data) % row_elem_bytes(r->type))
        return invalid("%s: data not aligned to its elements", what);
    return GS3D_OK;
}

// `bytes` bytes between global and shared memory, 16 at a time where both sides allow it: the shared
// side's first byte is head_of(global side) bytes behind `sh`, which is 16-byte aligned, so that the
// borders of both coincide. Blocks of 16 threads or more.
__device__ __forceinline__ int head_of(const void* p) { return (int)(reinterpret_cast<uintptr_t>(p) & 15); }

__device__ __forceinline__ void copy_in(unsigned char* sh, const unsigned char* gl, int bytes) {
    const int h = head_of(gl), end = h + bytes, first = h ? 16 : 0, last = max(end & ~15, first);
    const unsigned char* g0 = gl - h;
    const int t = threadIdx.x;
    if (t >= h && t < min(first, end)) sh[t] = __ldg(g0 + t);
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(sh);
    for (int i = first + 16 * t; i < last; i += 16 * blockDim.x)  // asynchronous: all of them in flight
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i), "l"(g0 + i) : "memory");
    if (last + t < end) sh[last + t] = __ldg(g0 + last + t);
    asm volatile("cp.async.wait_all;" ::: "memory");
}

__device__ __forceinline__ void copy_out(unsigned char* gl, const unsigned char* sh, int bytes) {
    const int h = head_of(gl), end = h + bytes, first = h ? 16 : 0, last = max(end & ~15, first);
    unsigned char* g0 = gl - h;
    const int t = threadIdx.x;
    if (t >= h && t < min(first, end)) g0[t] = sh[t];
    for (int i = first + 16 * t; i < last; i += 16 * blockDim.x)
        __stcs(reinterpret_cast<uint4*>(g0 + i), *reinterpret_cast<const uint4*>(sh + i));
    if (last + t < end) g0[last + t] = sh[last + t];
}

constexpr int kRowsBytes = 16 << 10;  // the most that a CTA's rows take in shared memory

// Call f(integral constant) with the element type of a checked gs3d_rows.
template <typename F>
inline int dispatch_type(int type, F&& f) {
    switch (type) {
        case GS3D_F32: return f(RowElem<GS3D_F32>{});
        case GS3D_F16: return f(RowElem<GS3D_F16>{});
        default: return f(RowElem<GS3D_BF16>{});
    }
}

}  // namespace gs3d
