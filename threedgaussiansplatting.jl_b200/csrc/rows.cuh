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

inline int check_rows(const gs3d_rows* r, const char* what) {
    if (!r) return invalid("NULL %s", what);
    if (r->rows < 0 || r->rows > kMaxRows) return invalid("%s: %lld rows", what, (long long)r->rows);
    if (r->dim < 1 || r->dim > kMaxRowDim) return invalid("%s: dim = %d (1 .. %d)", what, r->dim, kMaxRowDim);
    if (r->row_stride < r->dim || r->row_stride > ((int64_t)1 << 32))
        return invalid("%s: row stride %lld with dim %d", what, (long long)r->row_stride, r->dim);
    if (r->type != GS3D_F32 && r->type != GS3D_F16 && r->type != GS3D_BF16)
        return invalid("%s: element type %d", what, r->type);
    if (r->rows > 0 && !r->data) return invalid("%s: NULL data", what);
    if (reinterpret_cast<uintptr_t>(r->data) % row_elem_bytes(r->type))
        return invalid("%s: data not aligned to its elements", what);
    return GS3D_OK;
}

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
