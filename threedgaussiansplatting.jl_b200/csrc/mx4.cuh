// mx4.cuh — microscaled 4-bit elements (e2m1) and their block scales, decoded.
#pragma once
#include "common.cuh"

namespace gs3d {

template <int FMT>
struct Mx4Block {
    static constexpr int size = FMT == GS3D_NVFP4 ? 16 : 32;
};
inline int mx4_block(int format) { return format == GS3D_NVFP4 ? 16 : 32; }
inline int mx4_blocks(int dim, int format) { return (dim + mx4_block(format) - 1) / mx4_block(format); }
inline int mx4_code_bytes(int dim) { return (dim + 1) / 2; }

// 0, 1/2, 1, 3/2, 2, 3, 4, 6 with a sign: exponent and mantissa bit placed at bits 24..22 of an
// fp32 read as element * 2^-126 (its subnormal is fp32's), the sign at bit 31.
__device__ __forceinline__ float e2m1_value(uint32_t code) {
    const uint32_t bits = ((code & 7u) << 22) | ((code & 8u) << 28);
    return u2f(bits) * 0x1p126f;
}

// An unsigned e4m3 byte (the top bit is not part of it): subnormals m 2^-9, 0x7f NaN.
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
    const uint32_t b = byte & 0x7fu;
    if (b == 0x7fu) return u2f(0x7fc00000u);
    return u2f(b << 20) * 0x1p120f;  // exponent bits at 26..23: value * 2^-120, subnormals included
}

// An e8m0 byte: 2^(byte - 127), 0xff NaN; byte 0 is the subnormal 2^-127.
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    if (byte == 0xffu) return u2f(0x7fc00000u);
    return byte == 0 ? 0x1p-127f : u2f(byte << 23);
}

template <int FMT>
__device__ __forceinline__ float mx4_scale(uint32_t byte) {
    return FMT == GS3D_NVFP4 ? e4m3_value(byte) : e8m0_value(byte);
}

// element * block scale (exact: 2 and 4 significant bits) * tensor scale, rounded once.
template <int FMT>
__device__ __forceinline__ float mx4_value(uint32_t code, float scale, float tensor_scale) {
    const float v = e2m1_value(code) * scale;
    return FMT == GS3D_NVFP4 ? v * tensor_scale : v;
}

// 4-bit SH rows as a colour source: row i, or row indices[i].
struct Mx4Sh {
    const uint8_t* codes;
    const uint8_t* scales;
    const float* tensor_scale;
    const int32_t* indices;
    int64_t rows;
    int code_bytes, blocks;
};

}  // namespace gs3d
