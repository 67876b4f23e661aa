// mx4.cuh — microscaled 4-bit elements (e2m1) and their block scales, decoded.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace gs3d {

template <int FMT>
struct Mx4Block {
    static constexpr int size = FMT == GS3D_NVFP4 ? 16 : 32;
};
inline int mx4_block(int format) { return format == GS3D_NVFP4 ? 16 : 32; }
inline int mx4_blocks(int dim, int format) { return (dim + mx4_block(format) - 1) / mx4_block(format); }
inline int mx4_code_bytes(int dim) { return (dim + 1) / 2; }

// An unsigned e4m3 byte (the top bit is not part of it): subnormals m 2^-9, 0x7f NaN.
__device__ __forceinline__ __half e4m3_half(uint32_t byte) {
    return __half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)(byte & 0x7fu), __NV_E4M3));
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) { return __half2float(e4m3_half(byte)); }

// An e8m0 byte: 2^(byte - 127), 0xff NaN; byte 0 is the subnormal 2^-127.
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    if (byte == 0xffu) return u2f(0x7fc00000u);
    return byte == 0 ? 0x1p-127f : u2f(byte << 23);
}

// The two elements of a byte, exactly, in fp16: exponent and mantissa bits placed at bits 11..9 are
// the element * 2^-14 (its subnormal is fp16's).
__device__ __forceinline__ __half2 e2m1_pair_half(uint32_t byte) {
    const uint32_t h = ((byte & 0x07u) << 9) | ((byte & 0x08u) << 12) | ((byte & 0x70u) << 21) | ((byte & 0x80u) << 24);
    return __hmul2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x7400)));  // 2^14
}

// The eight elements of a word, lowest bits first, by the hardware's conversion. Only for words that
// come from 32-bit loads or arithmetic: fed straight from a 16- or 8-bit load it returned wrong
// elements (nvcc 12.9; the tests go through every code).
__device__ __forceinline__ void e2m1_word_half(uint32_t word, __half2 (&e)[4]) {
    uint32_t h[4];
    asm("{ .reg .b8 a, b, c, d; mov.b32 {a, b, c, d}, %4;\n"
        "  cvt.rn.f16x2.e2m1x2 %0, a; cvt.rn.f16x2.e2m1x2 %1, b;\n"
        "  cvt.rn.f16x2.e2m1x2 %2, c; cvt.rn.f16x2.e2m1x2 %3, d; }"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(word));
#pragma unroll
    for (int k = 0; k < 4; ++k) e[k] = *reinterpret_cast<__half2*>(&h[k]);
}

// The values of the two elements of a byte: element * block scale * tensor scale, rounded once.
// NVFP4: element * block scale has 6 significant bits between 2^-10 and 2688, exact in fp16.
// MXFP4: element * 2^k, exact in fp32 up to its overflow and underflow.
template <int FMT>
struct Mx4Decode;

template <>
struct Mx4Decode<GS3D_NVFP4> {
    __half2 s;
    float g;
    __device__ __forceinline__ Mx4Decode(uint32_t byte, float tensor_scale)
        : s(__half2half2(e4m3_half(byte))), g(tensor_scale) {}
    __device__ __forceinline__ float2 value(__half2 e) const {
        const float2 v = __half22float2(__hmul2(e, s));
        return make_float2(v.x * g, v.y * g);
    }
};

template <>
struct Mx4Decode<GS3D_MXFP4> {
    float s;
    __device__ __forceinline__ Mx4Decode(uint32_t byte, float) : s(e8m0_value(byte)) {}
    __device__ __forceinline__ float2 value(__half2 e) const {
        const float2 v = __half22float2(e);
        return make_float2(v.x * s, v.y * s);
    }
};

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
