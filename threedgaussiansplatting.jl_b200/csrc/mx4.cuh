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

template <int FMT>
__device__ __forceinline__ float mx4_scale(uint32_t byte) {
    return FMT == GS3D_NVFP4 ? e4m3_value(byte) : e8m0_value(byte);
}

// Elements as fp16, times 2^-14: exponent and mantissa bits at bits 11..9 (the element's subnormal is
// then fp16's), the sign at bit 15. By integer operations: the hardware's conversion from e2m1x2 is
// shorter, but as nvcc 12.9 compiles it the elements are wrong (for 252 of the 256 bytes) where its byte
// comes straight from an 8-bit load through __ldg or from shared memory, as some of the uses here do; from
// 16- and 32-bit words, shifted or joined, they are right.
// The two elements of a byte:
__device__ __forceinline__ __half2 e2m1_pair_half(uint32_t byte) {
    const uint32_t h = ((byte << 9) & 0x0e00u) | ((byte << 12) & 0x8000u) | ((byte << 21) & 0x0e000000u) |
                       ((byte << 24) & 0x80000000u);
    return *reinterpret_cast<const __half2*>(&h);
}
// Elements k and k + 4 of a word (lowest bits first) in e[k]: one pair of shifts for both.
__device__ __forceinline__ void e2m1_word_half(uint32_t word, __half2 (&e)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t mag = k < 3 ? word << (9 - 4 * k) : word >> 3;
        const uint32_t h = (mag & 0x0e000e00u) | ((word << (12 - 4 * k)) & 0x80008000u);
        e[k] = *reinterpret_cast<const __half2*>(&h);
    }
}

// The values of two elements: element * block scale * tensor scale, rounded once, as scaled(element *
// 2^-14) * factor().
// NVFP4: element * block scale has 6 significant bits and is a multiple of 2^-10 up to 2688: exact in
// fp16 times 2^-7, with 2^7 of the 2^14 in the scale (at most 57344). The other 2^7 is the factor's, which
// stays finite for every tensor scale up to 2^117. MXFP4: element * 2^k, exact in fp32 up to its overflow
// and underflow.
template <int FMT>
struct Mx4Decode;

template <>
struct Mx4Decode<GS3D_NVFP4> {
    __half2 s;
    float g;
    __device__ __forceinline__ Mx4Decode(uint32_t byte, float tensor_scale)
        : s(__half2half2(__hmul(e4m3_half(byte), __ushort_as_half(0x5800)))), g(tensor_scale * 0x1p7f) {}  // 2^7
    __device__ __forceinline__ float2 scaled(__half2 e) const { return __half22float2(__hmul2(e, s)); }
    __device__ __forceinline__ float factor() const { return g; }
};

template <>
struct Mx4Decode<GS3D_MXFP4> {
    float s;
    __device__ __forceinline__ Mx4Decode(uint32_t byte, float) : s(e8m0_value(byte)) {}
    __device__ __forceinline__ float2 scaled(__half2 e) const {
        return __half22float2(__hmul2(e, __half2half2(__ushort_as_half(0x7400))));  // * 2^14
    }
    __device__ __forceinline__ float factor() const { return s; }
};

template <int FMT>
__device__ __forceinline__ float2 mx4_value(const Mx4Decode<FMT>& d, __half2 e) {
    const float2 v = d.scaled(e);
    return make_float2(v.x * d.factor(), v.y * d.factor());
}

}  // namespace gs3d
