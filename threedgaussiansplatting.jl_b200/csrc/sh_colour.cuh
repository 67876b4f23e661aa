// sh_colour.cuh — a Gaussian's colour from its SH coefficients (sh_coeffs_to_color, sh.jl:38-112),
// shared by every kernel that computes colours so that they agree bit for bit.
#pragma once
#include "common.cuh"

namespace gs3d {

// sh_coeffs_to_color (sh.jl:38-112) for one channel; hc = coefficient 1 of that channel
template <int DEG>
__device__ __forceinline__ float sh_channel(const float* hc, float x, float y, float z) {
    float cc = sh_basis(1, x, y, z) * hc[0];
    if (DEG >= 1) {
        cc += (sh_basis(2, x, y, z) * hc[1] + sh_basis(3, x, y, z) * hc[2] +
               sh_basis(4, x, y, z) * hc[3]);
        if (DEG >= 2) {
            cc += (sh_basis(5, x, y, z) * hc[4] + sh_basis(6, x, y, z) * hc[5] +
                   sh_basis(7, x, y, z) * hc[6] + sh_basis(8, x, y, z) * hc[7] +
                   sh_basis(9, x, y, z) * hc[8]);
            if (DEG >= 3) {
                cc += (sh_basis(10, x, y, z) * hc[9] + sh_basis(11, x, y, z) * hc[10] +
                       sh_basis(12, x, y, z) * hc[11] + sh_basis(13, x, y, z) * hc[12] +
                       sh_basis(14, x, y, z) * hc[13] + sh_basis(15, x, y, z) * hc[14] +
                       sh_basis(16, x, y, z) * hc[15]);
            }
        }
    }
    cc += 0.5f;
    if (cc < 0.0f) cc = 0.0f;
    return cc;
}

// sh_coeffs_to_color (sh.jl:38-112) seen from camera position p: the clamped colour.
template <int DEG>
__device__ __forceinline__ float3 colour_from_sh(const float (&hc)[3][(DEG + 1) * (DEG + 1)],
                                                 const float* p, float mx0, float my0, float mz0) {
    const float vx = mx0 - p[0], vy = my0 - p[1], vz = mz0 - p[2];
    const float inv = 1.0f / sqrtf(vx * vx + vy * vy + vz * vz);
    const float dx = vx * inv, dy = vy * inv, dz = vz * inv;
    return make_float3(sh_channel<DEG>(hc[0], dx, dy, dz), sh_channel<DEG>(hc[1], dx, dy, dz),
                       sh_channel<DEG>(hc[2], dx, dy, dz));
}

// Two fp32 values in one 64-bit register, for the packed instructions (one issue slot for two
// operations, each rounded as the scalar one): two Gaussians side by side. Products, sums and
// differences are all fma (a b + -0, a 1 + b, b (-1) + a round as they do) with 1, -1 and -0 from
// memory: mul.rn.f32x2 followed by add.rn.f32x2 came back as one fused operation (nvcc 12.9), and so
// did fma with constants the compiler could see.
struct Float2 {
    float x, y;
    __device__ __forceinline__ Float2() {}
    __device__ __forceinline__ explicit Float2(float v) : x(v), y(v) {}
    __device__ __forceinline__ Float2(float a, float b) : x(a), y(b) {}
};
static __constant__ float kPackedUnits[3] = {1.0f, -1.0f, -0.0f};
__device__ __forceinline__ Float2 fma2(Float2 a, Float2 b, Float2 c) {
    Float2 r;
    asm("{ .reg .b64 a, b, c, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 c, {%6, %7};\n"
        "  fma.rn.f32x2 d, a, b, c; mov.b64 {%0, %1}, d; }"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ Float2 operator*(Float2 a, Float2 b) { return fma2(a, b, Float2(kPackedUnits[2])); }
__device__ __forceinline__ Float2 operator+(Float2 a, Float2 b) { return fma2(a, Float2(kPackedUnits[0]), b); }
__device__ __forceinline__ Float2 operator-(Float2 a, Float2 b) { return fma2(b, Float2(kPackedUnits[1]), a); }
__device__ __forceinline__ Float2 operator*(Float2 a, float b) { return a * Float2(b); }
__device__ __forceinline__ Float2 operator*(float a, Float2 b) { return Float2(a) * b; }
__device__ __forceinline__ Float2 operator-(Float2 a) { return Float2(-a.x, -a.y); }

// The basis functions at the unit directions from p to two means, with colour_from_sh's operations.
template <int DEG>
__device__ __forceinline__ void sh_basis_pair(const float* p, Float2 mx, Float2 my, Float2 mz,
                                              Float2 (&basis)[(DEG + 1) * (DEG + 1)]) {
    const Float2 vx = mx - Float2(p[0]), vy = my - Float2(p[1]), vz = mz - Float2(p[2]);
    const Float2 ss = vx * vx + vy * vy + vz * vz;
    const Float2 inv(1.0f / sqrtf(ss.x), 1.0f / sqrtf(ss.y));
    const Float2 dx = vx * inv, dy = vy * inv, dz = vz * inv;
#pragma unroll
    for (int k = 0; k < (DEG + 1) * (DEG + 1); ++k) basis[k] = sh_basis(k + 1, dx, dy, dz);
}

// sh_channel for two Gaussians, with its operations in its order.
template <int DEG>
__device__ __forceinline__ Float2 sh_channel_pair(const Float2* hc, const Float2* basis) {
    Float2 cc = basis[0] * hc[0];
#pragma unroll
    for (int d = 1; d <= DEG; ++d) {
        Float2 band = basis[d * d] * hc[d * d];
#pragma unroll
        for (int k = d * d + 1; k < (d + 1) * (d + 1); ++k) band = band + basis[k] * hc[k];
        cc = cc + band;
    }
    cc = cc + Float2(0.5f);
    if (cc.x < 0.0f) cc.x = 0.0f;
    if (cc.y < 0.0f) cc.y = 0.0f;
    return cc;
}

}  // namespace gs3d
