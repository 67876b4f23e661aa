// sh_colour.cuh — a Gaussian's colour from its SH coefficients (sh_coeffs_to_color, sh.jl:38-112),
// shared by every kernel that computes colours from fp32 coefficients so that they agree bit for bit; and
// the SH basis with fused multiply-adds, of the colours from 4-bit rows.
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

// Two fp32 values in one 64-bit register, for the packed fused multiply-add (one issue slot for two):
// two Gaussians side by side.
struct Float2 {
    float x, y;
    __device__ __forceinline__ Float2() {}
    __device__ __forceinline__ explicit Float2(float v) : x(v), y(v) {}
    __device__ __forceinline__ Float2(float a, float b) : x(a), y(b) {}
};
__device__ __forceinline__ Float2 fma2(Float2 a, Float2 b, Float2 c) {
    Float2 r;
    asm("{ .reg .b64 a, b, c, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 c, {%6, %7};\n"
        "  fma.rn.f32x2 d, a, b, c; mov.b64 {%0, %1}, d; }"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ Float2 operator*(Float2 a, Float2 b) {
    Float2 r;
    asm("{ .reg .b64 a, b, c; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mul.rn.f32x2 c, a, b; mov.b64 {%0, %1}, c; }"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

__device__ __forceinline__ float fma2(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float rsqrt2(float v) { return rsqrtf(v); }
__device__ __forceinline__ Float2 rsqrt2(Float2 v) { return Float2(rsqrtf(v.x), rsqrtf(v.y)); }

// The basis functions (sh.jl:123-149) at the unit direction from p to a mean (V: float) or to two
// (Float2), with fused multiply-adds and the reciprocal square root (rsqrtf, 2 ulp): within a few ulp of
// sh_basis.
template <int DEG, typename V>
__device__ __forceinline__ void sh_basis_fused(const float* p, V mx, V my, V mz, V (&b)[(DEG + 1) * (DEG + 1)]) {
    b[0] = V(sh_c(1));
    if constexpr (DEG >= 1) {
        const V one(1.0f), minus(-1.0f);
        V x = fma2(mx, one, V(-p[0])), y = fma2(my, one, V(-p[1])), z = fma2(mz, one, V(-p[2]));
        const V inv = rsqrt2(fma2(z, z, fma2(y, y, x * x)));
        x = x * inv, y = y * inv, z = z * inv;
        b[1] = y * V(-sh_c(2));
        b[2] = z * V(sh_c(3));
        b[3] = x * V(-sh_c(4));
        if constexpr (DEG >= 2) {
            const V xx = x * x, yy = y * y, zz = z * z, xy = x * y;
            const V sum = fma2(xx, one, yy), diff = fma2(yy, minus, xx), less = sum * minus;
            b[4] = xy * V(sh_c(5));
            b[5] = y * z * V(sh_c(6));
            b[6] = fma2(zz, V(2.0f), less) * V(sh_c(7));
            b[7] = x * z * V(sh_c(8));
            b[8] = diff * V(sh_c(9));
            if constexpr (DEG >= 3) {
                const V four = fma2(zz, V(4.0f), less);
                b[9] = y * V(sh_c(10)) * fma2(xx, V(3.0f), yy * minus);
                b[10] = xy * z * V(sh_c(11));
                b[11] = y * V(sh_c(12)) * four;
                b[12] = z * V(sh_c(13)) * fma2(zz, V(2.0f), sum * V(-3.0f));
                b[13] = x * V(sh_c(14)) * four;
                b[14] = z * V(sh_c(15)) * diff;
                b[15] = x * V(sh_c(16)) * fma2(yy, V(-3.0f), xx);
            }
        }
    }
}

}  // namespace gs3d
