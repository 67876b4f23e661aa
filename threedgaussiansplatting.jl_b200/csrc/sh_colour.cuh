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

}  // namespace gs3d
