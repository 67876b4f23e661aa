// mx4_colour.cuh — the colours of Gaussians whose SH coefficients are 4-bit rows, of one Gaussian (V:
// float) or of two side by side in packed fp32 (V: Float2).
#pragma once
#include "mx4.cuh"
#include "sh_colour.cuh"

namespace gs3d {

// 4-bit SH rows as a colour source: row i, or row indices[i].
struct Mx4Sh {
    const uint8_t* codes;
    const uint8_t* scales;
    const float* tensor_scale;
    const int32_t* indices;
    int64_t rows;
    int code_bytes, blocks;
};

inline Mx4Sh mx4_sh_source(const gs3d_mx4_rows* sh, const int32_t* indices) {
    return Mx4Sh{sh->codes, sh->scales, sh->tensor_scale, indices, sh->rows, mx4_code_bytes(sh->dim),
                 mx4_blocks(sh->dim, sh->format)};
}

// Whether ShRow can load the rows: exactly the rendered degree, codes aligned for its loads.
inline bool mx4_sh_whole(const gs3d_mx4_rows* sh, int degree) {
    return sh->dim == 3 * (degree + 1) * (degree + 1) &&
           reinterpret_cast<uintptr_t>(sh->codes) % (degree == 3 ? 8 : 2) == 0;
}

// The 4-bit row of a Gaussian in registers: words of eight codes, and the block scales' bytes. Rows of
// exactly the rendered degree, their codes aligned to 8 bytes at degree 3 (24 bytes a row) and to 2
// below (2, 6 and 14 bytes).
template <int DEG, int FMT>
struct ShRow {
    static constexpr int DIM = 3 * (DEG + 1) * (DEG + 1), CB = (DIM + 1) / 2, NW = (CB + 3) / 4;
    static constexpr int BS = Mx4Block<FMT>::size, NB = (DIM + BS - 1) / BS;
    uint32_t w[NW], scale[NB];

    __device__ __forceinline__ void load(const Mx4Sh& a, int64_t r) {
        if (r < 0) {  // no row: zero codes with zero scales
#pragma unroll
            for (int k = 0; k < NW; ++k) w[k] = 0;
#pragma unroll
            for (int b = 0; b < NB; ++b) scale[b] = 0;
            return;
        }
        if constexpr (DEG == 3) {
            const uint2* p = reinterpret_cast<const uint2*>(a.codes + r * CB);
#pragma unroll
            for (int k = 0; k < NW / 2; ++k) {
                const uint2 v = __ldg(p + k);
                w[2 * k] = v.x;
                w[2 * k + 1] = v.y;
            }
        } else {
            const uint16_t* p = reinterpret_cast<const uint16_t*>(a.codes + r * CB);
#pragma unroll
            for (int k = 0; k < NW; ++k) {
                // the last word may be half: what is doubled then lies behind the row's end
                const uint32_t lo = __ldg(p + 2 * k), hi = 4 * k + 2 < CB ? __ldg(p + 2 * k + 1) : lo;
                w[k] = lo | (hi << 16);
            }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) scale[b] = __ldg(a.scales + r * NB + b);
    }
};

template <typename V>
struct Lanes;
template <>
struct Lanes<float> {
    static constexpr int n = 1;
    static __device__ __forceinline__ void set(float& v, int, float x) { v = x; }
};
template <>
struct Lanes<Float2> {
    static constexpr int n = 2;
    static __device__ __forceinline__ void set(Float2& v, int lane, float x) { (lane ? v.y : v.x) = x; }
};

// Elements 8 k .. 8 k + 7 of the rows, times 2^-14.
template <typename V, int DEG, int FMT>
__device__ __forceinline__ void decode_word(const ShRow<DEG, FMT>* s, int k, V* h) {
#pragma unroll
    for (int l = 0; l < Lanes<V>::n; ++l) {
        __half2 e[4];
        e2m1_word_half(s[l].w[k], e);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 v = __half22float2(e[j]);
            Lanes<V>::set(h[j], l, v.x);
            Lanes<V>::set(h[j + 4], l, v.y);
        }
    }
}

// Block scale * tensor scale of every block of the rows.
template <typename V, int DEG, int FMT>
__device__ __forceinline__ void block_factors(const ShRow<DEG, FMT>* s, float g, V (&factor)[ShRow<DEG, FMT>::NB]) {
#pragma unroll
    for (int l = 0; l < Lanes<V>::n; ++l)
#pragma unroll
        for (int b = 0; b < ShRow<DEG, FMT>::NB; ++b) Lanes<V>::set(factor[b], l, mx4_scale<FMT>(s[l].scale[b]) * g);
}

__device__ __forceinline__ float at_least_zero(float c) { return c < 0.0f ? 0.0f : c; }
__device__ __forceinline__ Float2 at_least_zero(Float2 c) { return Float2(at_least_zero(c.x), at_least_zero(c.y)); }

// 1/2 + the channel's products with the basis, clamped at 0. WHOLE: h are elements times 2^-14, and what
// lies in one block is summed before its factor multiplies it; else h are the coefficients.
template <typename V, int DEG, int FMT, bool WHOLE>
__device__ __forceinline__ V mx4_channel(int ch, const V* h, const V* factor, const V* basis) {
    constexpr int NC = (DEG + 1) * (DEG + 1), BS = Mx4Block<FMT>::size;
    V c(0.5f);
    if constexpr (WHOLE) {
        const int b0 = ch * NC / BS, b1 = ((ch + 1) * NC - 1) / BS;
#pragma unroll
        for (int b = b0; b <= b1; ++b) {
            const int k0 = max(b * BS - ch * NC, 0), k1 = min((b + 1) * BS - ch * NC, NC);
            V s = basis[k0] * h[k0];
#pragma unroll
            for (int k = k0 + 1; k < k1; ++k) s = fma2(basis[k], h[k], s);
            c = fma2(s * V(0x1p14f), factor[b], c);
        }
    } else {
#pragma unroll
        for (int k = 0; k < NC; ++k) c = fma2(basis[k], h[k], c);
    }
    return at_least_zero(c);
}

// The rows r (-1: zeros): elements and block factors, or (not WHOLE) the coefficients.
template <typename V, int DEG, int FMT, bool WHOLE>
__device__ __forceinline__ void load_sh(const Mx4Sh& a, int order, const int64_t (&r)[Lanes<V>::n], float g,
                                        V (&h)[(3 * (DEG + 1) * (DEG + 1) + 7) / 8 * 8],
                                        V (&factor)[ShRow<DEG, FMT>::NB]) {
    constexpr int NC = (DEG + 1) * (DEG + 1);
    if constexpr (WHOLE) {
        ShRow<DEG, FMT> s[Lanes<V>::n];
#pragma unroll
        for (int l = 0; l < Lanes<V>::n; ++l) s[l].load(a, r[l]);
        block_factors<V, DEG, FMT>(s, g, factor);
#pragma unroll
        for (int k = 0; k < ShRow<DEG, FMT>::NW; ++k) decode_word<V, DEG, FMT>(s, k, h + 8 * k);
    } else {
        constexpr int BS = Mx4Block<FMT>::size;
#pragma unroll
        for (int l = 0; l < Lanes<V>::n; ++l)
#pragma unroll
            for (int c = 0; c < 3; ++c)
#pragma unroll
                for (int k = 0; k < NC; ++k) {
                    const int e = c * order + k;
                    float x = 0.0f;
                    if (r[l] >= 0) {
                        const Mx4Decode<FMT> d(a.scales[r[l] * a.blocks + e / BS], g);
                        const float2 v = mx4_value(d, e2m1_pair_half(a.codes[r[l] * a.code_bytes + e / 2]));
                        x = e & 1 ? v.y : v.x;
                    }
                    Lanes<V>::set(h[c * NC + k], l, x);
                }
    }
}

// Row of Gaussian i, -1 where its index names none.
__device__ __forceinline__ int64_t sh_row(const Mx4Sh& a, int64_t i) {
    if (!a.indices) return i;
    const int64_t r = (int64_t)__ldg(a.indices + i) - 1;
    return r < a.rows && r >= 0 ? r : -1;
}

// The colours seen from p: the three channels. At degree 3 a channel is decoded when it is summed, so
// that 16 coefficients of a Gaussian are live and not 48.
template <typename V, int DEG, int FMT, bool WHOLE>
__device__ __forceinline__ void mx4_colour(const Mx4Sh& a, int order, const int64_t (&r)[Lanes<V>::n], float g,
                                           const float* p, V mx, V my, V mz, V (&c)[3]) {
    constexpr int NC = (DEG + 1) * (DEG + 1);
    V basis[NC], factor[ShRow<DEG, FMT>::NB];
    if constexpr (WHOLE && DEG == 3) {
        ShRow<DEG, FMT> s[Lanes<V>::n];
#pragma unroll
        for (int l = 0; l < Lanes<V>::n; ++l) s[l].load(a, r[l]);
        sh_basis_fused<DEG>(p, mx, my, mz, basis);
        block_factors<V, DEG, FMT>(s, g, factor);
#pragma unroll
        for (int ch = 0; ch < 3; ++ch) {
            V h[16];
            decode_word<V, DEG, FMT>(s, 2 * ch, h);
            decode_word<V, DEG, FMT>(s, 2 * ch + 1, h + 8);
            c[ch] = mx4_channel<V, DEG, FMT, WHOLE>(ch, h, factor, basis);
        }
    } else {
        V h[(3 * NC + 7) / 8 * 8];
        load_sh<V, DEG, FMT, WHOLE>(a, order, r, g, h, factor);
        sh_basis_fused<DEG>(p, mx, my, mz, basis);
#pragma unroll
        for (int ch = 0; ch < 3; ++ch) c[ch] = mx4_channel<V, DEG, FMT, WHOLE>(ch, h + ch * NC, factor, basis);
    }
}

}  // namespace gs3d
