// Eight neighbouring values of a row and their e4m3 codes: what the quantizer and the norm with an 8-bit result share.
#pragma once

#include "fp8.cuh"

namespace mtc {
namespace fp8 {

// Eight neighbouring values of a row as they were read
template <int DT>
struct Eight {
    uint32_t w[DT == MTC_F32 ? 8 : 4];

    // `n` of them exist; VEC: all or none do, and they start at a 16-byte boundary
    template <bool VEC>
    __device__ __forceinline__ void load(const void *base, size_t at, int n) {
        constexpr int W = DT == MTC_F32 ? 8 : 4;
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = 0;
        if constexpr (VEC) {
            if (n <= 0) return;
            const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const char *>(base) + at * (DT == MTC_F32 ? 4 : 2));
#pragma unroll
            for (int i = 0; i < W / 4; ++i) {
                const uint4 q = p[i];
                w[4 * i] = q.x, w[4 * i + 1] = q.y, w[4 * i + 2] = q.z, w[4 * i + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i >= n) break;
                if constexpr (DT == MTC_F32) w[i] = static_cast<const uint32_t *>(base)[at + i];
                else w[i / 2] |= static_cast<uint32_t>(static_cast<const uint16_t *>(base)[at + i]) << (i & 1) * 16;
            }
        }
    }
    // The largest magnitude as a bit pattern (16-bit types: of either half); infinities and NaN are above all others.
    __device__ __forceinline__ uint32_t most() const {
        uint32_t m = 0;
        if constexpr (DT == MTC_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
        }
        return m;
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (DT == MTC_F32) return __uint_as_float(w[i]);
        const uint32_t u = w[i / 2];
        if constexpr (DT == MTC_BF16) return __uint_as_float(i & 1 ? u & 0xFFFF0000u : u << 16);
        return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? u >> 16 : u)));
    }
    // ... over the finite values only, as an f32
    __device__ __forceinline__ float most_finite() const {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = fabsf(value(i));
            if (a < INFINITY) m = fmaxf(m, a);
        }
        return m;
    }
};

template <int DT>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    if constexpr (DT == MTC_F32) return max(a, b);
    else return __vmaxu2(a, b);
}
// of a pattern that `larger` left: is there an infinity or a NaN, and the magnitude otherwise
template <int DT>
__device__ __forceinline__ bool has_special(uint32_t m) {
    if constexpr (DT == MTC_F32) return m >= 0x7F800000u;
    else return max(m & 0xFFFFu, m >> 16) >= (DT == MTC_BF16 ? 0x7F80u : 0x7C00u);
}
template <int DT>
__device__ __forceinline__ float magnitude(uint32_t m) {
    if constexpr (DT == MTC_F32) return __uint_as_float(m);
    const uint32_t h = max(m & 0xFFFFu, m >> 16);
    if constexpr (DT == MTC_BF16) return __uint_as_float(h << 16);
    return __half2float(__ushort_as_half(static_cast<unsigned short>(h)));
}

// What a block's values are multiplied with, so that a code is one multiplication and the conversion.  16-bit types: with x = X 2^a and amax
// = A 2^b (X, A below 2^11) a border between codes is B 2^c, B < 32, and 448 x / amax is either such a border or differs from it by at
// least 1 / (A B) > 2^-16 of it: 7 X and A B, times powers of two, are whole numbers.  So an error of 2^-20 changes no code but that of a
// value on a border, and these all lie on the same side, that on which s lies of amax / 448: `factor` is moved there by 2^-21, which is
// more than its own and the product's rounding.  Where s is amax / 448 exactly, or 2^-90, they are ties: `tie` has the product rounded to
// 18 bits, which leaves nothing but the border itself there.
template <int DT, bool POW2>
__device__ __forceinline__ float factor_of(float s, float amax, bool &tie) {
    const float inv = inverse_of(s);
    tie = false;
    if constexpr (POW2 || DT == MTC_F32) return inv;
    const float rest = fmaf(-s, 448.0f, amax);                       // exact
    tie = rest == 0.0f || s == kLeastScale;
    return tie ? inv : inv * (rest > 0.0f ? 1.0f + 0x1p-21f : 1.0f - 0x1p-21f);
}

// Eight codes.  special: infinities or NaN may be among the values.
template <int DT, bool POW2>
__device__ __forceinline__ uint2 codes_of(const Eight<DT> &v, float s, float factor, bool tie, bool special) {
    uint32_t c[4];
    if (!special) {
        float q[8];
        if constexpr (POW2 || DT != MTC_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = v.value(i) * factor;  // POW2: exact (or far below the least code)
            if (tie) {
#pragma unroll
                for (int i = 0; i < 8; ++i) q[i] = __uint_as_float((__float_as_uint(q[i]) + 32u) & ~63u);
            }
        } else {
            // Borders between codes are the numbers of exactly five bits, and below the least normal code the odd multiples of 2^-10: only
            // there can it matter on which side of its f32 the quotient is (code_quotient).
            float least = INFINITY;
            int border = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                q[i] = quotient(v.value(i), s, factor);
                border = min(border, static_cast<int>(__float_as_uint(q[i]) << 12));
                least = fminf(least, fabsf(q[i]));
            }
            if (border == static_cast<int>(0x80000000u) || least < 0.015625f) {
#pragma unroll
                for (int i = 0; i < 8; ++i) q[i] = odd_quotient(v.value(i), s, q[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = to_e4m3x2(q[2 * i], q[2 * i + 1]);
        return make_uint2(__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[2], c[3], 0x5410));
    }
    const float inv = inverse_of(s);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = to_e4m3x2(code_quotient(v.value(2 * i), s, inv), code_quotient(v.value(2 * i + 1), s, inv));
    return make_uint2(__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[2], c[3], 0x5410));
}
template <bool VEC>
__device__ __forceinline__ void store8(uint8_t *codes, size_t at, int n, uint2 c) {
    if constexpr (VEC) {
        if (n > 0) *reinterpret_cast<uint2 *>(codes + at) = c;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) codes[at + i] = static_cast<uint8_t>((i < 4 ? c.x : c.y) >> (i & 3) * 8);
    }
}

}  // namespace fp8
}  // namespace mtc
