// Float rows or matrices -> e4m3 codes with an f32 scale for each block of 128 (activations) or 128 x 128 (weights).
// The reference has no 8-bit float format; this stands next to its affine quantizer (crates/metaltile-std/src/mlx/quantized.rs:3629-3667).
//
//   s = max(max |x| / 448, 2^-90) over the finite values of the block (pow2: the least power of two that is not below)
//   code = x / s rounded to the nearest e4m3 value, ties to even; infinities and NaN become NaN
//
// Bound by memory: every value is read once and stays in registers, as it was read, between the maximum and the codes; sixteen lanes share
// a row of a block, eight values a lane.  What matters beside the loads in flight is the number of instructions a value: the maximum is
// that of the bit patterns (two 16-bit values at a time, monotone for all but NaN), and a quotient is one multiplication for 16-bit types
// (factor_of); f32 takes three and three that look whether it may be on a border.  Measured (graph, us): 14336 x 4096 in blocks of 128 x 128
// bf16 and f16 32.3 (176 MB, 5.45 TB/s; as f32 is quantized 46.9), with powers of two 28.1, f32 51.3 (294 MB); 8192 x 4096 rows bf16 23.3
// (31.7), f32 29.5.
#include <algorithm>

#include "fp8.cuh"

namespace mtc {
namespace {

using namespace fp8;

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

constexpr int kThreads = 256, kGroups = kThreads / 16;

// Blocks of 1 x 128.  A CTA has 16 groups of 16 lanes: 2^shift of them side by side in a row, TURNS times, the others in the next rows.
// first: the block of K that the launch starts with.
template <int DT, bool VEC, bool POW2, int TURNS>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const void *x, const uint32_t *rows, uint8_t *codes, float *scales, long long n_rows,
                                                                 long long n_src_rows, int K, int shift, int first, uint32_t *status) {
    pdl_enter();
    const int kb = blocks(K), lane = threadIdx.x & 15, g = threadIdx.x >> 4, wide = 1 << shift;
    const long long r = static_cast<long long>(blockIdx.x) * (kGroups >> shift) + (g >> shift);
    const int b0 = first + blockIdx.y * (wide * TURNS) + (g & (wide - 1));
    const bool row = r < n_rows;
    long long src = row ? r : 0;
    if (rows && row) {
        const uint32_t id = rows[r];
        src = id;
        if (id >= n_src_rows) {
            if (lane == 0 && b0 == 0) atomicCAS(status, 0u, 0x906u);         // an index outside the tensor reads row 0
            src = 0;
        }
    }
    Eight<DT> v[TURNS];
    int n[TURNS];
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
        const int b = b0 + u * wide;
        n[u] = row && b < kb ? K - b * kBlock - lane * 8 : 0;
        v[u].template load<VEC>(x, static_cast<size_t>(src) * K + b * kBlock + lane * 8, n[u]);
    }
    uint32_t m[TURNS];
#pragma unroll
    for (int u = 0; u < TURNS; ++u) m[u] = v[u].most();
    if constexpr (DT != MTC_F32 && TURNS == 2) {                     // both blocks' maxima in one word
        uint32_t both = __vmaxu2(__byte_perm(m[0], m[1], 0x5410), __byte_perm(m[0], m[1], 0x7632));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, o));
        m[0] = both & 0xFFFFu;
        m[1] = both >> 16;
    } else {
#pragma unroll
        for (int u = 0; u < TURNS; ++u)
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) m[u] = larger<DT>(m[u], __shfl_xor_sync(0xffffffffu, m[u], o));
    }
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
        const int b = b0 + u * wide;
        const bool special = has_special<DT>(m[u]);
        float amax = magnitude<DT>(m[u]);
        if (__any_sync(0xffffffffu, special)) {
            float f = v[u].most_finite();
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) f = fmaxf(f, __shfl_xor_sync(0xffffffffu, f, o));
            amax = f;
        }
        bool tie;
        const float s = scale_of(amax, POW2), factor = factor_of<DT, POW2>(s, amax, tie);
        if (lane == 0 && row && b < kb) scales[static_cast<size_t>(r) * kb + b] = s;
        store8<VEC>(codes, static_cast<size_t>(r) * K + b * kBlock + lane * 8, n[u], codes_of<DT, POW2>(v[u], s, factor, tie, special));
    }
}

// Blocks of 128 x 128: a CTA a block, 16 rows at a time.
template <int DT, bool VEC, bool POW2>
__global__ void __launch_bounds__(kThreads) quantize_blocks_kernel(const void *x, uint8_t *codes, float *scales, long long n_rows, int K, int row_blocks) {
    pdl_enter();
    const int kb = blocks(K);
    const uint32_t id = blockIdx.x, b = id % kb, rest = id / kb, rb = rest % row_blocks, mat = rest / row_blocks;      // (matrix, block of rows, block of columns)
    const int lane = threadIdx.x & 15, k0 = b * kBlock + lane * 8;
    const long long r0 = static_cast<long long>(rb) * kBlock + (threadIdx.x >> 4);
    const size_t at = (static_cast<size_t>(mat) * n_rows + r0) * K + k0;
    Eight<DT> v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].template load<VEC>(x, at + static_cast<size_t>(i) * 16 * K, r0 + i * 16 < n_rows ? K - k0 : 0);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = larger<DT>(m, v[i].most());
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = larger<DT>(m, __shfl_xor_sync(0xffffffffu, m, o));
    __shared__ uint32_t most[8];
    __shared__ float most_f[8];
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) m = larger<DT>(m, most[i]);
    const bool special = has_special<DT>(m);                         // the same in all threads
    float amax = magnitude<DT>(m);
    if (special) {
        amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, v[i].most_finite());
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if ((threadIdx.x & 31) == 0) most_f[threadIdx.x >> 5] = amax;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, most_f[i]);
    }
    bool tie;
    const float s = scale_of(amax, POW2), factor = factor_of<DT, POW2>(s, amax, tie);
    if (threadIdx.x == 0) scales[id] = s;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        store8<VEC>(codes, at + static_cast<size_t>(i) * 16 * K, r0 + i * 16 < n_rows ? K - k0 : 0, codes_of<DT, POW2>(v[i], s, factor, tie, special));
}

template <int DT, bool VEC, bool POW2>
cudaError_t launch(Ctx *ctx, cudaStream_t st, const void *x, const uint32_t *rows, uint8_t *codes, float *scales, int n_mats, long long n_rows,
                   long long n_src_rows, int K, int block_rows) {
    const int kb = blocks(K);
    if (block_rows == 1) {
        int shift = 0;
        while (shift < 4 && 1 << shift < kb) ++shift;
        const long long ctas = (n_rows + (kGroups >> shift) - 1) / (kGroups >> shift);
        // two blocks a group, all loads in flight at once, where that leaves every SM its eight CTAs
        const bool two = kb > 16 && ctas * ((kb + 31) / 32) >= 8ll * ctx->sm_count;
        const int wide = (two ? 2 : 1) << shift, most = 65535 * wide;        // blocks of a CTA, of a launch (the grid's second dimension holds no more)
        for (int first = 0; first < kb; first += most) {
            const cudaError_t e = launch_pdl(two ? quantize_rows_kernel<DT, VEC, POW2, 2> : quantize_rows_kernel<DT, VEC, POW2, 1>,
                                             dim3(static_cast<unsigned>(ctas), static_cast<unsigned>((std::min(kb - first, most) + wide - 1) / wide)), kThreads, 0, st, x,
                                             rows, codes, scales, n_rows, n_src_rows, K, shift, first, ctx->d_status);
            if (e != cudaSuccess) return e;
        }
        return cudaSuccess;
    }
    const long long row_blocks = (n_rows + kBlock - 1) / kBlock, ctas = n_mats * row_blocks * kb;
    if (ctas > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    return launch_pdl(quantize_blocks_kernel<DT, VEC, POW2>, static_cast<unsigned>(ctas), kThreads, 0, st, x, codes, scales, n_rows, K, static_cast<int>(row_blocks));
}
template <int DT>
cudaError_t launch(bool vec, bool pow2, Ctx *ctx, cudaStream_t st, const void *x, const uint32_t *rows, uint8_t *codes, float *scales, int n_mats, long long n_rows,
                   long long n_src_rows, int K, int block_rows) {
    auto *f = vec ? (pow2 ? launch<DT, true, true> : launch<DT, true, false>) : (pow2 ? launch<DT, false, true> : launch<DT, false, false>);
    return f(ctx, st, x, rows, codes, scales, n_mats, n_rows, n_src_rows, K, block_rows);
}

}  // namespace

cudaError_t launch_fp8_quantize(Ctx *ctx, cudaStream_t st, const void *x, const uint32_t *rows, uint8_t *codes, float *scales, int n_mats, long long n_rows,
                                long long n_src_rows, int K, int block_rows, int pow2, int dt) {
    const bool vec = K % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 8 == 0;
    return (dt == MTC_F32 ? launch<MTC_F32> : dt == MTC_BF16 ? launch<MTC_BF16> : launch<MTC_F16>)(vec, pow2 != 0, ctx, st, x, rows, codes, scales, n_mats, n_rows,
                                                                                                n_src_rows, K, block_rows);
}

}  // namespace mtc
