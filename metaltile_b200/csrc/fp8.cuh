// e4m3 codes with an f32 scale for each block of 128 values: what the quantizer and the products share.
//   activations  codes u8[M, K], scales f32[M, ceil(K/128)]                  (blocks of 1 x 128)
//   weights      codes u8[N, K], scales f32[ceil(N/128), ceil(K/128)]        (blocks of 128 x 128)
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace mtc {
namespace fp8 {

constexpr int kBlock = 128;
constexpr float kLeastScale = 8.077935669463161e-28f;      // 2^-90: below it the residual of a quotient could underflow (code_quotient)

constexpr int kMostSize = 0x7FFFFFFF - 1024;    // of rows and columns: what is rounded up to a tile stays an int

__host__ __device__ constexpr int blocks(int n) { return (n + kBlock - 1) / kBlock; }

// two codes; lo in the low byte.  |v| above 448 becomes 448, NaN the code 0x7F.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t codes) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(codes)));
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

// The scale of a block with this largest magnitude: amax / 448 correctly rounded, by Markstein's theorem (P. W. Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", IBM J. Res. Develop. 34(1), 1990): with y the reciprocal of b correctly
// rounded and q within a unit of a / b, the remainder r = a - q b is exact in one fma, and q + r y is a / b correctly rounded.  Here b =
// 448 and y is a constant.  tests/test_fp8_division_gpu.py compares all 2^23 mantissas; a division takes 120 instructions.  (Where r would
// be below the least number of f32, the quotient is far below 2^-90.)
__device__ __forceinline__ float scale_of(float amax, int pow2) {
    constexpr float r = 1.0f / 448.0f;
    const float q = amax * r;
    float s = fmaxf(fmaf(fmaf(-q, 448.0f, amax), r, q), kLeastScale);
    if (pow2) s = __uint_as_float((__float_as_uint(s) + 0x7FFFFFu) & 0xFF800000u);
    return s;
}
// 1 / s, within a unit or two; exact where s is a power of two (s is never subnormal, nor is this)
__device__ __forceinline__ float inverse_of(float s) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    return r;
}

// x / s within a unit: the same step, from a reciprocal within a unit or two
__device__ __forceinline__ float quotient(float x, float s, float inv) {
    const float r = x * inv;
    return fmaf(fmaf(-r, s, x), inv, r);
}
// ... such that rounding it to a code gives the code nearest to the true quotient.  A quotient rounded to f32 may land on the border
// between two codes that the true one lies beside (with s = amax / 448 rounded that is one value in a few hundred, since x and amax have
// few bits), so it is rounded to odd: its exact remainder tells the side, and an even result is moved there.  Borders are even numbers, so
// none is hit unless the quotient is exact.  Below 2^-11 every quotient becomes zero anyway.
__device__ __forceinline__ float odd_quotient(float x, float s, float r) {       // r: quotient()
    const float rest = fmaf(-r, s, x);
    const uint32_t b = __float_as_uint(r), away = (__float_as_uint(rest) ^ b) >> 31;       // 1: the true one is smaller in magnitude
    return rest != 0.0f && !(b & 1u) && fabsf(r) >= 4.8828125e-4f ? __uint_as_float(b + 1u - 2u * away) : r;
}
__device__ __forceinline__ float code_quotient(float x, float s, float inv) {
    return fabsf(x) < INFINITY ? odd_quotient(x, s, quotient(x, s, inv)) : __int_as_float(0x7FC00000);        // infinities have no code: NaN, as NaN is
}

}  // namespace fp8

// Launchers
cudaError_t launch_fp8_quantize(Ctx *ctx, cudaStream_t st, const void *x, const uint32_t *rows, uint8_t *codes, float *scales, int n_mats,
                                long long n_rows, long long n_src_rows, int K, int block_rows, int pow2, int dt);
cudaError_t launch_fp8_mm_generic(Ctx *ctx, cudaStream_t st, const uint8_t *x, const float *xs, const uint8_t *w, const float *ws, const uint32_t *expert_offsets,
                                  void *out, int M, int N, int K, int n_experts, int out_dt);
bool fp8_tile_supported(int M, int N, int K, int n_experts, const void *x, const void *w);
cudaError_t launch_fp8_tile(Ctx *ctx, cudaStream_t st, const uint8_t *x, const float *xs, const uint8_t *w, const float *ws, const uint32_t *expert_offsets, void *out,
                            int M, int N, int K, int n_experts, int out_dt, std::string *why);
bool fp8_pair_supported(int M, int N, int K, int n_experts, const void *x, const void *w);
cudaError_t launch_fp8_pair(Ctx *ctx, cudaStream_t st, const uint8_t *x, const float *xs, const uint8_t *w, const float *ws, const uint32_t *expert_offsets, void *out,
                            int M, int N, int K, int n_experts, int out_dt, std::string *why);
size_t moe_balance_workspace(int sms, int n_rows, int n_experts);
cudaError_t launch_moe_balance(Ctx *ctx, cudaStream_t st, const void *logits, const uint32_t *topk_idx, const uint8_t *mask, float coef, float *loss,
                               int *counts, float *mean_probs, int *n_counted, int n_rows, int n_experts, int k, int dt, void *workspace);
cudaError_t launch_moe_balance_grad(Ctx *ctx, cudaStream_t st, const void *logits, const uint8_t *mask, const int *counts, const int *n_counted,
                                    const float *grad_loss, float coef, void *grad, int n_rows, int n_experts, int k, int dt);

}  // namespace mtc
