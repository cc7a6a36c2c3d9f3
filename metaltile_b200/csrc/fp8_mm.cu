// Products of e4m3 codes with block scales, any shape and alignment, on CUDA cores:
//   out[m, n] = sum_b xs[m, b] * ws[n / 128, b] * sum_{k in block b} x[m, k] * w[n, k]
// The reference has no 8-bit float product; this stands next to mt_qmm and mt_moe_gather_qmm (crates/metaltile-std/src/mlx/quantized.rs:5040-5065,
// crates/metaltile-std/src/ffai/moe.rs:358-433).  The products of two codes are exact in f32; sums are f32.
#include "fp8.cuh"

namespace mtc {
namespace {

using namespace fp8;

__device__ __forceinline__ float value(uint8_t code) { return from_e4m3x2(code).x; }

// One warp per column n and kRows rows; a lane takes four consecutive values of every block.
constexpr int kRows = 4;
__global__ void __launch_bounds__(256) fp8_mm_generic_kernel(const uint8_t *x, const float *xs, const uint8_t *w, const float *ws,
                                                             const uint32_t *expert_offsets, void *out, int M, int N, int K, int n_experts, int out_dt,
                                                             uint32_t *status) {
    pdl_enter();
    if (expert_offsets && blockIdx.x == 0)
        for (int e = threadIdx.x; e < n_experts; e += blockDim.x)
            if (expert_offsets[e] > expert_offsets[e + 1] || expert_offsets[e + 1] > static_cast<uint32_t>(M)) atomicCAS(status, 0u, 0x901u);
    const int lane = threadIdx.x & 31, kb = blocks(K), nb = blocks(N);
    const long long gw = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const long long tiles = (M + kRows - 1) / kRows;
    if (gw >= tiles * N) return;
    const int n = static_cast<int>(gw % N), m0 = static_cast<int>(gw / N) * kRows;
    for (int i = 0; i < kRows && m0 + i < M; ++i) {
        const int m = m0 + i;
        size_t expert = 0;
        if (expert_offsets) {                    // the first range that holds the row; a row in none is left as it is
            int e = 0;
            while (e < n_experts && !(static_cast<uint32_t>(m) >= expert_offsets[e] && static_cast<uint32_t>(m) < expert_offsets[e + 1])) ++e;
            if (e == n_experts) continue;
            expert = e;
        }
        const uint8_t *wr = w + (expert * N + n) * static_cast<size_t>(K), *xr = x + static_cast<size_t>(m) * K;
        const float *wsr = ws + (expert * nb + n / kBlock) * static_cast<size_t>(kb), *xsr = xs + static_cast<size_t>(m) * kb;
        float acc = 0.0f;
        for (int b = 0; b < kb; ++b) {
            float part = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = b * kBlock + lane * 4 + j;
                if (k < K) part = fmaf(value(xr[k]), value(wr[k]), part);
            }
            acc = fmaf(part, xsr[b] * wsr[b], acc);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
        if (lane == 0) st_from_f32(out, static_cast<size_t>(m) * N + n, acc, out_dt);
    }
}

}  // namespace

cudaError_t launch_fp8_mm_generic(Ctx *ctx, cudaStream_t st, const uint8_t *x, const float *xs, const uint8_t *w, const float *ws, const uint32_t *expert_offsets,
                                  void *out, int M, int N, int K, int n_experts, int out_dt) {
    const long long warps = static_cast<long long>((M + kRows - 1) / kRows) * N, ctas = (warps + 7) / 8;
    if (ctas > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    return launch_pdl(fp8_mm_generic_kernel, static_cast<unsigned>(ctas), 256, 0, st, x, xs, w, ws, expert_offsets, out, M, N, K, n_experts, out_dt,
                      ctx->d_status);
}

}  // namespace mtc
