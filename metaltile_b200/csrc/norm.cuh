// Arguments of the norm kernels (norm.cu) and their launchers.
#pragma once

#include "fp8_codes.cuh"

namespace mtc {

constexpr int kMostNorm = 1 << 30;               // values of a row

struct NormArgs {
    const void *x, *residual, *weight;           // residual: or null
    void *sum, *y;                               // sum: where there is a residual; y: may be null where there are codes
    uint8_t *codes;
    float *scales;
    long long n_rows;
    int K, threads;                              // threads of a row
    float eps;
};
struct NormGradArgs {
    const void *dy, *s, *weight, *dsum;          // dsum: or null
    void *dx;
    float *part;                                 // shares of dw f32[workers][K]
    float2 *rows;                                // 1 / root and the mean of every row (any alignment and length only)
    long long n_rows;
    int K, threads, workers;
    float eps;
};

cudaError_t launch_add_rms_norm(Ctx *ctx, cudaStream_t st, const NormArgs &a, int mode, int dt);
size_t norm_grad_workspace(int sms, long long n_rows, int K, int dt);
cudaError_t launch_norm_grad(Ctx *ctx, cudaStream_t st, NormGradArgs a, void *dweight, void *workspace, int dt);

}  // namespace mtc
