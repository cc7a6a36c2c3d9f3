// Low-rank adapters of many requests beside a shared projection: what the kernels (lora.cu) share, and their launchers.
//   rows of one adapter stand together in `order` (row numbers, a permutation); adapter e has the places offsets[e] <= p < offsets[e + 1]
//   forward   h_t = x_t A_e^T [rank]      out_t = base_t + scale_e h_t B_e^T
//   backward  u_t = dy_t B_e  [rank]      dx_t  = base_t + scale_e u_t A_e      dA_e = scale_e sum_t u_t x_t      dB_e = scale_e sum_t dy_t h_t
#pragma once

#include "common.cuh"

namespace mtc {

constexpr int kMostRank = 1024, kMostAdapters = 65536;

// One of the two directions: rows [n_rows, c_in] -> low [n_rows, rank] -> rows [n_rows, c_out]
struct LoraArgs {
    const void *in, *down, *up;                  // forward: x, a, b; backward: dy, b, a
    const uint32_t *order, *offsets;
    const float *scales;                         // null: 1
    const void *base;                            // null: 0; may be out
    void *out;
    float *low;                                  // f32[n_rows, rank], where it is kept: h, or u
    int n_rows, c_in, c_out, rank, n_adapters;
    uint32_t *status;
};
// dw[e][i][c] (a) or dw[e][c][i] (b) = scale_e sum over the rows of e of low[t][i] * in[t][c]
struct LoraWeight {
    const void *in;
    const float *low;
    void *grad;
    int c;
};
struct LoraWeights {
    LoraWeight a, b;                             // of a: (x, u); of b: (dy, h)
    const uint32_t *order, *offsets;
    const float *scales;
    int n_rows, rank, n_adapters;
    uint32_t *status;
};

// keep: `low` is wanted; all: with zeros for the rows of no adapter
cudaError_t launch_lora(Ctx *ctx, cudaStream_t st, const LoraArgs &a, bool backward, bool keep, bool all, int dt);

// The tensor-core kernels (lora_mma.cu, lora_grad.cu) and what they take; `none`: rows of no adapter have something to be written
enum class LoraForm { none, values, pieces };    // rows of any length, or of whole 16-byte pieces
LoraForm lora_mma_form(const LoraArgs &a, bool backward, int dt);
cudaError_t launch_lora_mma(cudaStream_t st, const LoraArgs &a, bool backward, bool keep, bool none, int dt);
bool lora_tile_supported(const LoraArgs &a, bool keep, int dt);       // (lora_tcgen05.cu) what of the above it takes
cudaError_t launch_lora_tile(cudaStream_t st, const LoraArgs &a, bool backward, bool keep, bool none, int dt);
// (lora_grad.cu) any size and alignment
cudaError_t launch_lora_grad(Ctx *ctx, cudaStream_t st, const LoraWeights &w, int dt);

}  // namespace mtc
