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

inline bool lora_on_16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
// Rows on a side that can be loaded 16 bytes at a time: x and, forward, a; base and out and, back, a
inline bool lora_pieces_in(const LoraArgs &a) { return a.c_in % 8 == 0 && lora_on_16(a.in) && lora_on_16(a.down); }
inline bool lora_pieces_out(const LoraArgs &a) { return a.c_out % 8 == 0 && lora_on_16(a.up) && lora_on_16(a.out) && (!a.base || lora_on_16(a.base)); }
// What a row has on both sides (each may be near 2^31)
inline long long lora_width(const LoraArgs &a) { return static_cast<long long>(a.c_in) + a.c_out; }

// Warp-level tensor cores (lora_rows.cuh, a file a type); `none`: rows of no adapter have something to be written
template <int DT>
cudaError_t launch_lora_mma(cudaStream_t st, const LoraArgs &a, bool backward, bool keep, bool none);
// tcgen05 (lora_tcgen05.cu), and what it takes of rows of whole pieces
bool lora_tile_supported(const LoraArgs &a, bool keep, int dt);
cudaError_t launch_lora_tile(cudaStream_t st, const LoraArgs &a, bool backward, bool keep, bool none, int dt);
// (lora_grad.cu) any size and alignment
cudaError_t launch_lora_grad(Ctx *ctx, cudaStream_t st, const LoraWeights &w, int dt);

}  // namespace mtc
