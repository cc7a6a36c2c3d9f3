// Low-rank adapters: which kernel runs, and the products of any rank and alignment on CUDA cores, for what the others do not take: ranks above 256, above 16 and no multiple of 8, above 8 and
// no multiple of 4, odd, 2 and 6 beside rows of no whole pieces, and weights along the rank that do not start at 16 bytes.  A CTA has one row and reads its whole adapter: far from what the
// others do where rows are many (us, bf16, 4096 x 4096: 64 rows of rank 20 41 where rank 24 takes 7, 4096 rows 335 and
// back 393 where rank 24 takes 29 and 82, 2048 rows of rank 512 17,700 where rank 256 takes 139).  No counterpart in the reference; this stands next to its projections
// (crates/metaltile-std/src/mlx/quantized.rs:5040-5065), whose quantized weights stay as they are while adapters are trained or swapped.
#include <algorithm>

#include "lora.cuh"

namespace mtc {
namespace {

// The adapter of place p, n_adapters for none.  Offsets that run backwards name some adapter or none (and are reported).
__device__ __forceinline__ int owner(const uint32_t *offsets, int n_adapters, uint32_t p) {
    if (p < offsets[0]) return n_adapters;
    int lo = 0, hi = n_adapters;                 // offsets[lo] <= p; hi: n_adapters or offsets[hi] > p
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid] <= p) lo = mid;
        else hi = mid;
    }
    return p < offsets[lo + 1] ? lo : n_adapters;
}
__device__ __forceinline__ void check_offsets(const uint32_t *offsets, int n_adapters, int n_rows, uint32_t *status) {
    if (blockIdx.x != 0 || blockIdx.y != 0) return;
    for (int e = threadIdx.x; e < n_adapters; e += blockDim.x)
        if (offsets[e] > offsets[e + 1] || offsets[e + 1] > static_cast<uint32_t>(n_rows)) atomicCAS(status, 0u, 0x901u);
}
__device__ __forceinline__ bool row_ok(uint32_t t, int n_rows, uint32_t *status) {
    if (t < static_cast<uint32_t>(n_rows)) return true;
    atomicCAS(status, 0u, 0x908u);               // a row that does not exist: recorded, left out
    return false;
}

// A row a CTA: its h by warps, in shared memory, then its columns.  The weights' value of rank i and column c lies at i * down_i + c * down_c (up_i, up_c) of an adapter.
template <int DT>
__global__ void __launch_bounds__(256) lora_any_kernel(const LoraArgs a, long long down_i, long long down_c, long long up_i, long long up_c, bool keep, bool none) {
    pdl_enter();
    __shared__ float low[kMostRank];
    check_offsets(a.offsets, a.n_adapters, a.n_rows, a.status);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t p = blockIdx.x, t = a.order[p];
    if (!row_ok(t, a.n_rows, a.status)) return;
    const int e = owner(a.offsets, a.n_adapters, p);
    const bool has = e < a.n_adapters;
    if (!has && !none) return;                   // a row of no adapter stays as it is
    const size_t in = static_cast<size_t>(t) * a.c_in, out = static_cast<size_t>(t) * a.c_out, down = static_cast<size_t>(e) * a.rank * a.c_in,
                 up = static_cast<size_t>(e) * a.rank * a.c_out;
    for (int i = warp; i < a.rank; i += 8) {
        float acc = 0.0f;
        if (has) {
            for (int c = lane; c < a.c_in; c += 32) acc = fmaf(ld_written_as_f32(a.in, in + c, DT), ld_written_as_f32(a.down, down + i * down_i + c * down_c, DT), acc);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
        }
        if (lane == 0) {
            low[i] = acc;
            if (keep) a.low[static_cast<size_t>(t) * a.rank + i] = acc;
        }
    }
    __syncthreads();
    if (!has && a.base == a.out) return;
    const float scale = has && a.scales ? a.scales[e] : 1.0f;
    for (int c = threadIdx.x; c < a.c_out; c += 256) {
        float acc = 0.0f;
        if (has)
            for (int i = 0; i < a.rank; ++i) acc = fmaf(low[i], ld_written_as_f32(a.up, up + i * up_i + c * up_c, DT), acc);
        acc *= scale;
        if (a.base) acc += ld_written_as_f32(a.base, out + c, DT);
        st_from_f32(a.out, out + c, acc, DT);
    }
}

template <int DT>
cudaError_t launch_any(cudaStream_t st, const LoraArgs &a, bool backward, bool keep, bool none) {
    const long long in = a.c_in, out = a.c_out, rank = a.rank;           // a [rank][K], b [N][rank]
    return backward ? launch_pdl(lora_any_kernel<DT>, dim3(a.n_rows), 256, 0, st, a, 1ll, rank, out, 1ll, keep, none)
                    : launch_pdl(lora_any_kernel<DT>, dim3(a.n_rows), 256, 0, st, a, in, 1ll, 1ll, rank, keep, none);
}

enum class LoraForm { none, values, pieces };    // of rows of any length, or of whole 16-byte pieces
// Loads of 2, 4 or 8 values along the rank, of the weights that lie so (b): their rows are aligned where the rank is a multiple of that
LoraForm lora_mma_form(const LoraArgs &a, bool backward) {
    const bool pieces = lora_pieces_in(a) && lora_pieces_out(a);
    const int step = a.rank <= 8 && pieces ? 2 : a.rank <= 16 ? 4 : 8;              // (the least size of the rank of a form with values is 16)
    if (a.rank % step || a.rank > 256 || !lora_on_16(backward ? a.down : a.up)) return LoraForm::none;
    return pieces ? LoraForm::pieces : LoraForm::values;
}

}  // namespace

cudaError_t launch_lora(Ctx *, cudaStream_t st, const LoraArgs &a, bool backward, bool keep, bool all, int dt) {
    const LoraForm form = lora_mma_form(a, backward);
    const bool none = (keep && all) || a.base != a.out;
    if (form != LoraForm::none) {
        // Tiles of 128 rows on tcgen05 where they are many.  us of the warp-level and the tcgen05 kernel, bf16, rows of one adapter, three sets of inputs in turn:
        //   forward, 4096 + 4096   rank 16: 2200 rows 18.6 and 23.1, 2304 26.9 and 23.2, 4096 30.5 and 27.4; rank 32: 2200 21.2 and 25.1, 2304 31.1 and 25.2; rank 64: 1100 19.2 and 21.3,
        //                          1152 28.2 and 21.2, 2048 32.8 and 29.2
        //            2048 + 2048   rank 16: 2304 15.2 and 15.4, 4096 17.9 and 18.5; rank 32: 2304 19.1 and 17.2; rank 64: 1100 12.4 and 14.4, 1152 18.3 and 14.4, 4096 31.7 and 22.8
        //            1024 + 1024   rank 16: 4096 10.3 and 13.8; rank 32: 4096 11.5 and 14.6 (`narrow`); rank 64: 1152 13.7 and 11.0, 2048 13.7 and 14.8, 4096 19.3 and 17.2
        //   back, with the weights' gradient
        //            4096 + 4096   rank 16: 1024 31.6 and 29.0, 1160 40.8 and 30.8, 4096 78.4 and 68.2; rank 32: 768 25.8 and 28.8, 1024 38.9 and 39.9, 1150 48.2 and 42.6; rank 64: 448 35.7 and
        //                          37.3, 512 35.0 and 34.3, 1024 61.7 and 54.5
        //            2048 + 2048   rank 16: 1024 20.4 and 23.4, 1160 24.6 and 25.3, 4096 45.4 and 40.6; rank 32: 768 20.6 and 22.6, 1024 24.1 and 23.9; rank 64: 512 29.3 and 27.4
        //            1024 + 1024   rank 16: 1160 21.3 and 21.3, 4096 35.1 and 33.4; rank 32: 768 18.5 and 17.2, 1024 18.6 and 20.6, 1150 23.9 and 21.9; rank 64: 448 26.7 and 23.3, 512 24.6 and 20.6
        // (The warp-level kernel's steps at 1152 and 2304 rows are those of its tiles of 16 and 32 rows.)  Adapters whose rows do not fill a good part of a tile stay with it: 1024 rows of 32
        // adapters, rank 32, forward 21.3 and 23.7.  The number of rows and of adapters is all that the host knows: adapters that have no rows count as if they had their share.
        const bool narrow = lora_width(a) <= 2048;
        const int least = backward ? (a.rank <= 16 ? 1152 : a.rank <= 32 ? 1024 : 512) : a.rank > 32 ? 1152 : narrow ? 0x7FFFFFFF : 2304;
        if (form == LoraForm::pieces && lora_tile_supported(a, keep, dt) && a.n_rows >= least && a.n_rows >= 48ll * a.n_adapters) return launch_lora_tile(st, a, backward, keep, none, dt);
        return (dt == MTC_F32 ? launch_lora_mma<MTC_F32> : dt == MTC_BF16 ? launch_lora_mma<MTC_BF16> : launch_lora_mma<MTC_F16>)(st, a, backward, keep, none);
    }
    return (dt == MTC_F32 ? launch_any<MTC_F32> : dt == MTC_BF16 ? launch_any<MTC_BF16> : launch_any<MTC_F16>)(st, a, backward, keep, none);
}
}  // namespace mtc
