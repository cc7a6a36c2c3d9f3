// Low-rank adapters: which kernel runs, and the products of any rank and alignment on CUDA cores, for what the others do not take (ranks that are no multiple of 2, 4 or 8,
// or more than 256).  No counterpart in the reference; this stands next to its projections
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
        // Tiles of 128 rows on tcgen05 where they are many (us of the warp-level and the tcgen05 kernel, bf16, 4096 x 4096).  Forward: rank 16, 2048 rows 16.6 and 21.1, 2560 24.0 and 22.1,
        // 4096 30.2 and 26.4 (narrow layers have no time to win: 1024 x 1024, 4096 rows 9.6 and 13.1), rank 64, 1024 rows 18.6 and 20.0, 2048 30.4 and 27.8.  Back, with
        // the weights' gradient: rank 16, 512 rows 23.6 and 25.5, 1536 36.4 and 30.8, 4096 79.5 and 65.4; rank 32, 512 26.0 and 27.6, 768 33.5 and 28.9; rank 64, 512 40.9 and 36.4.
        // Adapters whose rows do not fill a good part of a tile stay with the other one: 1024 rows of 32 adapters, rank 32, 14.0 and 21.
        const bool narrow = lora_width(a) <= 2048;
        const int least = backward ? (a.rank <= 16 ? 1152 : a.rank <= 32 ? 768 : 512) : a.rank > 32 ? 1152 : narrow ? 0x7FFFFFFF : 2304;
        if (form == LoraForm::pieces && lora_tile_supported(a, keep, dt) && a.n_rows >= least && a.n_rows >= 48ll * a.n_adapters) return launch_lora_tile(st, a, backward, keep, none, dt);
        return (dt == MTC_F32 ? launch_lora_mma<MTC_F32> : dt == MTC_BF16 ? launch_lora_mma<MTC_BF16> : launch_lora_mma<MTC_F16>)(st, a, backward, keep, none);
    }
    return (dt == MTC_F32 ? launch_any<MTC_F32> : dt == MTC_BF16 ? launch_any<MTC_BF16> : launch_any<MTC_F16>)(st, a, backward, keep, none);
}
}  // namespace mtc
