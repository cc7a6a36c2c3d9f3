// Low-rank adapters: any type, size and alignment, on CUDA cores.  No counterpart in the reference; this stands next to its projections
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

// low[t][i] by a warp.  The weights' value of (i, c) lies at i * si + c * sc of an adapter.
template <int DT>
__global__ void __launch_bounds__(256) lora_low_kernel(const LoraArgs a, long long si, long long sc, bool all) {
    pdl_enter();
    check_offsets(a.offsets, a.n_adapters, a.n_rows, a.status);
    const int lane = threadIdx.x & 31;
    const long long item = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (item >= static_cast<long long>(a.n_rows) * a.rank) return;
    const uint32_t p = static_cast<uint32_t>(item / a.rank), i = static_cast<uint32_t>(item % a.rank), t = a.order[p];
    if (!row_ok(t, a.n_rows, a.status)) return;
    const int e = owner(a.offsets, a.n_adapters, p);
    if (e == a.n_adapters && !all) return;
    float acc = 0.0f;
    if (e < a.n_adapters) {
        const size_t x = static_cast<size_t>(t) * a.c_in, w = static_cast<size_t>(e) * a.rank * a.c_in + i * si;
        for (int c = lane; c < a.c_in; c += 32) acc = fmaf(ld_written_as_f32(a.in, x + c, DT), ld_written_as_f32(a.down, w + c * sc, DT), acc);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    }
    if (lane == 0) a.low[static_cast<size_t>(t) * a.rank + i] = acc;
}

// out[t][c] by a thread
template <int DT>
__global__ void __launch_bounds__(256) lora_out_kernel(const LoraArgs a, long long si, long long sc) {
    pdl_enter();
    const long long ctas_a_row = (a.c_out + 255) / 256;
    const uint32_t p = static_cast<uint32_t>(blockIdx.x / ctas_a_row), t = a.order[p];
    const long long c = blockIdx.x % ctas_a_row * 256 + threadIdx.x;
    if (c >= a.c_out || t >= static_cast<uint32_t>(a.n_rows)) return;
    const int e = owner(a.offsets, a.n_adapters, p);
    const size_t at = static_cast<size_t>(t) * a.c_out + c;
    float acc = 0.0f;
    if (e < a.n_adapters) {
        const size_t w = static_cast<size_t>(e) * a.rank * a.c_out + c * sc;
        for (int i = 0; i < a.rank; ++i) acc = fmaf(a.low[static_cast<size_t>(t) * a.rank + i], ld_written_as_f32(a.up, w + i * si, DT), acc);
        if (a.scales) acc *= a.scales[e];
    } else if (a.base == a.out) {
        return;                                  // a row of no adapter stays as it is
    }
    if (a.base) acc += ld_written_as_f32(a.base, at, DT);
    st_from_f32(a.out, at, acc, DT);
}

// A value of a weight's gradient by a thread; sums of 64 rows, then of these
template <int DT>
__global__ void __launch_bounds__(256) lora_weight_kernel(const LoraWeights w, bool of_a) {
    pdl_enter();
    const LoraWeight &g = of_a ? w.a : w.b;
    const long long each = static_cast<long long>(w.rank) * g.c;
    for (long long id = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; id < each * w.n_adapters; id += static_cast<long long>(gridDim.x) * 256) {
        const int e = static_cast<int>(id / each);
        const long long v = id % each;
        const int i = static_cast<int>(of_a ? v / g.c : v % w.rank), c = static_cast<int>(of_a ? v % g.c : v / w.rank);
        const uint32_t from = min(w.offsets[e], static_cast<uint32_t>(w.n_rows)), to = min(w.offsets[e + 1], static_cast<uint32_t>(w.n_rows));
        float sum = 0.0f;
        for (uint32_t p0 = from; p0 < to; p0 += 64) {
            float acc = 0.0f;
            for (uint32_t p = p0; p < min(p0 + 64, to); ++p) {
                const uint32_t t = w.order[p];
                if (t < static_cast<uint32_t>(w.n_rows))
                    acc = fmaf(g.low[static_cast<size_t>(t) * w.rank + i], ld_written_as_f32(g.in, static_cast<size_t>(t) * g.c + c, DT), acc);
            }
            sum += acc;
        }
        st_from_f32(g.grad, id, w.scales ? sum * w.scales[e] : sum, DT);
    }
}

template <int DT>
cudaError_t launch_any(cudaStream_t st, const LoraArgs &a, bool backward, bool all) {
    const long long low = (static_cast<long long>(a.n_rows) * a.rank + 7) / 8, high = static_cast<long long>(a.n_rows) * ((a.c_out + 255) / 256);
    if (low > 0x7FFFFFFF || high > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    // a [rank][K], b [N][rank]
    cudaError_t e = launch_pdl(lora_low_kernel<DT>, dim3(static_cast<unsigned>(low)), 256, 0, st, a, backward ? 1ll : static_cast<long long>(a.c_in),
                               backward ? static_cast<long long>(a.rank) : 1ll, all);
    if (e != cudaSuccess) return e;
    return launch_pdl(lora_out_kernel<DT>, dim3(static_cast<unsigned>(high)), 256, 0, st, a, backward ? static_cast<long long>(a.c_out) : 1ll,
                      backward ? 1ll : static_cast<long long>(a.rank));
}
template <int DT>
cudaError_t launch_weights_any(cudaStream_t st, const LoraWeights &w) {
    for (int of_a = 1; of_a >= 0; --of_a) {
        const long long values = static_cast<long long>(w.rank) * (of_a ? w.a.c : w.b.c) * w.n_adapters;
        const cudaError_t e = launch_pdl(lora_weight_kernel<DT>, dim3(static_cast<unsigned>(std::min<long long>((values + 255) / 256, 1 << 20))), 256, 0, st, w, of_a != 0);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t launch_lora(Ctx *, cudaStream_t st, const LoraArgs &a, bool backward, bool keep, bool all, int dt) {
    if (lora_mma_supported(a)) {
        const bool none = (keep && all) || a.base != a.out;
        // Tiles of 128 rows on tcgen05 where they are many (us of the warp-level and the tcgen05 kernel, bf16, 4096 x 4096).  Forward: rank 16, 1024 rows 10.7 and 15.1, 2048 21.2 and
        // 20.8, 4096 39 and 26; rank 32, 1024 13.9 and 16.1, 2048 26 and 23; rank 64, 512 14.5 and 19.7, 1024 26 and 20.  Back (with the weights' gradients, which are the
        // same): rank 16, 1024 30.4 and 29.3, 2048 52 and 46; rank 32, 512 34.6 and 35.8, 1024 49 and 38; rank 64, 256 25.5 and 27.8, 512 57 and 52.  Adapters with fewer rows than
        // fill a good part of a tile stay with the other one: 1024 rows of 32 adapters, rank 32, 14.0 and 21.
        const int least = backward ? (a.rank <= 16 ? 2048 : a.rank <= 32 ? 1024 : 512) : a.rank <= 32 ? 2048 : 1024;
        if (lora_tile_supported(a, keep, dt) && a.n_rows >= least && a.n_rows >= 48ll * a.n_adapters) return launch_lora_tile(st, a, backward, keep, none, dt);
        return launch_lora_mma(st, a, backward, keep, none, dt);
    }
    return (dt == MTC_F32 ? launch_any<MTC_F32> : dt == MTC_BF16 ? launch_any<MTC_BF16> : launch_any<MTC_F16>)(st, a, backward, keep && all);
}
cudaError_t launch_lora_weights(Ctx *ctx, cudaStream_t st, const LoraWeights &w, int dt) {
    if (lora_grad_supported(w)) return launch_lora_grad(ctx, st, w, dt);
    return (dt == MTC_F32 ? launch_weights_any<MTC_F32> : dt == MTC_BF16 ? launch_weights_any<MTC_BF16> : launch_weights_any<MTC_F16>)(st, w);
}

}  // namespace mtc
