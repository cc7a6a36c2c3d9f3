// The balance loss of a mixture-of-experts router, its per-expert counts and the gradient of the logits.  The reference routes
// (crates/metaltile-std/src/ffai/moe.rs:65-192) but has no training side; this stands next to its router.
//
// Over the n counted rows (mask not zero): p_t = softmax(logits_t), a row of minus infinities only has p = 0;
//   c_e = slots of these rows that chose expert e,  f_e = c_e / (n k),  P_e = (1 / n) sum_t p_te
//   loss = coef * E * sum_e f_e P_e;  n = 0: f, P and loss are 0
//   d loss / d logit_te = coef * E / n * p_te * (f_e - sum_j f_j p_tj)       (counts are constants)
//
// Bound by reading the logits: a warp has a row in registers (two at a time while there are many), every lane adds up its own experts over the rows of the warp; rows are
// dealt out to the warps of the grid in turn, so that masked ones, which lie together, are spread.  Sums over rows are f32 in a warp and in its CTA (at most a few dozen
// rows a warp) and f64 from there on, always in the same order; counts are integers, whose order does not matter.  A second launch, a cluster of eight CTAs with an
// eighth of the experts each, adds up the CTAs' parts and meets over distributed shared memory for the loss.
#include <algorithm>

#include "common.cuh"

namespace mtc {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;      // of the gradient

// Expert of slot (chunk c, i) of a lane: (c * 32 + lane) * V + i; V neighbours are one load.
template <int DT, int V>
__device__ __forceinline__ void load_v(const void *base, size_t at, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = ld_written_as_f32(base, at, DT);
    } else if constexpr (DT == MTC_F32) {
        const float4 q = *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
        const uint2 q = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(base) + at);
        const uint32_t u[2] = {q.x, q.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (DT == MTC_BF16) {
                v[2 * i] = __uint_as_float(u[i] << 16);
                v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    }
}
template <int DT, int V>
__device__ __forceinline__ void store_v(void *base, size_t at, const float (&v)[V]) {
    if constexpr (V == 1) {
        st_from_f32(base, at, v[0], DT);
    } else if constexpr (DT == MTC_F32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(base) + at) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        uint32_t u[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (DT == MTC_BF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                u[i] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                u[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(base) + at) = make_uint2(u[0], u[1]);
    }
}

// The logits of a row (minus infinity where there is no expert)
template <int DT, int V, int CH>
__device__ __forceinline__ void load_row(const void *logits, size_t row, int n_experts, float (&z)[CH][V]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int i = 0; i < V; ++i) z[c][i] = -INFINITY;
        const int e = (c * 32 + lane) * V;
        if (e < n_experts) load_v<DT, V>(logits, row * n_experts + e, z[c]);
    }
}
// ... become its probabilities
template <int V, int CH>
__device__ __forceinline__ void softmax_row(float (&z)[CH][V]) {
    float most = -INFINITY;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) most = fmaxf(most, z[c][i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    // exp(z - most) as a power of two; below 2^-126 it is zero
    if (most == -INFINITY) most = 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(z[c][i]) : "f"((z[c][i] - most) * 1.4426950408889634f));
            sum += z[c][i];
        }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) z[c][i] *= inv;
}

// Warps of a CTA that adds up rows: a lane holds two sets of CH x V values, so few warps where that is many registers
__host__ __device__ constexpr int row_warps(int ch, int v) { return ch * v <= 8 ? 32 : 16; }

// Sums of each CTA: part_p f32[grid][E], part_c i32[grid][E], part_n i32[grid]
template <int DT, int V, int CH>
__global__ void __launch_bounds__(32 * row_warps(CH, V)) balance_rows_kernel(const void *logits, const uint32_t *topk_idx, const uint8_t *mask, float *part_p, int *part_c,
                                                                           int *part_n, int n_rows, int n_experts, int k, uint32_t *status) {
    pdl_enter();
    constexpr int W = row_warps(CH, V), T = 32 * W;
    extern __shared__ float sm[];
    float *const warp_p = sm;                                    // [W][E]
    int *const hist = reinterpret_cast<int *>(sm + W * n_experts);
    __shared__ int counted;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e < n_experts; e += T) hist[e] = 0;
    if (threadIdx.x == 0) counted = 0;
    __syncthreads();
    float acc[CH][V] = {};
    int n = 0;
    auto kept = [&](long long r) { return r < n_rows && (!mask || mask[r] != 0); };
    auto count = [&](long long r) {
        ++n;
        for (int j = lane; j < k; j += 32) {
            const uint32_t e = topk_idx[static_cast<size_t>(r) * k + j];
            if (e < static_cast<uint32_t>(n_experts)) atomicAdd(&hist[e], 1);
            else atomicCAS(status, 0u, 0x907u);                  // an expert that does not exist: recorded, not counted
        }
    };
    auto add = [&](const float (&z)[CH][V]) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) acc[c][i] += z[c][i];
    };
    const long long step = static_cast<long long>(gridDim.x) * W;
    for (long long r = static_cast<long long>(warp) * gridDim.x + blockIdx.x; r < n_rows; r += 2 * step) {
        const bool one = kept(r), two = kept(r + step);
        float a[CH][V], b[CH][V];
        if (one) load_row<DT, V, CH>(logits, r, n_experts, a);
        if (two) load_row<DT, V, CH>(logits, r + step, n_experts, b);
        if (one) {
            count(r);
            softmax_row<V, CH>(a);
            add(a);
        }
        if (two) {
            count(r + step);
            softmax_row<V, CH>(b);
            add(b);
        }
    }
    if (lane == 0 && n) atomicAdd(&counted, n);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = (c * 32 + lane) * V + i;
            if (e < n_experts) warp_p[warp * n_experts + e] = acc[c][i];
        }
    __syncthreads();
    for (int e = threadIdx.x; e < n_experts; e += T) {
        float s = 0.0f;
#pragma unroll 8
        for (int w = 0; w < W; ++w) s += warp_p[w * n_experts + e];
        part_p[static_cast<size_t>(blockIdx.x) * n_experts + e] = s;
        part_c[static_cast<size_t>(blockIdx.x) * n_experts + e] = hist[e];
    }
    if (threadIdx.x == 0) part_n[blockIdx.x] = counted;
}

constexpr int kJoinCtas = 8, kJoinThreads = 512;
// A CTA has the experts of its eighth side by side (2^shift of its threads) and as many groups of parts as threads are left.
__global__ void __cluster_dims__(kJoinCtas, 1, 1) __launch_bounds__(kJoinThreads)
balance_join_kernel(const float *part_p, const int *part_c, const int *part_n, int parts, float coef, float *loss, int *counts, float *mean_probs, int *n_counted,
                    int n_experts, int k, int shift) {
    pdl_enter();
    __shared__ double sums[kJoinThreads];
    __shared__ int cnts[kJoinThreads];
    __shared__ int total;
    __shared__ double share;
    const int rank = blockIdx.x, e0 = n_experts * rank / kJoinCtas, e1 = n_experts * (rank + 1) / kJoinCtas;
    const int wide = 1 << shift, groups = kJoinThreads >> shift, g = threadIdx.x >> shift, e = e0 + (threadIdx.x & (wide - 1));
    if (threadIdx.x == 0) total = 0;
    __syncthreads();
    int mine = 0;
    for (int i = threadIdx.x; i < parts; i += kJoinThreads) mine += part_n[i];
    if (mine) atomicAdd(&total, mine);
    double p = 0.0;
    int c = 0;
    if (e < e1) {
#pragma unroll 4
        for (int i = g; i < parts; i += groups) {
            p += part_p[static_cast<size_t>(i) * n_experts + e];
            c += part_c[static_cast<size_t>(i) * n_experts + e];
        }
    }
    sums[threadIdx.x] = p;
    cnts[threadIdx.x] = c;
    for (int o = groups >> 1; o > 0; o >>= 1) {
        __syncthreads();
        if (g < o) {
            sums[threadIdx.x] += sums[threadIdx.x + (o << shift)];
            cnts[threadIdx.x] += cnts[threadIdx.x + (o << shift)];
        }
    }
    __syncthreads();
    const int n = total;
    double term = 0.0;
    if (g == 0 && e < e1) {
        const double mean = n ? sums[threadIdx.x] / n : 0.0;
        counts[e] = cnts[threadIdx.x];
        mean_probs[e] = static_cast<float>(mean);
        term = n ? mean * cnts[threadIdx.x] / (static_cast<double>(n) * k) : 0.0;
    }
    __syncthreads();
    if (g == 0) sums[threadIdx.x] = term;
    for (int o = wide >> 1; o > 0; o >>= 1) {
        __syncthreads();
        if (threadIdx.x < o) sums[threadIdx.x] += sums[threadIdx.x + o];
    }
    if (threadIdx.x == 0) share = sums[0];
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0 && threadIdx.x == 0) {
        double all = 0.0;
        for (int q = 0; q < kJoinCtas; ++q) {
            uint32_t there;
            double v;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(&share))), "r"(q));
            asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(there) : "memory");
            all += v;
        }
        *loss = static_cast<float>(static_cast<double>(coef) * n_experts * all);
        *n_counted = n;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");      // nobody leaves while its share is read
}

template <int DT, int V, int CH>
__global__ void __launch_bounds__(kThreads) balance_grad_kernel(const void *logits, const uint8_t *mask, const int *counts, const int *n_counted,
                                                                const float *grad_loss, float coef, void *grad, int n_rows, int n_experts, int k) {
    pdl_enter();
    const int lane = threadIdx.x & 31, warps = gridDim.x * kWarps;
    const int n = *n_counted;
    const float each = n > 0 ? 1.0f / (static_cast<float>(n) * k) : 0.0f;
    const float g = n > 0 ? (grad_loss ? *grad_loss : 1.0f) * coef * n_experts / n : 0.0f;
    float f[CH][V];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = (c * 32 + lane) * V + i;
            f[c][i] = e < n_experts ? static_cast<float>(counts[e]) * each : 0.0f;
        }
    auto finish = [&](long long r, bool kept, float (&z)[CH][V]) {
        if (kept) {
            softmax_row<V, CH>(z);
            float dot = 0.0f;
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < V; ++i) dot = fmaf(z[c][i], f[c][i], dot);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < V; ++i) z[c][i] = g * z[c][i] * (f[c][i] - dot);
        } else {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < V; ++i) z[c][i] = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e = (c * 32 + lane) * V;
            if (e < n_experts) store_v<DT, V>(grad, static_cast<size_t>(r) * n_experts + e, z[c]);
        }
    };
    for (long long r = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5); r < n_rows; r += 2 * warps) {
        const long long r2 = r + warps;
        const bool one = !mask || mask[r] != 0, two = r2 < n_rows && (!mask || mask[r2] != 0);
        float a[CH][V], b[CH][V];
        if (one) load_row<DT, V, CH>(logits, r, n_experts, a);
        if (two) load_row<DT, V, CH>(logits, r2, n_experts, b);
        finish(r, one, a);
        if (r2 < n_rows) finish(r2, two, b);
    }
}

// CTAs that add up rows: eight rows each at least, so that few rows make few parts
int balance_ctas(int sms, int n_rows) { return std::max(1, std::min(sms, (n_rows + 7) / 8)); }

// The instance that holds a row: four neighbouring experts a load where rows of them are aligned
template <template <int, int, int> class F, int DT, typename... A>
cudaError_t with_form(bool vec, int n_experts, A... args) {
    if (vec) {
        if (n_experts <= 128) return F<DT, 4, 1>::run(args...);
        if (n_experts <= 256) return F<DT, 4, 2>::run(args...);
        return F<DT, 4, 8>::run(args...);
    }
    if (n_experts <= 32) return F<DT, 1, 1>::run(args...);
    if (n_experts <= 64) return F<DT, 1, 2>::run(args...);
    if (n_experts <= 256) return F<DT, 1, 8>::run(args...);
    return F<DT, 1, 32>::run(args...);
}
template <template <int, int, int> class F, typename... A>
cudaError_t with_form(int dt, bool vec, int n_experts, A... args) {
    return dt == MTC_F32 ? with_form<F, MTC_F32>(vec, n_experts, args...)
           : dt == MTC_BF16 ? with_form<F, MTC_BF16>(vec, n_experts, args...) : with_form<F, MTC_F16>(vec, n_experts, args...);
}
template <int DT, int V, int CH>
struct RowsForm {
    static cudaError_t run(Ctx *ctx, cudaStream_t st, int ctas, const void *logits, const uint32_t *idx, const uint8_t *mask, float *pp, int *pc, int *pn, int n_rows,
                           int n_experts, int k) {
        constexpr int W = row_warps(CH, V);
        const size_t smem = static_cast<size_t>(W + 1) * n_experts * 4;
        static PerDeviceAttr attr;
        if (smem > 48 * 1024) {
            const cudaError_t e = attr.set(balance_rows_kernel<DT, V, CH>, static_cast<size_t>(W + 1) * 1024 * 4);
            if (e != cudaSuccess) return e;
        }
        return launch_pdl(balance_rows_kernel<DT, V, CH>, ctas, 32 * W, smem, st, logits, idx, mask, pp, pc, pn, n_rows, n_experts, k, ctx->d_status);
    }
};
template <int DT, int V, int CH>
struct GradForm {
    static cudaError_t run(cudaStream_t st, int ctas, const void *logits, const uint8_t *mask, const int *counts, const int *n_counted, const float *gl, float coef,
                           void *grad, int n_rows, int n_experts, int k) {
        return launch_pdl(balance_grad_kernel<DT, V, CH>, ctas, kThreads, 0, st, logits, mask, counts, n_counted, gl, coef, grad, n_rows, n_experts, k);
    }
};
bool in_fours(int n_experts, int dt, const void *a, const void *b) {
    const uintptr_t align = dt == MTC_F32 ? 16 : 8;
    return n_experts % 4 == 0 && n_experts > 64 && reinterpret_cast<uintptr_t>(a) % align == 0 && reinterpret_cast<uintptr_t>(b) % align == 0;
}

}  // namespace

size_t moe_balance_workspace(int sms, int n_rows, int n_experts) {
    return static_cast<size_t>(balance_ctas(sms, n_rows)) * (2 * static_cast<size_t>(n_experts) + 1) * 4;
}

cudaError_t launch_moe_balance(Ctx *ctx, cudaStream_t st, const void *logits, const uint32_t *topk_idx, const uint8_t *mask, float coef, float *loss,
                               int *counts, float *mean_probs, int *n_counted, int n_rows, int n_experts, int k, int dt, void *workspace) {
    const int ctas = balance_ctas(ctx->sm_count, n_rows);
    float *pp = static_cast<float *>(workspace);
    int *pc = reinterpret_cast<int *>(pp + static_cast<size_t>(ctas) * n_experts), *pn = pc + static_cast<size_t>(ctas) * n_experts;
    cudaError_t e = with_form<RowsForm>(dt, in_fours(n_experts, dt, logits, logits), n_experts, ctx, st, ctas, logits, topk_idx, mask, pp, pc, pn, n_rows, n_experts, k);
    if (e != cudaSuccess) return e;
    int shift = 0;
    while (1 << shift < (n_experts + kJoinCtas - 1) / kJoinCtas) ++shift;
    return launch_pdl(balance_join_kernel, kJoinCtas, kJoinThreads, 0, st, pp, pc, pn, ctas, coef, loss, counts, mean_probs, n_counted, n_experts, k, shift);
}

cudaError_t launch_moe_balance_grad(Ctx *ctx, cudaStream_t st, const void *logits, const uint8_t *mask, const int *counts, const int *n_counted,
                                    const float *grad_loss, float coef, void *grad, int n_rows, int n_experts, int k, int dt) {
    if (n_rows <= 0) return cudaSuccess;
    const int ctas = std::min(ctx->sm_count * 8, (n_rows + kWarps - 1) / kWarps);
    return with_form<GradForm>(dt, in_fours(n_experts, dt, logits, grad), n_experts, st, ctas, logits, mask, counts, n_counted, grad_loss, coef, grad, n_rows,
                               n_experts, k);
}

}  // namespace mtc
