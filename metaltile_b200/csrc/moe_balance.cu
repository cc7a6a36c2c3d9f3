// The balance loss of a mixture-of-experts router, its per-expert counts and the gradient of the logits.  The reference routes
// (crates/metaltile-std/src/ffai/moe.rs:65-192) but has no training side; this stands next to its router.
//
// Over the n counted rows (mask not zero): p_t = softmax(logits_t), a row of minus infinities only has p = 0;
//   c_e = slots of these rows that chose expert e,  f_e = c_e / (n k),  P_e = (1 / n) sum_t p_te
//   loss = coef * E * sum_e f_e P_e;  n = 0: f, P and loss are 0
//   d loss / d logit_te = coef * E / n * p_te * (f_e - sum_j f_j p_tj)       (counts are constants)
//
// Bound by reading the logits where there are many rows, by launches and latencies where there are few.  A warp has two or four rows in
// registers at a time, every lane adds up its own experts over the rows of the warp; rows are dealt out to the warps of the grid in turn,
// so that masked ones, which lie together, are spread.  Sums over rows are f32 for 32 rows of a warp at most and f64 from there on, always
// in the same order; counts are integers, whose order does not matter.  Few rows are one launch, a cluster of eight CTAs that meet over
// distributed shared memory; many are a launch of a CTA an SM and one of such a cluster that adds up their parts.
#include <algorithm>
#include <type_traits>

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

// The logits of a row, minus infinity where there is no expert or (there: false) no row
template <int DT, int V, int CH>
__device__ __forceinline__ void load_row(const void *logits, size_t row, bool there, int n_experts, float (&z)[CH][V]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int i = 0; i < V; ++i) z[c][i] = -INFINITY;
        const int e = (c * 32 + lane) * V;
        if (there && e < n_experts) load_v<DT, V>(logits, row * n_experts + e, z[c]);
    }
}
// Which of the next 32 rows of a warp (r0, r0 + step, ...) count: a bit each, so that no load of logits waits for the mask's
// (65536 x 128 bf16 17.5 -> 16.0 us; in the gradient it was 3 % at 128 experts and -4 % at 256, and is left out)
__device__ __forceinline__ uint32_t kept_rows(const uint8_t *mask, long long r0, long long step, int n_rows) {
    const long long r = r0 + (threadIdx.x & 31) * step;
    return __ballot_sync(0xffffffffu, r < n_rows && (!mask || mask[r] != 0));
}
// ... of the first N of R rows become their probabilities, the steps of the rows side by side
template <int N, int V, int CH, int R>
__device__ __forceinline__ void softmax_rows(float (&z)[R][CH][V]) {
    float most[N], sum[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        float m = -INFINITY;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) m = fmaxf(m, z[u][c][i]);
        asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(most[u]) : "f"(m));
    }
    // exp(z - most) as a power of two; below 2^-126 it is zero.  The product is rounded, so that a probability errs by 1.5 |z - most| 2^-24
    // of itself and the two units of ex2: more the smaller it is, of the size of what the rounding of f32 logits' difference costs, and next
    // to nothing for those that make up the sums.
#pragma unroll
    for (int u = 0; u < N; ++u) {
        if (most[u] == -INFINITY) most[u] = 0.0f;
        sum[u] = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(z[u][c][i]) : "f"((z[u][c][i] - most[u]) * 1.4426950408889634f));
                sum[u] += z[u][c][i];
            }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int u = 0; u < N; ++u) sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], o);
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const float inv = sum[u] == 0.0f ? 0.0f : 1.0f / sum[u];
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) z[u][c][i] *= inv;
    }
}

constexpr int kCluster = 8;
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t on_cta(const void *p, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
    return r;
}
__device__ __forceinline__ double ld_double(uint32_t at) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ int ld_int(uint32_t at) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

struct Results {
    float coef;
    float *loss;
    int *counts;
    float *mean_probs;
    int *n_counted;
};
// What comes of the sums of an expert (thread e - e0 of a CTA of the cluster has that of expert e, `mine`: it has one), and of all: the
// loss.  scratch: a double a warp and one more.
__device__ __forceinline__ void conclude(const Results &out, int rank, bool mine, int e, double p, int c, int n, int n_experts, int k, double *scratch) {
    double term = 0.0;
    if (mine) {
        const double mean = n ? p / n : 0.0;
        out.counts[e] = c;
        out.mean_probs[e] = static_cast<float>(mean);
        term = n ? mean * c / (static_cast<double>(n) * k) : 0.0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) term += __shfl_xor_sync(0xffffffffu, term, o);
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = term;
    __syncthreads();
    if (threadIdx.x == 0) {
        double all = 0.0;
        for (int w = 0; w < warps; ++w) all += scratch[w];
        scratch[warps] = all;
    }
    cluster_sync();
    if (rank == 0 && threadIdx.x == 0) {
        double all = 0.0;
        for (int q = 0; q < kCluster; ++q) all += ld_double(on_cta(scratch + warps, q));
        *out.loss = static_cast<float>(static_cast<double>(out.coef) * n_experts * all);
        *out.n_counted = n;
    }
    cluster_sync();                              // nobody leaves while its share is read
}

// Warps of a CTA that adds up rows: a lane holds so many rows' values and their sums, so few warps where that is many registers
__host__ __device__ constexpr int row_warps(int ch, int v) { return ch * v <= 8 ? 32 : 16; }

// Sums of each CTA: part_p f64[grid][E], part_c i32[grid][E], part_n i32[grid]; ONE: the grid is a cluster that goes on to the results
template <int DT, int V, int CH, bool ONE>
__global__ void __launch_bounds__(32 * row_warps(CH, V)) balance_rows_kernel(const void *logits, const uint32_t *topk_idx, const uint8_t *mask, double *part_p, int *part_c,
                                                                           int *part_n, Results out, int n_rows, int n_experts, int k, uint32_t *status) {
    pdl_enter();
    constexpr int W = row_warps(CH, V), T = 32 * W, R = CH * V <= 4 ? 4 : 2;
    extern __shared__ double sm[];
    constexpr int ROW = 32 * CH * V;             // a warp's sums: those of a lane under each other, so that no bank is met twice
    auto place = [](int e) { return (e / (32 * V) * V + e % V) * 32 + e / V % 32; };
    double *const warp_p = sm;                                   // [W][ROW]
    int *const hist = reinterpret_cast<int *>(sm + W * ROW);
    __shared__ int counted;
    __shared__ double scratch[W + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e < n_experts; e += T) hist[e] = 0;
    if (threadIdx.x == 0) counted = 0;
    __syncthreads();
    float acc[CH][V] = {};
    int n = 0, held = 0;
    bool first = true;
    auto flush = [&] {                           // a lane has its own places
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                double &at = warp_p[warp * ROW + (c * V + i) * 32 + lane];
                at = first ? static_cast<double>(acc[c][i]) : at + acc[c][i];
                acc[c][i] = 0.0f;
            }
        first = false;
        held = 0;
    };
    const long long step = static_cast<long long>(gridDim.x) * W;
    uint32_t keep = 0;
    int known = 0;
    for (long long r0 = static_cast<long long>(warp) * gridDim.x + blockIdx.x; r0 < n_rows; r0 += R * step) {
        bool kept[R];
        float z[R][CH][V];
        uint32_t id[R];                          // a lane a slot (k <= 32)
        if (known == 0) keep = kept_rows(mask, r0, step, n_rows), known = 32;
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const long long r = r0 + u * step;
            kept[u] = keep >> u & 1u;
            load_row<DT, V, CH>(logits, r, kept[u], n_experts, z[u]);
            id[u] = kept[u] && lane < k ? topk_idx[static_cast<size_t>(r) * k + lane] : 0;
        }
#pragma unroll
        for (int u = 0; u < R; ++u) {
            if (!kept[u]) continue;
            ++n;
            if (lane < k) {
                if (id[u] < static_cast<uint32_t>(n_experts)) atomicAdd(&hist[id[u]], 1);
                else atomicCAS(status, 0u, 0x907u);              // an expert that does not exist: recorded, not counted
            }
        }
        auto add = [&](auto rows) {
            constexpr int N = decltype(rows)::value;
            softmax_rows<N>(z);
#pragma unroll
            for (int u = 0; u < N; ++u)
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int i = 0; i < V; ++i) acc[c][i] += z[u][c][i];
        };
        if (r0 + step < n_rows) add(std::integral_constant<int, R>{});       // (a masked row adds zeros)
        else add(std::integral_constant<int, 1>{});
        keep >>= R;
        known -= R;
        if ((held += R) >= 32) flush();
    }
    flush();
    if (lane == 0 && n) atomicAdd(&counted, n);
    __syncthreads();
    for (int e = threadIdx.x; e < n_experts; e += T) {
        double s = 0.0;
#pragma unroll 8
        for (int w = 0; w < W; ++w) s += warp_p[w * ROW + place(e)];
        if constexpr (ONE) {
            warp_p[place(e)] = s;
        } else {
            part_p[static_cast<size_t>(blockIdx.x) * n_experts + e] = s;
            part_c[static_cast<size_t>(blockIdx.x) * n_experts + e] = hist[e];
        }
    }
    if constexpr (ONE) {
        cluster_sync();
        const int rank = blockIdx.x, e = n_experts * rank / kCluster + threadIdx.x;
        const bool mine = e < n_experts * (rank + 1) / kCluster;
        double p = 0.0;
        int c = 0, all = 0;
#pragma unroll
        for (int q = 0; q < kCluster; ++q) {
            all += ld_int(on_cta(&counted, q));
            if (mine) {
                p += ld_double(on_cta(warp_p + place(e), q));
                c += ld_int(on_cta(hist + e, q));
            }
        }
        conclude(out, rank, mine, e, p, c, all, n_experts, k, scratch);
    } else if (threadIdx.x == 0) {
        part_n[blockIdx.x] = counted;
    }
}

constexpr int kJoinThreads = 512;
// A CTA has the experts of its eighth side by side (2^shift of its threads) and as many groups of parts as threads are left.
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kJoinThreads)
balance_join_kernel(const double *part_p, const int *part_c, const int *part_n, int parts, Results out, int n_experts, int k, int shift) {
    pdl_enter();
    __shared__ double sums[kJoinThreads], scratch[kJoinThreads / 32 + 1];
    __shared__ int cnts[kJoinThreads];
    __shared__ int total;
    const int rank = blockIdx.x, e0 = n_experts * rank / kCluster, e1 = n_experts * (rank + 1) / kCluster;
    const int wide = 1 << shift, groups = kJoinThreads >> shift, g = threadIdx.x >> shift, e = e0 + (threadIdx.x & (wide - 1));
    if (threadIdx.x == 0) total = 0;
    __syncthreads();
    int mine = 0;
    for (int i = threadIdx.x; i < parts; i += kJoinThreads) mine += part_n[i];
    if (mine) atomicAdd(&total, mine);
    double p = 0.0;
    int c = 0;
    if (e < e1) {
#pragma unroll 8
        for (int i = g; i < parts; i += groups) {            // (eight parts in flight)
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
    conclude(out, rank, g == 0 && e < e1, e, sums[threadIdx.x], cnts[threadIdx.x], total, n_experts, k, scratch);
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
    constexpr int R = 2;
    for (long long r0 = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5); r0 < n_rows; r0 += R * warps) {
        float z[R][CH][V], dot[R];
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const long long r = r0 + u * warps;
            load_row<DT, V, CH>(logits, r, r < n_rows && (!mask || mask[r] != 0), n_experts, z[u]);
        }
        auto finish = [&](auto rows) {
            constexpr int N = decltype(rows)::value;
            softmax_rows<N>(z);                  // (a masked row: zeros)
#pragma unroll
            for (int u = 0; u < N; ++u) {
                dot[u] = 0.0f;
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int i = 0; i < V; ++i) dot[u] = fmaf(z[u][c][i], f[c][i], dot[u]);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                for (int u = 0; u < N; ++u) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], o);
#pragma unroll
            for (int u = 0; u < N; ++u)
#pragma unroll
                for (int c = 0; c < CH; ++c) {
#pragma unroll
                    for (int i = 0; i < V; ++i) z[u][c][i] = g * z[u][c][i] * (f[c][i] - dot[u]);
                    const int e = (c * 32 + lane) * V;
                    if (e < n_experts) store_v<DT, V>(grad, static_cast<size_t>(r0 + u * warps) * n_experts + e, z[u][c]);
                }
        };
        if (r0 + warps < n_rows) finish(std::integral_constant<int, R>{});
        else finish(std::integral_constant<int, 1>{});
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
    template <bool ONE>
    static cudaError_t go(Ctx *ctx, cudaStream_t st, int ctas, const void *logits, const uint32_t *idx, const uint8_t *mask, double *pp, int *pc, int *pn, const Results &out,
                          int n_rows, int n_experts, int k) {
        constexpr int W = row_warps(CH, V);
        const size_t smem = static_cast<size_t>(W) * 32 * CH * V * 8 + static_cast<size_t>(n_experts) * 4;
        static PerDeviceAttr attr;
        const cudaError_t e = attr.set(balance_rows_kernel<DT, V, CH, ONE>, static_cast<size_t>(2 * W + 1) * 32 * CH * V * 4);
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(ctas);
        cfg.blockDim = dim3(32 * W);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cudaLaunchAttribute la[2];
        la[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        la[0].val.programmaticStreamSerializationAllowed = 1;
        la[1].id = cudaLaunchAttributeClusterDimension;
        la[1].val.clusterDim.x = kCluster;
        la[1].val.clusterDim.y = la[1].val.clusterDim.z = 1;
        cfg.attrs = la;
        cfg.numAttrs = ONE ? 2 : 1;
        return cudaLaunchKernelEx(&cfg, balance_rows_kernel<DT, V, CH, ONE>, logits, idx, mask, pp, pc, pn, out, n_rows, n_experts, k, ctx->d_status);
    }
    static cudaError_t run(bool one, Ctx *ctx, cudaStream_t st, int ctas, const void *logits, const uint32_t *idx, const uint8_t *mask, double *pp, int *pc, int *pn,
                           const Results &out, int n_rows, int n_experts, int k) {
        return one ? go<true>(ctx, st, kCluster, logits, idx, mask, pp, pc, pn, out, n_rows, n_experts, k)
                   : go<false>(ctx, st, ctas, logits, idx, mask, pp, pc, pn, out, n_rows, n_experts, k);
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

// One launch up to here (128 experts, us: 64 rows 6.3 in one and 6.8 in two, 256 6.6 and 6.8, 512 7.5 and 7.2, 1024 9.3 and 7.5)
static bool in_one(int n_rows) { return n_rows <= 256; }

size_t moe_balance_workspace(int sms, int n_rows, int n_experts) {
    return in_one(n_rows) ? 0 : static_cast<size_t>(balance_ctas(sms, n_rows)) * (12 * static_cast<size_t>(n_experts) + 4);
}

cudaError_t launch_moe_balance(Ctx *ctx, cudaStream_t st, const void *logits, const uint32_t *topk_idx, const uint8_t *mask, float coef, float *loss,
                               int *counts, float *mean_probs, int *n_counted, int n_rows, int n_experts, int k, int dt, void *workspace) {
    const int ctas = balance_ctas(ctx->sm_count, n_rows);
    double *pp = static_cast<double *>(workspace);
    int *pc = reinterpret_cast<int *>(pp + static_cast<size_t>(ctas) * n_experts), *pn = pc + static_cast<size_t>(ctas) * n_experts;
    const Results out{coef, loss, counts, mean_probs, n_counted};
    const bool one = in_one(n_rows);
    cudaError_t e = with_form<RowsForm>(dt, in_fours(n_experts, dt, logits, logits), n_experts, one, ctx, st, ctas, logits, topk_idx, mask, pp, pc, pn, out, n_rows, n_experts, k);
    if (e != cudaSuccess || one) return e;
    int shift = 0;
    while (1 << shift < (n_experts + kCluster - 1) / kCluster) ++shift;
    return launch_pdl(balance_join_kernel, kCluster, kJoinThreads, 0, st, pp, pc, pn, ctas, out, n_experts, k, shift);
}

cudaError_t launch_moe_balance_grad(Ctx *ctx, cudaStream_t st, const void *logits, const uint8_t *mask, const int *counts, const int *n_counted,
                                    const float *grad_loss, float coef, void *grad, int n_rows, int n_experts, int k, int dt) {
    if (n_rows <= 0) return cudaSuccess;
    const int ctas = std::min(ctx->sm_count * 8, (n_rows + kWarps - 1) / kWarps);
    return with_form<GradForm>(dt, in_fours(n_experts, dt, logits, grad), n_experts, st, ctas, logits, mask, counts, n_counted, grad_loss, coef, grad, n_rows,
                               n_experts, k);
}

}  // namespace mtc
