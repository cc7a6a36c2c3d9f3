// Residual addition and root-mean-square norm in front of a projection, with results in the type of the activations or as e4m3 codes, and the
// gradients.  The reference norms one row inside a projection (crates/metaltile-std/src/ffai/rms_norm_qgemv.rs:51-107); these take any number
// of rows, and the codes are those that the products of 8-bit floats read.
//
//   s = T(x + residual),  inv = 1 / sqrt(mean(s^2) + eps),  y = T(s inv w), or its codes
//   ds = inv (w dy - n mean(w dy n)) + dsum  with n = s inv,  dw = sum over rows of dy n
//
// Bound by memory: every value is read once and stays in the registers of the row's threads, eight neighbours a thread and turn, between the sum
// over the row and the results.  Sums are f32 within a row and within the rows that a CTA adds up for dw, f64 over the CTAs, always in the same
// order.  The codes are made from the f32 results: the rounding to T between a norm and a quantizer of its own does not happen here.  Against results in 64 bits some 1.5 codes of
// 10000 are the neighbour: quotients of few bits lie on the borders between codes, and the f32 rounding of y or of the scale decides on which side.
// Measured (graph, three sets of inputs in turn, us): y, 1 x 4096 bf16 2.1, 2048 x 4096 12.8 (67 MB, 5.2 TB/s), 8192 x 4096 42; codes, 8192 x 4096 43.6 (236 MB, 5.4 TB/s;
// bound by instructions, 73 % of the issue slots: 18 a value and some 250 a thread and row); gradients, 8192 x 4096 with dsum 50 (268 MB, 5.4 TB/s; of it the join of 296 shares
// about 3), 333 x 2880 f32 8.3.
// Less near to the memory: gradients of 8193 to 16,384 values, whose four turns of sums do not fit the registers (220 bytes of a thread are spilled, 430 in f32): 4096 x 14336 bf16 115 us where the
// bytes need 54; rows of no whole 16-byte pieces, values one by one and read twice, by the gradient three times: 2048 x 4095 bf16 y 55, codes 48, gradients 50 (of 4096 values 13, 16, 16); rows past
// 16,384 values, read twice: 2048 x 20000 bf16 82, 110, 249 (the bytes need 50, 44, 37).
#include <algorithm>

#include "norm.cuh"

namespace mtc {
namespace {

using namespace fp8;

template <int DT>
__device__ __forceinline__ Eight<DT> packed(const float (&v)[8]) {
    Eight<DT> r;
    if constexpr (DT == MTC_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == MTC_BF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                r.w[i] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                r.w[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
    }
    return r;
}
template <int DT, bool VEC>
__device__ __forceinline__ void store(void *base, size_t at, int n, const Eight<DT> &v) {
    if constexpr (VEC) {
        if (n <= 0) return;
        uint4 *p = reinterpret_cast<uint4 *>(static_cast<char *>(base) + at * (DT == MTC_F32 ? 4 : 2));
        p[0] = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
        if constexpr (DT == MTC_F32) p[1] = make_uint4(v.w[4], v.w[5], v.w[6], v.w[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i >= n) break;
            if constexpr (DT == MTC_F32) static_cast<uint32_t *>(base)[at + i] = v.w[i];
            else static_cast<uint16_t *>(base)[at + i] = static_cast<uint16_t>(v.w[i / 2] >> (i & 1) * 16);
        }
    }
}
template <int DT>
__device__ __forceinline__ Eight<DT> plus(const Eight<DT> &a, const Eight<DT> &b) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = a.value(i) + b.value(i);
    return packed<DT>(v);
}

// Sums over the threads of a row (all of a CTA but where a row is one warp).  scratch: N floats a warp.
template <int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float *scratch, bool one_warp) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (one_warp) return;
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) scratch[i * 32 + warp] = v[i];
    if (warps <= 8) {                            // few parts: every thread adds them up (five more exchanges are 130 cycles)
        if (warp == 0 && lane >= warps && lane < 8)
#pragma unroll
            for (int i = 0; i < N; ++i) scratch[i * 32 + lane] = 0.0f;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float4 a = *reinterpret_cast<const float4 *>(scratch + i * 32), b = *reinterpret_cast<const float4 *>(scratch + i * 32 + 4);
            v[i] = ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
        }
        return;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float s = lane < warps ? scratch[i * 32 + lane] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        v[i] = s;
    }
}

__device__ __forceinline__ float inverse_root(float sum, int K, float eps) { return 1.0f / sqrtf(sum / static_cast<float>(K) + eps); }

// MODE 0: y; 1, 2: codes with scales (2: powers of two), and y where it is wanted.  NV: turns whose values stay in registers (0: any number,
// the row is read again).  A row's threads: a warp (several rows a CTA), or the CTA.
template <int DT, bool VEC, int NV, int MODE>
__global__ void __launch_bounds__(NV == 4 ? 256 : 1024, NV == 4 && MODE ? 4 : 1) add_norm_kernel(const NormArgs a) {
    pdl_enter();
    __shared__ __align__(16) float scratch[32];
    const bool one_warp = a.threads == 32;
    const int t = one_warp ? threadIdx.x & 31 : threadIdx.x, K = a.K;
    const long long row = one_warp ? static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    const size_t at = static_cast<size_t>(row) * K;
    const bool there = row < a.n_rows;
    const int turns = NV ? NV : (K + a.threads * 8 - 1) / (a.threads * 8);
    auto first = [&](int u) { return (u * a.threads + t) * 8; };
    auto count = [&](int u) { return there ? K - first(u) : 0; };

    Eight<DT> s[NV ? NV : 1], w[NV ? NV : 1];
    float sum[1] = {0.0f};
    auto squares = [&](const Eight<DT> &v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[0] = fmaf(v.value(i), v.value(i), sum[0]);
    };
    if constexpr (NV > 0) {
        Eight<DT> r[NV];
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            s[u].template load<VEC>(a.x, at + first(u), count(u));
            if (a.residual) r[u].template load<VEC>(a.residual, at + first(u), count(u));
        }
#pragma unroll
        for (int u = 0; u < NV; ++u) w[u].template load<VEC>(a.weight, first(u), count(u));
        if (a.residual) {
#pragma unroll
            for (int u = 0; u < NV; ++u) {
                s[u] = plus<DT>(s[u], r[u]);
                store<DT, VEC>(a.sum, at + first(u), count(u), s[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < NV; ++u) squares(s[u]);
    } else {
        for (int u = 0; u < turns; ++u) {
            s[0].template load<VEC>(a.x, at + first(u), count(u));
            if (a.residual) {
                Eight<DT> r;
                r.template load<VEC>(a.residual, at + first(u), count(u));
                s[0] = plus<DT>(s[0], r);
                store<DT, VEC>(a.sum, at + first(u), count(u), s[0]);
            }
            squares(s[0]);
        }
    }
    row_sums(sum, scratch, one_warp);
    const float inv = inverse_root(sum[0], K, a.eps);

    auto finish = [&](int u, const Eight<DT> &sv, const Eight<DT> &wv) {
        const int n = count(u);
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = sv.value(i) * inv * wv.value(i);
        if (MODE == 0 || a.y) store<DT, VEC>(a.y, at + first(u), n, packed<DT>(y));
        if constexpr (MODE != 0) {
            // sixteen threads share a block of 128; what lies behind the row counts as zero, whatever its norm is
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (VEC ? n <= 0 : i >= n) y[i] = 0.0f;
            const Eight<MTC_F32> v = packed<MTC_F32>(y);
            float amax = 0.0f;                   // (a NaN stays one)
#pragma unroll
            for (int i = 0; i < 8; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(amax) : "f"(fabsf(y[i])));
            uint32_t most = __float_as_uint(amax);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            const bool special = has_special<MTC_F32>(most);
            amax = __uint_as_float(most);
            if (__any_sync(0xffffffffu, special)) {
                float f = v.most_finite();
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) f = fmaxf(f, __shfl_xor_sync(0xffffffffu, f, o));
                amax = f;
            }
            bool tie;
            const float scale = scale_of(amax, MODE == 2), factor = factor_of<MTC_F32, MODE == 2>(scale, amax, tie);
            const int block = first(u) / kBlock;
            if ((t & 15) == 0 && there && block < blocks(K)) a.scales[static_cast<size_t>(row) * blocks(K) + block] = scale;
            store8<VEC>(a.codes, at + first(u), n, codes_of<MTC_F32, MODE == 2>(v, scale, factor, tie, special));
        }
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int u = 0; u < NV; ++u) finish(u, s[u], w[u]);
    } else {
        for (int u = 0; u < turns; ++u) {        // a thread reads what it wrote itself, or x once more
            s[0].template load<VEC>(a.residual ? a.sum : a.x, at + first(u), count(u));
            w[0].template load<VEC>(a.weight, first(u), count(u));
            finish(u, s[0], w[0]);
        }
    }
}

// ds of every row, and a CTA's (or warp's) share of dw in registers over its rows: part f32[workers][K].
// The next row is requested before the sums of this one where registers allow it (two turns of 16-bit values, one of f32); so are the weights held.
template <int DT, int NV>
__global__ void __launch_bounds__(512) norm_grad_kernel(const NormGradArgs a) {
    pdl_enter();
    constexpr bool AHEAD = DT != MTC_F32 ? NV <= 2 : NV == 1, WEIGHTS = DT != MTC_F32 ? NV <= 2 : NV == 1;
    __shared__ __align__(16) float scratch[2][64];
    const bool one_warp = a.threads == 32;
    const int t = one_warp ? threadIdx.x & 31 : threadIdx.x, K = a.K;
    const long long worker = one_warp ? static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    auto first = [&](int u) { return (u * a.threads + t) * 8; };
    Eight<DT> w[NV], s[NV], g[NV];
    float acc[NV][8] = {};
    if constexpr (WEIGHTS) {
#pragma unroll
        for (int u = 0; u < NV; ++u) w[u].template load<true>(a.weight, first(u), K - first(u));
    }
    auto request = [&](long long row) {
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int n = row < a.n_rows ? K - first(u) : 0;
            s[u].template load<true>(a.s, static_cast<size_t>(row) * K + first(u), n);
            g[u].template load<true>(a.dy, static_cast<size_t>(row) * K + first(u), n);
        }
    };
    if (AHEAD) request(worker);
    int turn = 0;
    for (long long row = worker < a.workers ? worker : a.n_rows; row < a.n_rows; row += a.workers, turn ^= 1) {
        const size_t at = static_cast<size_t>(row) * K;
        if constexpr (!AHEAD) request(row);
        Eight<DT> sv[NV], gv[NV], dv[NV];
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            sv[u] = s[u];
            gv[u] = g[u];
            if (a.dsum) dv[u].template load<true>(a.dsum, at + first(u), K - first(u));
            if constexpr (!WEIGHTS) w[u].template load<true>(a.weight, first(u), K - first(u));
        }
        if constexpr (AHEAD) request(row + a.workers);
        float v[2] = {0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[0] = fmaf(sv[u].value(i), sv[u].value(i), v[0]);
                v[1] = fmaf(gv[u].value(i) * w[u].value(i), sv[u].value(i), v[1]);
            }
        row_sums(v, scratch[turn], one_warp);
        const float inv = inverse_root(v[0], K, a.eps), mean = v[1] * inv / static_cast<float>(K);
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            float d[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float n = sv[u].value(i) * inv, gi = gv[u].value(i);
                acc[u][i] = fmaf(gi, n, acc[u][i]);
                d[i] = inv * fmaf(-n, mean, gi * w[u].value(i));
                if (a.dsum) d[i] += dv[u].value(i);
            }
            store<DT, true>(a.dx, at + first(u), K - first(u), packed<DT>(d));
        }
    }
    if (worker < a.workers) {
#pragma unroll
        for (int u = 0; u < NV; ++u)
            store<MTC_F32, true>(a.part, static_cast<size_t>(worker) * K + first(u), K - first(u), packed<MTC_F32>(acc[u]));
    }
}

// Any alignment and length: what a row's results need by a CTA a row, ...
template <int DT>
__global__ void __launch_bounds__(256) norm_grad_rows_kernel(const NormGradArgs a) {
    pdl_enter();
    __shared__ __align__(16) float scratch[64];
    const size_t at = static_cast<size_t>(blockIdx.x) * a.K;
    float v[2] = {0.0f, 0.0f};
    for (int k = threadIdx.x; k < a.K; k += blockDim.x) {
        const float s = ld_written_as_f32(a.s, at + k, DT);
        v[0] = fmaf(s, s, v[0]);
        v[1] = fmaf(ld_written_as_f32(a.dy, at + k, DT) * ld_written_as_f32(a.weight, k, DT), s, v[1]);
    }
    row_sums(v, scratch, false);
    if (threadIdx.x == 0) {
        const float inv = inverse_root(v[0], a.K, a.eps);
        a.rows[blockIdx.x] = make_float2(inv, v[1] * inv / static_cast<float>(a.K));
    }
}
// ... the shares of dw by a thread a column over a range of rows, ...
template <int DT>
__global__ void __launch_bounds__(128) norm_grad_columns_kernel(const NormGradArgs a) {
    pdl_enter();
    const long long k = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (k >= a.K) return;
    float acc = 0.0f;
    for (long long row = blockIdx.y; row < a.n_rows; row += a.workers) {
        const size_t at = static_cast<size_t>(row) * a.K + k;
        acc = fmaf(ld_written_as_f32(a.dy, at, DT), ld_written_as_f32(a.s, at, DT) * a.rows[row].x, acc);
    }
    a.part[static_cast<size_t>(blockIdx.y) * a.K + k] = acc;
}

// ... and ds, last: it may take the place of dy.
template <int DT>
__global__ void __launch_bounds__(256) norm_grad_values_kernel(const NormGradArgs a) {
    pdl_enter();
    const size_t at = static_cast<size_t>(blockIdx.x) * a.K;
    const float inv = a.rows[blockIdx.x].x, mean = a.rows[blockIdx.x].y;
    for (int k = threadIdx.x; k < a.K; k += blockDim.x) {
        const float n = ld_written_as_f32(a.s, at + k, DT) * inv, g = ld_written_as_f32(a.dy, at + k, DT);
        float d = inv * fmaf(-n, mean, g * ld_written_as_f32(a.weight, k, DT));
        if (a.dsum) d += ld_written_as_f32(a.dsum, at + k, DT);
        st_from_f32(a.dx, at + k, d, DT);
    }
}

// dw = the shares added up in f64: 32 columns a CTA, whose warps take the shares in turn
template <int WARPS>
__global__ void __launch_bounds__(32 * WARPS) norm_grad_join_kernel(const float *part, void *dweight, int workers, int K, int dt) {
    pdl_enter();
    __shared__ double sums[WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long k = static_cast<long long>(blockIdx.x) * 32 + lane;
    double acc = 0.0;
    if (k < K) {
#pragma unroll 8
        for (int p = warp; p < workers; p += WARPS) acc += part[static_cast<size_t>(p) * K + k];
    }
    sums[warp][lane] = acc;
    __syncthreads();
    if (warp == 0 && k < K) {
#pragma unroll
        for (int i = 1; i < WARPS; ++i) acc += sums[i][lane];
        st_from_f32(dweight, k, static_cast<float>(acc), dt);
    }
}

bool on_16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int round_up(int v, int step) { return (v + step - 1) / step * step; }

// The gradient's rows are dealt out to this many workers (CTAs, or warps that have rows of their own): what a worker adds up for dw is written once and read again.
struct GradShape {
    int turns, threads, block, workers;          // threads of a row, of a CTA
};
// Two turns of 16-bit values a thread, 512 threads an SM (their registers hold a row and the next one: 8192 x 4096 bf16 54 us, in one turn of 512 threads 64; 4096 x 8192 56);
// one turn where rows are few or f32 (333 x 2880 bf16 7.6 and 10.0, f32 8.3 and 10.7, since there are fewer shares to add up).  Rows past 8192 take four turns.
GradShape grad_shape(int sms, long long n_rows, int K, int dt) {
    const int eights = static_cast<int>((static_cast<long long>(K) + 7) / 8);
    GradShape g{};
    const bool few = n_rows < 4ll * sms;
    g.turns = eights <= 32 ? 1 : eights > 1024 ? 4 : eights > 512 || !(few || dt == MTC_F32) ? 2 : 1;
    g.threads = std::min(512, round_up((eights + g.turns - 1) / g.turns, 32));
    const int rows = g.threads == 32 ? 4 : 1;
    g.block = g.threads * rows;
    const long long ctas = static_cast<long long>(sms) * (few && rows == 1 ? 1 : std::max(1, 512 / g.block));
    g.workers = static_cast<int>(std::min<long long>(n_rows, ctas * rows));
    return g;
}

template <int DT, int MODE>
cudaError_t launch_norm(Ctx *ctx, cudaStream_t st, NormArgs a) {
    const bool vec = a.K % 8 == 0 && on_16(a.x) && on_16(a.weight) && (!a.residual || (on_16(a.residual) && on_16(a.sum))) && (!a.y || on_16(a.y)) &&
                     reinterpret_cast<uintptr_t>(a.codes) % 8 == 0;
    const int eights = (a.K + 7) / 8;
    // One turn of many threads where rows are few, two turns of half as many where they fill the GPU, four of 16-bit values where there are many rows: what a thread does
    // once a row costs as much as sixteen values (codes of 8192 x 4096 bf16 52 us in two turns, 49 in four, 46 with four CTAs of it an SM; 333 rows 4.8 and 5.2; f32 65 and
    // 69; y instead of codes: 2048 x 4096 9.3 and 9.5, 4096 x 8192 43.9 and 41.3)
    const int turns = a.n_rows <= ctx->sm_count && eights <= 1024 ? 1 : DT != MTC_F32 && a.n_rows >= 4ll * ctx->sm_count && eights >= (MODE ? 256 : 513) && eights <= 1024 ? 4 : 2;
    a.threads = std::min(1024, round_up((eights + turns - 1) / turns, 32));
    const int rows_a_cta = a.threads == 32 ? 4 : 1;
    const long long ctas = (a.n_rows + rows_a_cta - 1) / rows_a_cta;
    const dim3 grid(static_cast<unsigned>(ctas));
    const int block = a.threads * rows_a_cta;
    if (!vec) return launch_pdl(add_norm_kernel<DT, false, 0, MODE>, grid, block, 0, st, a);
    if (eights > turns * a.threads) return launch_pdl(add_norm_kernel<DT, true, 0, MODE>, grid, block, 0, st, a);
    if constexpr (DT != MTC_F32) {
        if (turns == 4) return launch_pdl(add_norm_kernel<DT, true, 4, MODE>, grid, block, 0, st, a);
    }
    return turns == 1 ? launch_pdl(add_norm_kernel<DT, true, 1, MODE>, grid, block, 0, st, a) : launch_pdl(add_norm_kernel<DT, true, 2, MODE>, grid, block, 0, st, a);
}
template <int DT>
cudaError_t launch_norm(Ctx *ctx, cudaStream_t st, const NormArgs &a, int mode) {
    return mode == 0 ? launch_norm<DT, 0>(ctx, st, a) : mode == 1 ? launch_norm<DT, 1>(ctx, st, a) : launch_norm<DT, 2>(ctx, st, a);
}

template <int DT>
cudaError_t launch_grad(const GradShape &g, cudaStream_t st, NormGradArgs a) {
    const bool vec = a.K % 8 == 0 && on_16(a.dy) && on_16(a.s) && on_16(a.weight) && on_16(a.dx) && (!a.dsum || on_16(a.dsum));
    const int eights = (a.K + 7) / 8;
    if (!vec || eights > 4 * 512) {
        const dim3 rows(static_cast<unsigned>(a.n_rows));
        cudaError_t e = launch_pdl(norm_grad_rows_kernel<DT>, rows, 256, 0, st, a);
        if (e == cudaSuccess) e = launch_pdl(norm_grad_columns_kernel<DT>, dim3((a.K + 127u) / 128u, a.workers), 128, 0, st, a);
        return e == cudaSuccess ? launch_pdl(norm_grad_values_kernel<DT>, rows, 256, 0, st, a) : e;
    }
    a.threads = g.threads;
    const int rows = g.block / g.threads, turns = g.turns, block = g.block;
    const dim3 grid((a.workers + rows - 1) / rows);
    return turns == 1   ? launch_pdl(norm_grad_kernel<DT, 1>, grid, block, 0, st, a)
           : turns == 2 ? launch_pdl(norm_grad_kernel<DT, 2>, grid, block, 0, st, a)
                        : launch_pdl(norm_grad_kernel<DT, 4>, grid, block, 0, st, a);
}

}  // namespace

cudaError_t launch_add_rms_norm(Ctx *ctx, cudaStream_t st, const NormArgs &a, int mode, int dt) {
    return (dt == MTC_F32 ? launch_norm<MTC_F32> : dt == MTC_BF16 ? launch_norm<MTC_BF16> : launch_norm<MTC_F16>)(ctx, st, a, mode);
}

size_t norm_grad_workspace(int sms, long long n_rows, int K, int dt) {
    return n_rows <= 0 ? 0 : static_cast<size_t>(grad_shape(sms, n_rows, K, dt).workers) * K * 4 + static_cast<size_t>((n_rows + 1) / 2) * 16;
}

cudaError_t launch_norm_grad(Ctx *ctx, cudaStream_t st, NormGradArgs a, void *dweight, void *workspace, int dt) {
    const GradShape g = grad_shape(ctx->sm_count, a.n_rows, a.K, dt);
    a.workers = g.workers;
    a.rows = static_cast<float2 *>(workspace);
    a.part = reinterpret_cast<float *>(a.rows + (a.n_rows + 1) / 2 * 2);
    if (a.n_rows > 0) {
        const cudaError_t e = (dt == MTC_F32 ? launch_grad<MTC_F32> : dt == MTC_BF16 ? launch_grad<MTC_BF16> : launch_grad<MTC_F16>)(g, st, a);
        if (e != cudaSuccess) return e;
    }
    const dim3 grid((a.K + 31u) / 32u);          // (no rows: zeros)
    return a.workers > 256 ? launch_pdl(norm_grad_join_kernel<32>, grid, 1024, 0, st, a.part, dweight, a.workers, a.K, dt)
                           : launch_pdl(norm_grad_join_kernel<16>, grid, 512, 0, st, a.part, dweight, a.workers, a.K, dt);
}

}  // namespace mtc
