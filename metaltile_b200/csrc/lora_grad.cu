// The gradients of low-rank adapters' weights on warp-level tensor cores:
//   dA_e[i][c] = scale_e sum over the rows t of e of u_t[i] x_t[c],      dB_e[c][i] = scale_e sum of h_t[i] dy_t[c]
//
// One launch for both.  A CTA has a block of columns of one adapter, all its ranks (64 at a time), and a part of its rows; the CTAs of a cluster share the
// rows and add up over distributed shared memory in a fixed order.  Bound by reading x and dy, which pass once.  Rows are the k of the MMAs: u and h are
// staged in shared memory as operand pieces with the rows side by side, x and dy go from global memory into fragments, four rows of eight neighbours a lane,
// paired up.  All operands are bf16 pieces: f16 values are two (11 bits), since u and h have no bound that f16 would hold.
#include <algorithm>

#include "lora_mma.cuh"

namespace mtc {
namespace {

using namespace lora;

constexpr int kThreads = 256, kStage = 64, kStride = kStage + 16;        // rows at a time, and apart in 16-bit values (no two lanes of a load in one bank)

// W neighbours as bf16 pieces, pairs
template <int DT, int W>
struct Split {
    static constexpr int P = DT == MTC_BF16 ? 1 : DT == MTC_F16 ? 2 : 3, N = W / 2;
    uint32_t w[P][N];
    __device__ __forceinline__ void load(const void *base, size_t at, bool there) {
        if constexpr (DT != MTC_F16) {
            Vals<DT, W> v;
            v.load(base, at, there);
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int i = 0; i < N; ++i) w[p][i] = v.w[p][i];
        } else {
            Vals<DT, W> v;
            v.load(base, at, there);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&v.w[0][i]));
                const uint32_t lo = __float_as_uint(f.x), hi = __float_as_uint(f.y);
                w[0][i] = high_halves(lo, hi);
                w[1][i] = high_halves(__float_as_uint(f.x - __uint_as_float(lo & 0xFFFF0000u)), __float_as_uint(f.y - __uint_as_float(hi & 0xFFFF0000u)));
            }
        }
    }
    static __device__ __forceinline__ uint32_t pair(const Split &x, const Split &y, int p, int j) {
        return j & 1 ? high_halves(x.w[p][j / 2], y.w[p][j / 2]) : low_halves(x.w[p][j / 2], y.w[p][j / 2]);
    }
};

// RB: ranks a pass.  Columns of a CTA: four warps of NT tiles of eight; the other four take the other half of the rows.
template <int DT, int RB>
struct Form {
    static constexpr int NT = DT == MTC_F32 || RB == 64 ? 4 : 8, CB = 32 * NT, RP = RB < 16 ? 16 : RB, MT = RP / 16, H = DT == MTC_F32 ? 3 : 2;
    static constexpr int sums = 2 * (RP * (CB + 4) > CB * (RP + 4) ? RP * (CB + 4) : CB * (RP + 4)), staged = 2 * H * RP * kStride;
    static constexpr size_t smem = static_cast<size_t>(sums) * 4 + static_cast<size_t>(staged) * 2;
};

template <int DT, int RB>
__global__ void __launch_bounds__(kThreads) lora_weights_kernel(const LoraWeights w, int blocks_a, int blocks_b, int rank_blocks) {
    pdl_enter();
    using F = Form<DT, RB>;
    using S = Split<DT, F::NT>;
    constexpr int NT = F::NT, CB = F::CB, RP = F::RP, MT = F::MT, H = F::H, P = S::P, DEEP = P == 1 ? 2 : P;
    extern __shared__ __align__(16) float sm[];
    float *const sums = sm;                                                      // [2][RP][CB + 4], or [2][CB][RP + 4]
    uint16_t *const held = reinterpret_cast<uint16_t *>(sums + F::sums);         // [2][H][RP][kStride]
    __shared__ int row_of[2][kStage];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, half = warp >> 2;
    const int cs = cluster_size(), cr = cluster_rank();
    const uint32_t id = blockIdx.x / cs;
    const int blocks = blocks_a + blocks_b, block = id % blocks, rb = id / blocks % rank_blocks;
    const size_t e = id / blocks / rank_blocks;
    const bool of_a = block < blocks_a;
    const LoraWeight &W = of_a ? w.a : w.b;
    const int c0 = (of_a ? block : block - blocks_a) * CB, r0 = rb * RB, n_cols = min(CB, W.c - c0), n_ranks = min(RB, w.rank - r0);
    const uint32_t from = min(w.offsets[e], static_cast<uint32_t>(w.n_rows)), to = min(w.offsets[e + 1], static_cast<uint32_t>(w.n_rows));
    const uint32_t n = to > from ? to - from : 0;

    const int stages = static_cast<int>((static_cast<long long>(n) + kStage - 1) / kStage);
    const int s0 = static_cast<int>(static_cast<long long>(stages) * cr / cs), s1 = static_cast<int>(static_cast<long long>(stages) * (cr + 1) / cs);
    // rows of a stage: two neighbours of them and a rank a thread and turn
    auto stage = [&](int s) {
        const int b = s & 1;
        if (threadIdx.x < kStage) {
            const uint32_t at = static_cast<uint32_t>(s) * kStage + threadIdx.x;
            int row = -1;
            if (at < n) {
                const uint32_t v = w.order[from + at];
                if (v < static_cast<uint32_t>(w.n_rows)) row = static_cast<int>(v);
                else atomicCAS(w.status, 0u, 0x908u);
            }
            row_of[b][threadIdx.x] = row;
        }
        __syncthreads();
#pragma unroll 4
        for (int i = threadIdx.x; i < RP * kStage / 2; i += kThreads) {
            const int r = i % RP, k = i / RP * 2;
            float v[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int row = row_of[b][k + q];
                v[q] = row >= 0 && r < n_ranks ? W.low[static_cast<size_t>(row) * w.rank + r0 + r] : 0.0f;
            }
#pragma unroll
            for (int p = 0; p < H; ++p) {
                uint32_t lo = __float_as_uint(v[0]), hi = __float_as_uint(v[1]);
                if (p + 1 == H) {                // the last piece is rounded
                    const __nv_bfloat162 z = __floats2bfloat162_rn(v[0], v[1]);
                    *reinterpret_cast<uint32_t *>(held + ((b * H + p) * RP + r) * kStride + k) = *reinterpret_cast<const uint32_t *>(&z);
                } else {
                    *reinterpret_cast<uint32_t *>(held + ((b * H + p) * RP + r) * kStride + k) = high_halves(lo, hi);
                    v[0] = fabsf(v[0]) < INFINITY ? v[0] - __uint_as_float(lo & 0xFFFF0000u) : 0.0f;
                    v[1] = fabsf(v[1]) < INFINITY ? v[1] - __uint_as_float(hi & 0xFFFF0000u) : 0.0f;
                }
            }
        }
    };

    float acc[MT][NT][4] = {};
    const int col = c0 + (warp & 3) * 8 * NT + g * NT;
    if (s0 < s1) stage(s0);
    for (int s = s0; s < s1; ++s) {
        const int b = s & 1;
        __syncthreads();
        S x[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = row_of[b][16 * (2 * i + half) + 4 * t + q];
                x[i][q].load(W.in, static_cast<size_t>(row) * W.c + col, row >= 0 && col < W.c);
            }
        if (s + 1 < s1) stage(s + 1);
        float part[P == 3 ? MT : 1][P == 3 ? NT : 1][4] = {};    // f32: the sums of a stage, small products first, are added to the others as f32 numbers
#pragma unroll
        for (int order = DEEP - 1; order >= 0; --order)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int p = 0; p <= order && p < H; ++p) {
                    const int q = order - p;     // piece of x
                    if (q >= P) continue;
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const uint16_t *const at = held + ((b * H + p) * RP + 16 * m + g) * kStride + 16 * (2 * i + half) + 4 * t;
                        const uint2 lo = *reinterpret_cast<const uint2 *>(at), hi = *reinterpret_cast<const uint2 *>(at + 8 * kStride);
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            float (&d)[4] = P == 3 ? part[P == 3 ? m : 0][P == 3 ? j : 0] : acc[m][j];
                            mma<false>(d, lo.x, hi.x, lo.y, hi.y, S::pair(x[i][0], x[i][1], q, j), S::pair(x[i][2], x[i][3], q, j));
                        }
                    }
                }
        if constexpr (P == 3) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][j][i] += part[m][j][i];
        }
    }

    // ---- the warps' and the CTAs' sums, along what lies next to each other in the result
    const int lines = of_a ? RP : CB, stride = of_a ? CB + 4 : RP + 4;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * m + g + (i >= 2 ? 8 : 0), c = (warp & 3) * 8 * NT + (2 * t + (i & 1)) * NT + j;
                sums[half * lines * stride + (of_a ? r * stride + c : c * stride + r)] = acc[m][j][i];
            }
    cluster_arrive();
    cluster_wait();
    const float scale = w.scales ? w.scales[e] : 1.0f;
    const int used = of_a ? n_ranks : n_cols, wide = of_a ? n_cols : n_ranks, fours = (wide + 3) / 4;
    for (int i = threadIdx.x + cr * kThreads; i < used * fours; i += kThreads * cs) {
        const int line = i / fours, k = i % fours * 4;
        float v[4] = {};
        for (int q = 0; q < cs; ++q)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 f = ld_cta(sums + (h * lines + line) * stride + k, q);
                v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
            }
        const size_t at = of_a ? (e * w.rank + r0 + line) * W.c + c0 + k : (e * W.c + c0 + line) * w.rank + r0 + k;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (k + q < wide) st_from_f32(W.grad, at + q, v[q] * scale, DT);
    }
    cluster_arrive();
    cluster_wait();                              // nobody leaves while its sums are read
}

bool on_16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <int DT, int RB>
cudaError_t launch(Ctx *ctx, cudaStream_t st, const LoraWeights &w) {
    using F = Form<DT, RB>;
    const long long rank_blocks = (w.rank + RB - 1) / RB, blocks_a = (w.a.c + F::CB - 1) / F::CB, blocks_b = (w.b.c + F::CB - 1) / F::CB;
    const long long items = (blocks_a + blocks_b) * rank_blocks * w.n_adapters;
    // Rows are shared by as many CTAs as fill the GPU twice, where an adapter of average length leaves each of them two stages
    const long long rows = w.n_rows / w.n_adapters;
    int cs = 1;
    while (cs < 8 && items * cs < 2ll * ctx->sm_count && rows >= 2ll * kStage * cs * 2) cs *= 2;
    if (items * cs > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    static PerDeviceAttr attr;
    const cudaError_t e = attr.set(lora_weights_kernel<DT, RB>, F::smem);
    if (e != cudaSuccess) return e;
    return launch_cluster(lora_weights_kernel<DT, RB>, static_cast<unsigned>(items * cs), kThreads, cs, F::smem, st, w, static_cast<int>(blocks_a), static_cast<int>(blocks_b),
                          static_cast<int>(rank_blocks));
}
template <int DT>
cudaError_t launch(Ctx *ctx, cudaStream_t st, const LoraWeights &w) {
    if (w.rank <= 8) return launch<DT, 8>(ctx, st, w);
    if (w.rank <= 16) return launch<DT, 16>(ctx, st, w);
    if (DT == MTC_F32 || w.rank <= 32) return launch<DT, 32>(ctx, st, w);
    return launch<DT, DT == MTC_F32 ? 32 : 64>(ctx, st, w);
}

}  // namespace

bool lora_grad_supported(const LoraWeights &w) { return w.a.c % 8 == 0 && w.b.c % 8 == 0 && on_16(w.a.in) && on_16(w.b.in); }
cudaError_t launch_lora_grad(Ctx *ctx, cudaStream_t st, const LoraWeights &w, int dt) {
    return (dt == MTC_F32 ? launch<MTC_F32> : dt == MTC_BF16 ? launch<MTC_BF16> : launch<MTC_F16>)(ctx, st, w);
}

}  // namespace mtc
