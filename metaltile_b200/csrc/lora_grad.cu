// The gradients of low-rank adapters' weights on warp-level tensor cores:
//   dA_e[i][c] = scale_e sum over the rows t of e of u_t[i] x_t[c],      dB_e[c][i] = scale_e sum of h_t[i] dy_t[c]
//
// One launch for both.  A CTA has a block of columns of one adapter, all its ranks (64 at a time), and a part of its rows; the CTAs of a cluster share the
// rows and add up over distributed shared memory in a fixed order.  x and dy pass once, by cp.async, 64 rows a stage, up to two stages ahead.  Rows are the k of the MMAs: u and h
// are staged as operand pieces a stage ahead and transposed as they are loaded; of x and dy a lane takes eight neighbours of four
// rows and pairs them up.  All operands are bf16 pieces: f16 values are two (11 bits), since u and h have no bound that f16 would hold.  Of f16 all four products of pieces are
// taken: that of the small ones is up to 2^-14 of the whole, of one sign where the operands are (left out, it cost one result in 25 its last bit
// there); it costs a training step 3 to 6 % (2048 x 4096 -> 4096, rank 64, 108.5 -> 114.4 us).
//
// Measured: 4096 rows of 4096 + 4096, rank 16, bf16 some 33 us behind dx's kernel, 2 TB/s of x and dy (the bytes need 10.3 us); 512 rows of 2048 + 768 in f32, rank 8, 10.  Bound by what a CTA cannot overlap, in
// two waves of CTAs: of 25,000 cycles the start and the first stage take 8,000, the sums over the cluster 5,000.  A bulk copy a row and mbarriers take half the instructions and
// were no faster (34.9 us).
#include <algorithm>

#include "lora_mma.cuh"

namespace mtc {
namespace {

using namespace lora;

constexpr int kThreads = 256, kStage = 64, kRowsAhead = 4;                // rows of a stage; buffers of row numbers

// W neighbours as bf16 pieces, pairs
template <int DT, int W>
struct Split {
    static constexpr int P = DT == MTC_BF16 ? 1 : DT == MTC_F16 ? 2 : 3, N = W / 2;
    uint32_t w[P][N];
    __device__ __forceinline__ void load(const void *base, size_t at, bool there) {
        if constexpr (DT != MTC_F16) {
            Vals<DT, W> v;
            v.template load<Care::large>(base, at, there);
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int i = 0; i < N; ++i) w[p][i] = v.w[p][i];
        } else {
            Vals<DT, W> v;
            v.template load<Care::large>(base, at, there);
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
    static constexpr int NT = DT == MTC_F32 || RB >= 32 ? 4 : 8, CB = 32 * NT, RP = RB < 16 ? 16 : RB, MT = RP / 16, H = DT == MTC_F32 ? 3 : 2;
    static constexpr int AHEAD = DT == MTC_F32 ? 2 : 3;              // buffers of x or dy
    // bytes of a row of a stage (16 bytes apart modulo 128, so that the rows of a fragment do not meet in a bank), of a stage, of a row of an operand piece
    static constexpr int SIZE = DT == MTC_F32 ? 4 : 2, PITCH = CB * SIZE + 16, tile = kStage * PITCH, LOW = RP * 2;
    static constexpr int sums = 2 * (RP * (CB + 4) > CB * (RP + 4) ? RP * (CB + 4) : CB * (RP + 4)) * 4, staged = 2 * H * kStage * LOW;
    static constexpr size_t smem = (sums > AHEAD * tile + staged ? sums : AHEAD * tile + staged);    // (the sums take the stages' place)
};

template <int DT, int RB, bool VEC>
__global__ void __launch_bounds__(kThreads, DT == MTC_F32 ? 1 : 2) lora_weights_kernel(const LoraWeights w, int blocks_a, int blocks_b, int rank_blocks) {
    pdl_enter();
    using F = Form<DT, RB>;
    using S = Split<DT, F::NT>;
    constexpr int NT = F::NT, CB = F::CB, RP = F::RP, MT = F::MT, H = F::H, P = S::P, DEEP = P == 1 ? 2 : 3;   // products of pieces with p + q < DEEP: all of one or two, six of nine of three
    extern __shared__ __align__(128) uint8_t sm[];
    float *const sums = reinterpret_cast<float *>(sm);                           // [2][RP][CB + 4], or [2][CB][RP + 4]
    const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(sm)), held = base + F::AHEAD * F::tile;          // [2][H][kStage][RP] bf16, units of 16 bytes moved about
    __shared__ int row_of[kRowsAhead][kStage];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, half = warp >> 2;
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
    const int s0 = static_cast<int>(static_cast<long long>(stages) * cr / cs), mine = static_cast<int>(static_cast<long long>(stages) * (cr + 1) / cs) - s0;

    // row numbers of stage s of this CTA, by 64 threads
    auto row_at = [&](int s) {
        const uint32_t at = static_cast<uint32_t>(s0 + s) * kStage + tid;
        if (s >= mine || at >= n) return -1;
        const uint32_t v = w.order[from + at];
        if (v < static_cast<uint32_t>(w.n_rows)) return static_cast<int>(v);
        atomicCAS(w.status, 0u, 0x908u);
        return -1;
    };
    // x or dy of a stage, zeros where there is no row
    const bool pieces = VEC || (W.c % 8 == 0 && reinterpret_cast<uintptr_t>(W.in) % 16 == 0);
    constexpr int UNITS = CB * F::SIZE / 16, PASSES = kStage * UNITS / kThreads;
    auto copy = [&](int s) {
        if (s < mine) {
            const int u = tid % UNITS, c = c0 + u * (16 / F::SIZE);
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                const int r = (i * kThreads + tid) / UNITS, row = row_of[s % kRowsAhead][r];
                const bool ok = row >= 0 && c < W.c;
                if (!VEC && !pieces) {           // rows of any length: values one by one
                    constexpr int N = 16 / F::SIZE;
                    uint32_t v[4] = {};
#pragma unroll
                    for (int j = 0; j < N; ++j)
                        if (ok && c + j < W.c) {
                            const size_t at = static_cast<size_t>(row) * W.c + c + j;
                            if constexpr (DT == MTC_F32) v[j] = static_cast<const uint32_t *>(W.in)[at];
                            else v[j / 2] |= static_cast<uint32_t>(static_cast<const uint16_t *>(W.in)[at]) << (j & 1) * 16;
                        }
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(base + s % F::AHEAD * F::tile + r * F::PITCH + u * 16), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
                    continue;
                }
                const char *const src = static_cast<const char *>(W.in) + (ok ? (static_cast<size_t>(row) * W.c + c) * F::SIZE : 0);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(base + s % F::AHEAD * F::tile + r * F::PITCH + u * 16), "l"(src), "r"(ok ? 16 : 0) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // u or h of a stage: four ranks of a row a thread and turn
    constexpr int TURNS = RP * kStage / 4 / kThreads;
    const bool fours = w.rank % 4 == 0 && reinterpret_cast<uintptr_t>(W.low) % 16 == 0;
    auto load_low = [&](int s, float4 (&v)[TURNS]) {
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            const int q = i * kThreads + tid, r = q % (RP / 4) * 4, row = s < mine ? row_of[s % kRowsAhead][q / (RP / 4)] : -1;
            v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (row < 0 || r >= n_ranks) continue;
            const float *const p = W.low + static_cast<size_t>(row) * w.rank + r0 + r;
            if (fours) {
                v[i] = *reinterpret_cast<const float4 *>(p);
            } else {
                v[i].x = p[0];
                if (r + 1 < n_ranks) v[i].y = p[1];
                if (r + 2 < n_ranks) v[i].z = p[2];
                if (r + 3 < n_ranks) v[i].w = p[3];
            }
        }
    };
    // row k of a piece, 16-byte unit u
    auto piece_at = [&](int s, int p, int k, int u) {
        return held + (((s & 1) * H + p) * kStage + k) * F::LOW + ((u ^ (RP == 16 ? k >> 2 & 1 : RP == 32 ? k >> 1 & 3 : k & 7)) << 4);
    };
    auto hold_low = [&](int s, const float4 (&v)[TURNS]) {
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            const int q = i * kThreads + tid, u4 = q % (RP / 4);
            uint2 piece[3];
            hold_pieces<H == 3 ? MTC_F32 : MTC_BF16, Care::large>(v[i], 1.0f, piece);
#pragma unroll
            for (int p = 0; p < H; ++p)
                asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(piece_at(s, p, q / (RP / 4), u4 / 2) + (u4 & 1) * 8), "r"(piece[p].x), "r"(piece[p].y) : "memory");
        }
    };

    if (tid < kStage) {
        const int a = row_at(0), b = row_at(1), c = row_at(2);
        row_of[0][tid] = a, row_of[1][tid] = b, row_of[2][tid] = c;
    }
    __syncthreads();
    for (int s = 0; s + 1 < F::AHEAD; ++s) copy(s);
    {
        float4 v[TURNS];
        load_low(0, v);
        hold_low(0, v);
    }
    float acc[MT][NT][4] = {};
    for (int s = 0; s < mine; ++s) {
        const int b = s % F::AHEAD;
        asm volatile("cp.async.wait_group %0;" ::"n"(F::AHEAD - 2) : "memory");
        __syncthreads();                         // the stage is there, and everybody has done with the one before
        const int row3 = tid < kStage ? row_at(s + 3) : -1;
        copy(s + F::AHEAD - 1);
        float4 next[TURNS];
        load_low(s + 1, next);
        S x[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)          // rows 2t, 2t + 1, 2t + 8, 2t + 9 of sixteen; NT columns
                x[i][q].load(sm + b * F::tile + (16 * (2 * i + half) + 2 * t + (q & 1) + (q & 2) * 4) * F::PITCH + ((warp & 3) * 8 + g) * NT * F::SIZE, 0, true);
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
                        // 8 x 8 of (rows 0-7, ranks 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15), transposed
                        uint32_t l[4];
                        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(l[0]), "=r"(l[1]), "=r"(l[2]), "=r"(l[3])
                                     : "r"(piece_at(s, p, 16 * (2 * i + half) + (lane & 7) + (lane >> 4) * 8, 2 * m + (lane >> 3 & 1))) : "memory");
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            float (&d)[4] = P == 3 ? part[P == 3 ? m : 0][P == 3 ? j : 0] : acc[m][j];
                            mma<false>(d, l[0], l[1], l[2], l[3], S::pair(x[i][0], x[i][1], q, j), S::pair(x[i][2], x[i][3], q, j));
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
        hold_low(s + 1, next);
        if (tid < kStage) row_of[(s + 3) % kRowsAhead][tid] = row3;
    }
    __syncthreads();                             // the sums take the stages' place

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
    const bool alone = cs == 1;                  // (a barrier of the cluster is a thousand cycles)
    if (alone) __syncthreads();
    else cluster_arrive(), cluster_wait();
    const float scale = w.scales ? w.scales[e] : 1.0f;
    const bool aligned = reinterpret_cast<uintptr_t>(W.grad) % 16 == 0;
    const int used = of_a ? n_ranks : n_cols, wide = of_a ? n_cols : n_ranks, in_line = (wide + 3) / 4;
    for (int i = tid + cr * kThreads; i < used * in_line; i += kThreads * cs) {
        const int line = i / in_line, k = i % in_line * 4;
        float v[4] = {};
        if (alone) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 f = *reinterpret_cast<const float4 *>(sums + (h * lines + line) * stride + k);
                v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
            }
        } else {
            float4 part[8][2];                   // (all on their way at once: one after the other they took 5000 cycles)
#pragma unroll
            for (int q = 0; q < 8; ++q)
#pragma unroll
                for (int h = 0; h < 2; ++h) part[q][h] = q < cs ? ld_cta(sums + (h * lines + line) * stride + k, q) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int q = 0; q < 8; ++q)
#pragma unroll
                for (int h = 0; h < 2; ++h) v[0] += part[q][h].x, v[1] += part[q][h].y, v[2] += part[q][h].z, v[3] += part[q][h].w;
        }
        const size_t at = of_a ? (e * w.rank + r0 + line) * W.c + c0 + k : (e * W.c + c0 + line) * w.rank + r0 + k;
        if (k + 4 <= wide && at % 4 == 0 && aligned) {
            if constexpr (DT == MTC_F32) {
                *reinterpret_cast<float4 *>(static_cast<float *>(W.grad) + at) = make_float4(v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale);
            } else if constexpr (DT == MTC_BF16) {
                const __nv_bfloat162 x = __floats2bfloat162_rn(v[0] * scale, v[1] * scale), y = __floats2bfloat162_rn(v[2] * scale, v[3] * scale);
                *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(W.grad) + at) = make_uint2(*reinterpret_cast<const uint32_t *>(&x), *reinterpret_cast<const uint32_t *>(&y));
            } else {
                const __half2 x = __floats2half2_rn(v[0] * scale, v[1] * scale), y = __floats2half2_rn(v[2] * scale, v[3] * scale);
                *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(W.grad) + at) = make_uint2(*reinterpret_cast<const uint32_t *>(&x), *reinterpret_cast<const uint32_t *>(&y));
            }
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (k + q < wide) st_from_f32(W.grad, at + q, v[q] * scale, DT);
        }
    }
    if (!alone) cluster_arrive(), cluster_wait();        // nobody leaves while its sums are read
}

bool on_16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <int DT, int RB, bool VEC = true>
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
    const cudaError_t e = attr.set(lora_weights_kernel<DT, RB, VEC>, F::smem);
    if (e != cudaSuccess) return e;
    return launch_cluster(lora_weights_kernel<DT, RB, VEC>, static_cast<unsigned>(items * cs), kThreads, cs, F::smem, st, w, static_cast<int>(blocks_a), static_cast<int>(blocks_b),
                          static_cast<int>(rank_blocks));
}
template <int DT>
cudaError_t launch(Ctx *ctx, cudaStream_t st, const LoraWeights &w) {
    if (w.a.c % 8 || w.b.c % 8 || !on_16(w.a.in) || !on_16(w.b.in))                  // two sizes of the rank are enough
        return w.rank <= 16 ? launch<DT, 16, false>(ctx, st, w) : launch<DT, DT == MTC_F32 ? 32 : 64, false>(ctx, st, w);
    if (w.rank <= 8) return launch<DT, 8>(ctx, st, w);
    if (w.rank <= 16) return launch<DT, 16>(ctx, st, w);
    if (DT == MTC_F32 || w.rank <= 32) return launch<DT, 32>(ctx, st, w);
    return launch<DT, DT == MTC_F32 ? 32 : 64>(ctx, st, w);
}

}  // namespace

cudaError_t launch_lora_grad(Ctx *ctx, cudaStream_t st, const LoraWeights &w, int dt) {
    return (dt == MTC_F32 ? launch<MTC_F32> : dt == MTC_BF16 ? launch<MTC_BF16> : launch<MTC_F16>)(ctx, st, w);
}

}  // namespace mtc
