// Low-rank adapters on warp-level tensor cores: h = x A^T and out = base + scale h B^T (or, back, u = dy B and dx = base + scale u A) in one launch.
//
// A cluster of 8, 4 or 2 CTAs (launch) has one tile of rows of one adapter: each CTA, each of its eight warps, sums up a part of the long axis of the first product; the parts meet in
// shared memory, then over distributed shared memory, so that every CTA has the whole h of the tile; then each CTA takes a part of the
// columns of the second product.  x, base and out pass once, a tile's adapter is read by its cluster once, h never leaves the SM.
//
// Bound by latency where users decode: 64 rows of 32 adapters, 4096 -> 14336, rank 16, bf16 take 10.3 us where the bytes need 3; a row alone, 4096 -> 4096, takes 5.5.  Of that the launch is 2, and
// the chain is loads of x and A, the sums over the cluster (two barriers of it), loads of B and base, stores.  So everything that a CTA will read is asked for before
// it waits (prefetches into L2, and base and B into registers where they fit), and a tile is spread over up to 64 warps.  128-row tiles of tcgen05 would be empty for the most part there;
// from some hundreds of rows (back, rank 64) to 2304 (forward, ranks to 32) on the shared reading of the adapter and one thread that issues the MMAs win (lora.cu has both sides).
//
// Registers: two CTAs an SM leave 128 a thread, and with tiles of 32 rows, ranks 33 to 64 or f32 the second product keeps base, the weights of four ranks and its sums at once.  Back, these forms
// spill: 900 bytes at rank 64 and 32 rows (1550 where a side has no whole pieces), 220 at rank 64 and 16 rows, 330 at rank 32 and 32 rows, 570 to 750 of f32 at rank 32 and 32 rows.  They are what
// 200 rows of rank 64 take (back 27 us) and 2048 rows of 64 adapters (199).
#pragma once

#include <algorithm>
#include <type_traits>

#include "lora_mma.cuh"

namespace mtc {
namespace {

using namespace lora;

constexpr int kWarps = 8, kThreads = 32 * kWarps;

__host__ __device__ constexpr int part_stride(int rb) { return rb + 4; }
__host__ __device__ constexpr int held_stride(int rt) { return rt + 8; }         // in 16-bit values: rows 16 bytes apart modulo 128

// Into L2, 16-byte aligned pieces: a request a row (with one a line, 2000 cycles went into asking)
__device__ __forceinline__ void prefetch(const char *p, size_t bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(static_cast<uint32_t>(bytes)) : "memory");
}
// `bytes` of each of `rows` rows, a row `pitch` bytes; row_of: which rows (null: the first ones; negative: none); by the threads from `first` on
__device__ __forceinline__ void prefetch_rows(const void *from, size_t pitch, size_t bytes, int rows, const int *row_of, int first) {
    for (int i = (static_cast<int>(threadIdx.x) - first + kThreads) % kThreads; i < rows; i += kThreads) {
        const int row = row_of ? row_of[i] : i;
        if (row >= 0) prefetch(static_cast<const char *>(from) + row * pitch, bytes);
    }
}
__device__ __forceinline__ void prefetch_block(const void *from, size_t bytes, int first) {
    constexpr size_t piece = 4096;
    for (size_t i = static_cast<size_t>((static_cast<int>(threadIdx.x) - first + kThreads) % kThreads) * piece; i < bytes; i += kThreads * piece)
        prefetch(static_cast<const char *>(from) + i, min(piece, bytes - i));
}

using NoCare = std::integral_constant<Care, Care::none>;
using AllCare = std::integral_constant<Care, Care::all>;

// Whether all these sums are numbers
template <int A, int B>
__device__ __forceinline__ bool finite(const float (&large)[A][B][4], const float (&small)[A][B][4]) {
    float z = 0.0f;                              // (an infinity and a NaN times zero are NaN)
#pragma unroll
    for (int a = 0; a < A; ++a)
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) z = fmaf(large[a][b][i], 0.0f, fmaf(small[a][b][i], 0.0f, z));
    return z == 0.0f;
}
template <int A, int B>
__device__ __forceinline__ void clear(float (&sums)[A][B][4]) {
#pragma unroll
    for (int a = 0; a < A; ++a)
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[a][b][i] = 0.0f;
}

// RB: ranks a pass (a block of the rank, ONE: there is one), 8 to 64.  MT: tiles of 16 rows.  VIN, VOUT: rows on this side are whole 16-byte pieces; else their values are
// loaded one by one.  BACK: the first product's weights lie [c_in][rank], the second's
// [rank][c_out]; else [rank][c_in] and [c_out][rank].
template <int DT, int RB, int MT, bool BACK, bool ONE, bool VIN, bool VOUT>
__global__ void __launch_bounds__(kThreads, DT == MTC_F32 && RB > 16 ? 1 : 2) lora_mma_kernel(const LoraArgs a, int cluster_log, int rank_blocks_, bool keep, bool none) {
    pdl_enter();
    constexpr int ROWS = 16 * MT, PS = part_stride(RB), P = pieces<DT>, H = DT == MTC_F32 ? 3 : 2, NT = RB / 8, SIZE = DT == MTC_F32 ? 4 : 2;
    constexpr bool HALF = DT == MTC_F16;
    extern __shared__ __align__(16) float sm[];
    const int rank_blocks = ONE ? 1 : rank_blocks_, RT = rank_blocks * RB, HS = held_stride(RT);
    float *const part = sm;                                                      // [warps][ROWS][PS]
    uint16_t *const held = reinterpret_cast<uint16_t *>(part + kWarps * ROWS * PS);      // [H][ROWS][HS]
    float *const low = reinterpret_cast<float *>(held + H * ROWS * HS);          // [ROWS][RT], not ONE only
    __shared__ int row_of[ROWS];
    __shared__ float back_up[ROWS];              // f16: the power of two that a row's h was divided by
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int cr = cluster_rank();
    if (blockIdx.x == 0)
        for (int e = threadIdx.x; e < a.n_adapters; e += kThreads)
            if (a.offsets[e] > a.offsets[e + 1] || a.offsets[e + 1] > static_cast<uint32_t>(a.n_rows)) atomicCAS(a.status, 0u, 0x901u);
    const int cs = 1 << cluster_log;              // (shifts: with 64-bit divisions a single row took 6.1 us in place of 5.1)
    const Tile tile = find_tile(a, blockIdx.x >> cluster_log, ROWS, none);
    if (tile.e < 0) return;                      // the whole cluster
    if (threadIdx.x < ROWS) {
        int row = -1;
        if (threadIdx.x < tile.n) {
            const uint32_t v = a.order[tile.p0 + threadIdx.x];
            if (v < static_cast<uint32_t>(a.n_rows)) row = static_cast<int>(v);
            else atomicCAS(a.status, 0u, 0x908u);
        }
        row_of[threadIdx.x] = row;
    }
    constexpr int CW = BACK ? 64 : 32;           // columns of a warp's step
    const int units = (a.c_out + CW - 1) / CW, unit0 = static_cast<int>(static_cast<long long>(units) * cr >> cluster_log), unit1 = static_cast<int>(static_cast<long long>(units) * (cr + 1) >> cluster_log);
    const int chunks = (a.c_in + 31) / 32, me = cr * kWarps + warp;
    __syncthreads();
    if (tile.e >= a.n_adapters) {                // rows of no adapter: base, or zeros
        copy_rows<DT, kThreads, VOUT>(a, row_of, static_cast<int>(tile.n), unit0 * CW, min(unit1 * CW, a.c_out), keep, cr, cs);
        return;
    }
    const size_t expert = tile.e;
    if constexpr (VIN && VOUT) {                 // everything that this CTA will read is on its way before it waits for any of it
        const int k0 = static_cast<int>(static_cast<long long>(chunks) * cr >> cluster_log) * 32, k1 = min(static_cast<int>(static_cast<long long>(chunks) * (cr + 1) >> cluster_log) * 32, a.c_in);
        const int n0 = unit0 * CW, n1 = min(unit1 * CW, a.c_out);
        const size_t in_row = static_cast<size_t>(a.c_in) * SIZE, out_row = static_cast<size_t>(a.c_out) * SIZE, rank_row = static_cast<size_t>(a.rank) * SIZE;
        const char *const down = static_cast<const char *>(a.down) + expert * a.rank * in_row, *const up = static_cast<const char *>(a.up) + expert * a.rank * out_row;
        if (k1 > k0) {
            prefetch_rows(static_cast<const char *>(a.in) + static_cast<size_t>(k0) * SIZE, in_row, static_cast<size_t>(k1 - k0) * SIZE, ROWS, row_of, 0);
            if (BACK) prefetch_block(down + k0 * rank_row, (k1 - k0) * rank_row, 32);
            else prefetch_rows(down + static_cast<size_t>(k0) * SIZE, in_row, static_cast<size_t>(k1 - k0) * SIZE, a.rank, nullptr, 32);
        }
        if (n1 > n0) {
            if (BACK) prefetch_rows(up + static_cast<size_t>(n0) * SIZE, out_row, static_cast<size_t>(n1 - n0) * SIZE, a.rank, nullptr, 96);
            else prefetch_block(up + n0 * rank_row, (n1 - n0) * rank_row, 96);
            if (a.base) prefetch_rows(static_cast<const char *>(a.base) + static_cast<size_t>(n0) * SIZE, out_row, static_cast<size_t>(n1 - n0) * SIZE, ROWS, row_of, 160);
        }
    }

    // ---- the first product: this warp's part of c_in, 32 values at a time
    int rows[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) rows[m][0] = row_of[16 * m + g], rows[m][1] = row_of[16 * m + g + 8];
    const int chunk0 = static_cast<int>(static_cast<long long>(chunks) * me >> (cluster_log + 3)), chunk1 = static_cast<int>(static_cast<long long>(chunks) * (me + 1) >> (cluster_log + 3));

    // What a warp's step of the second product reads: weights of 32 ranks (tiles of columns, or four rows of ranks at a time), base.  EARLY: several steps'
    // are loaded at once, the first ones before the parts meet (64 rows of 32 adapters 12.1 us a step at a time); elsewhere, where registers do not allow
    // it, each right before its products.
    constexpr int TN = CW / 8, QS = RB >= 32 ? RB / 32 : 1, WIDE = RB >= 32 ? 8 : RB / 4, PARTS = WIDE == 8 ? 2 : 1, DEEP = WIDE == 2 ? 2 : 4;
    constexpr bool EARLY = VIN && VOUT && ONE && MT == 1 && P == 1 && (BACK ? RB <= 16 : RB <= 32);
    constexpr int STEPS = !EARLY ? 1 : BACK || RB == 32 ? 2 : 4;
    using V = Vals<DT, BACK ? 8 : WIDE>;
    struct Unit {
        V w[BACK ? DEEP * (EARLY ? PARTS : 1) : TN];
        lora::Eight<DT> base[MT][2][CW / 32];
    };
    auto load_base = [&](Unit &to, int n0) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < CW / 32; ++i) {
                    const int c = n0 + t * (CW / 4) + 8 * i;
                    const bool there = a.base && rows[m][h] >= 0;
                    const size_t at = static_cast<size_t>(rows[m][h]) * a.c_out + c;
                    if constexpr (VOUT) to.base[m][h][i].load(a.base, at, there && c < a.c_out);
                    else to.base[m][h][i].load_any(a.base, at, there ? a.c_out - c : 0);
                }
    };
    auto load_weights = [&](auto care, V *to, int n0, int r, int i) {     // r: this lane's first rank; i (BACK): four ranks behind
        constexpr Care CARE = decltype(care)::value;
        if constexpr (!BACK) {
            // column c of tile j is n0 + c / 2 * 8 + 2 j + c % 2, so that a lane's results are eight neighbours
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int n = n0 + (g >> 1) * 8 + 2 * j + (g & 1);
                to[j].template load<CARE>(a.up, (expert * a.c_out + n) * a.rank + r, n < a.c_out && r < a.rank);
            }
        } else {
            // column c of tile j is n0 + 8 c + j: a lane loads eight neighbours of four ranks' rows, its results are sixteen
            const int c = n0 + 8 * g;
#pragma unroll
            for (int s = 0; s < DEEP; ++s) {
                const int rr = r + 4 * i + s;
                if constexpr (VOUT) to[s].template load<CARE>(a.up, (expert * a.rank + rr) * a.c_out + c, rr < a.rank && c < a.c_out);
                else to[s].template load_any<CARE>(a.up, (expert * a.rank + rr) * a.c_out + c, rr < a.rank ? a.c_out - c : 0);
            }
        }
    };
    auto load_early = [&](Unit &to, int n0) {
        load_base(to, n0);
#pragma unroll
        for (int i = 0; i < (BACK ? PARTS : 1); ++i) load_weights(NoCare(), to.w + i * DEEP, n0, t * WIDE, i);
    };
    Unit steps[STEPS];
    auto load_steps = [&](int u) {               // steps u, u + kWarps ..
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
            if (u + i * kWarps < unit1) load_early(steps[i], (u + i * kWarps) * CW);
    };
    const float scale = a.scales ? a.scales[expert] : 1.0f;
    for (int rb = 0; rb < rank_blocks; ++rb) {
        float acc[MT][NT][4] = {};
        float fine[P > 1 ? MT : 1][P > 1 ? NT : 1][4] = {};      // f32: the products of small pieces, apart so that the large ones are cut off less often
        auto sum_up = [&](auto care) {
            constexpr Care CARE = decltype(care)::value;
#pragma unroll (CARE != Care::none ? 1 : MT == 1 && RB <= 16 && P == 1 ? 4 : 2)
            for (int c = chunk0; c < chunk1; ++c) {
                const int k = c * 32 + t * 8;
                const bool in = k < a.c_in;
                Vals<DT, 8> x[MT][2];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if constexpr (VIN) x[m][h].template load<CARE>(a.in, static_cast<size_t>(rows[m][h]) * a.c_in + k, in && rows[m][h] >= 0);
                        else x[m][h].template load_any<CARE>(a.in, static_cast<size_t>(rows[m][h]) * a.c_in + k, rows[m][h] >= 0 ? a.c_in - k : 0);
                    }
                auto step = [&](int j, int p, int i, uint32_t b0, uint32_t b1) {      // tile j of ranks, piece p of the weights, half i of the 32 values
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int q = 0; q + p < P; ++q) {
                            float (&d)[4] = P > 1 && q + p > 0 ? fine[P > 1 ? m : 0][P > 1 ? j : 0] : acc[m][j];
                            mma<HALF>(d, x[m][0].w[q][2 * i], x[m][1].w[q][2 * i], x[m][0].w[q][2 * i + 1], x[m][1].w[q][2 * i + 1], b0, b1);
                        }
                };
                if constexpr (!BACK) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const int r = rb * RB + 8 * j + g;
                        Vals<DT, 8> w;
                        if constexpr (VIN) w.template load<CARE>(a.down, (expert * a.rank + r) * a.c_in + k, in && r < a.rank);
                        else w.template load_any<CARE>(a.down, (expert * a.rank + r) * a.c_in + k, r < a.rank ? a.c_in - k : 0);
#pragma unroll
                        for (int p = 0; p < P; ++p)
#pragma unroll
                            for (int i = 0; i < 2; ++i) step(j, p, i, w.w[p][2 * i], w.w[p][2 * i + 1]);
                    }
                } else {
                    using V = Vals<DT, NT>;          // lane g has ranks g NT .. g NT + NT - 1: rank g NT + j is column g of tile j
                    const int r = rb * RB + g * NT;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        V w[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) w[q].template load<CARE>(a.down, (expert * a.c_in + k + 4 * i + q) * a.rank + r, (VIN ? in : k + 4 * i + q < a.c_in) && r < a.rank);
#pragma unroll
                        for (int j = 0; j < NT; ++j)
#pragma unroll
                            for (int p = 0; p < P; ++p) step(j, p, i, V::pair(w[0], w[1], p, j), V::pair(w[2], w[3], p, j));
                    }
                }
            }
        };
        sum_up(NoCare());
        if constexpr (P > 1) {                   // a sum that is no number, or values that 16 bits do not reach: once more, with more care
            if (__any_sync(0xffffffffu, !finite(acc, fine))) {
                clear(acc), clear(fine);
                sum_up(AllCare());
            }
        }
        if constexpr (EARLY) {
            load_steps(unit0 + warp);
        }
        // ---- the warps' parts, then the CTAs'
        if (rb) {                                // (the gather of the block before has read `part`)
            cluster_arrive();
            cluster_wait();
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = 16 * m + g + (i >= 2 ? 8 : 0), c = 2 * t + (i & 1), col = BACK ? c * NT + j : 8 * j + c;
                    part[(warp * ROWS + row) * PS + col] = P > 1 ? acc[m][j][i] + fine[P > 1 ? m : 0][P > 1 ? j : 0][i] : acc[m][j][i];
                }
        __syncthreads();
        for (int i = threadIdx.x; i < ROWS * RB / 4; i += kThreads) {
            float4 *const at = reinterpret_cast<float4 *>(part + i / (RB / 4) * PS + i % (RB / 4) * 4);
            float4 s = *at;
#pragma unroll
            for (int w = 1; w < kWarps; ++w) {
                const float4 v = at[w * ROWS * PS / 4];
                s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
            }
            *at = s;
        }
        cluster_arrive();
        cluster_wait();
        for (int i0 = 0; i0 < ROWS * RB / 4; i0 += kThreads) {
            const int i = i0 + threadIdx.x, row = i / (RB / 4), col = i % (RB / 4) * 4;
            const bool mine = ROWS * RB / 4 % kThreads == 0 || i < ROWS * RB / 4;
            float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            auto add = [&](auto count) {         // all loads first
                constexpr int N = decltype(count)::value;
                float4 v[N];
#pragma unroll
                for (int q = 0; q < N; ++q) v[q] = ld_cta(part + row * PS + col, q);
#pragma unroll
                for (int q = 0; q < N; ++q) s.x += v[q].x, s.y += v[q].y, s.z += v[q].z, s.w += v[q].w;
            };
            if (mine) {
                if (cluster_log == 3) add(std::integral_constant<int, 8>());
                else if (cluster_log == 2) add(std::integral_constant<int, 4>());
                else add(std::integral_constant<int, 2>());
                if (keep && (i & (cs - 1)) == cr) {      // the CTAs of the cluster share the writing
                    const int r = row_of[row], at = rb * RB + col;
                    if (r >= 0) {
                        float *const p = a.low + static_cast<size_t>(r) * a.rank + at;
                        if (at < a.rank) p[0] = s.x;
                        if (at + 1 < a.rank) p[1] = s.y;
                        if (at + 2 < a.rank) p[2] = s.z;
                        if (at + 3 < a.rank) p[3] = s.w;
                    }
                }
                s = ranks_of(s, rb * RB + col, a.rank);
            }
            if constexpr (ONE) {
                float f = 1.0f;
                if constexpr (HALF) {            // RB / 4 lanes have a row
                    float most = most_of(s);
#pragma unroll
                    for (int o = RB / 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                    f = unit_of(most);
                    if (mine && col == 0) back_up[row] = f;
                }
                if (mine) hold<DT>(s, f, held + row * HS + col, ROWS * HS);
            } else if (mine) {
                *reinterpret_cast<float4 *>(low + row * RT + rb * RB + col) = s;
            }
        }
    }
    cluster_arrive_relaxed();                    // nobody leaves while its part is read: waited for at the end
    if constexpr (!ONE) {
        __syncthreads();
        for (int row = warp; row < ROWS; row += kWarps) {
            float f = 1.0f;
            if constexpr (HALF) {
                float most = 0.0f;
                for (int i = lane; i < RT; i += 32) most = fmaxf(most, fabsf(or_zero(low[row * RT + i])));
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                f = unit_of(most);
                if (lane == 0) back_up[row] = f;
            }
            for (int i = lane * 4; i < RT; i += 128) hold<DT>(*reinterpret_cast<const float4 *>(low + row * RT + i), f, held + row * HS + i, ROWS * HS);
        }
    }
    __syncthreads();

    // ---- the second product
    auto multiply = [&](Unit &unit, int n0) {
        if constexpr (!EARLY) load_base(unit, n0);
        float acc[MT][TN][4] = {};
        float fine[P > 1 ? MT : 1][P > 1 ? TN : 1][4] = {};
        auto sum_up = [&](auto care) {
            for (int rb = 0; rb < rank_blocks; ++rb) {
#pragma unroll
                for (int q = 0; q < QS; ++q) {
                    const int r = rb * RB + q * 32 + t * WIDE;       // this lane's ranks: r .. r + WIDE - 1
                    uint32_t hw[MT][2][H][WIDE / 2];
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int p = 0; p < H; ++p) {
                                const uint16_t *const at = held + (p * ROWS + 16 * m + g + 8 * h) * HS + r;
                                if constexpr (WIDE == 8) {
                                    const uint4 v = *reinterpret_cast<const uint4 *>(at);
                                    hw[m][h][p][0] = v.x, hw[m][h][p][1] = v.y, hw[m][h][p][2] = v.z, hw[m][h][p][3] = v.w;
                                } else if constexpr (WIDE == 4) {
                                    const uint2 v = *reinterpret_cast<const uint2 *>(at);
                                    hw[m][h][p][0] = v.x, hw[m][h][p][1] = v.y;
                                } else {
                                    hw[m][h][p][0] = *reinterpret_cast<const uint32_t *>(at);
                                }
                            }
                    auto step = [&](int j, int p, int i, uint32_t b0, uint32_t b1) {  // tile j of columns, piece p of the weights, ranks 4 i .. of the lane's
#pragma unroll
                        for (int m = 0; m < MT; ++m)
#pragma unroll
                            for (int s = 0; s < H; ++s) {
                                if (P > 1 && s + p >= P) continue;
                                float (&d)[4] = P > 1 && s + p > 0 ? fine[P > 1 ? m : 0][P > 1 ? j : 0] : acc[m][j];
                                const uint32_t a2 = WIDE == 2 ? 0u : hw[m][0][s][WIDE == 2 ? 0 : 2 * i + 1], a3 = WIDE == 2 ? 0u : hw[m][1][s][WIDE == 2 ? 0 : 2 * i + 1];
                                mma<HALF>(d, hw[m][0][s][2 * i], hw[m][1][s][2 * i], a2, a3, b0, b1);
                            }
                    };
                    if constexpr (!BACK) {
                        if constexpr (!EARLY) load_weights(care, unit.w, n0, r, 0);
#pragma unroll
                        for (int j = 0; j < TN; ++j)
#pragma unroll
                            for (int p = 0; p < P; ++p)
#pragma unroll
                                for (int i = 0; i < PARTS; ++i) step(j, p, i, unit.w[j].w[p][2 * i], WIDE == 2 ? 0u : unit.w[j].w[p][WIDE == 2 ? 0 : 2 * i + 1]);
                    } else {
#pragma unroll
                        for (int i = 0; i < PARTS; ++i) {
                            V *const w = unit.w + (EARLY ? i * DEEP : 0);
                            if constexpr (!EARLY) load_weights(care, w, n0, r, i);
#pragma unroll
                            for (int j = 0; j < TN; ++j)
#pragma unroll
                                for (int p = 0; p < P; ++p) step(j, p, i, V::pair(w[0], w[1], p, j), WIDE == 2 ? 0u : V::pair(w[WIDE == 2 ? 0 : 2], w[WIDE == 2 ? 1 : 3], p, j));
                        }
                    }
                }
            }
        };
        sum_up(NoCare());
        if constexpr (P > 1) {
            if (__any_sync(0xffffffffu, !finite(acc, fine))) {
                clear(acc), clear(fine);
                sum_up(AllCare());
            }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (rows[m][h] < 0) continue;
                const float factor = HALF ? scale * back_up[16 * m + g + 8 * h] : scale;
#pragma unroll
                for (int i = 0; i < CW / 32; ++i) {
                    const int c = n0 + t * (CW / 4) + 8 * i;
                    float v[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int j = BACK ? k : k / 2, at = 2 * h + (BACK ? i : k & 1);
                        v[k] = acc[m][j][at];
                        if constexpr (P > 1) v[k] += fine[m][j][at];
                    }
                    if (c < a.c_out) unit.base[m][h][i].template add_and_store<VOUT>(a.out, static_cast<size_t>(rows[m][h]) * a.c_out + c, v, factor, a.c_out - c);
                }
            }
    };
    for (int u0 = unit0 + warp; u0 < unit1; u0 += STEPS * kWarps) {
        if (EARLY && u0 != unit0 + warp) load_steps(u0);
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
            if (u0 + i * kWarps < unit1) multiply(steps[i], (u0 + i * kWarps) * CW);
    }
    cluster_wait();
}

template <int DT, int RB, int MT, bool BACK, bool ONE, bool VIN = true, bool VOUT = true>
cudaError_t launch(cudaStream_t st, const LoraArgs &a, bool keep, bool none) {
    constexpr int ROWS = 16 * MT, H = DT == MTC_F32 ? 3 : 2;
    const int blocks = (a.rank + RB - 1) / RB;
    const size_t smem = static_cast<size_t>(kWarps * ROWS * part_stride(RB) + (ONE ? 0 : ROWS * blocks * RB)) * 4 + static_cast<size_t>(H * ROWS * held_stride(blocks * RB)) * 2;
    static PerDeviceAttr attr;
    cudaError_t e = attr.set(lora_mma_kernel<DT, RB, MT, BACK, ONE, VIN, VOUT>, 200 * 1024);
    if (e != cudaSuccess) return e;
    const long long tiles = most_tiles(a, ROWS);
    // The largest cluster of which all tiles' fit at once: with more CTAs a tile, each does less of the long axes, and a second wave costs as much as the first.  (Of eight CTAs 15 fit, of four
    // 36, and about twice that at two CTAs an SM; tiles are counted as if adapters ended at half a tile.)  us of clusters of 8, 4 and 2, f32, 4096 x 4096: rank 16, 256 rows 13.1, 16.5, 27.9,
    // 1024 35.8, 26.1, 39.1, 4096 112, 90, 89; rank 64, 1024 123, 93, 97.  Narrow layers have too little for eight: 1024 x 1024, rank 64, 64 rows 14.4, 14.4, 22.6, bf16 7.0, 6.9, 8.3; 4096
    // rows of f32 253, 116, 96.
    constexpr int ROOM = DT == MTC_F32 && RB > 16 ? 1 : 2;                       // CTAs an SM
    const long long about = a.n_rows / ROWS + std::min(a.n_adapters, a.n_rows) / 2;
    const int cluster_log = about <= 16 * ROOM - (ROOM == 1) && lora_width(a) > 2048 ? 3 : about <= 36 * ROOM ? 2 : 1;
    if ((tiles << cluster_log) > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    return launch_cluster(lora_mma_kernel<DT, RB, MT, BACK, ONE, VIN, VOUT>, static_cast<unsigned>(tiles << cluster_log), kThreads, 1 << cluster_log, smem, st, a, cluster_log, blocks, keep, none);
}
template <int DT, int MT, bool BACK>
cudaError_t launch_pieces(cudaStream_t st, const LoraArgs &a, bool keep, bool none) {
    constexpr int MOST = DT == MTC_F32 ? 32 : 64;
    if constexpr (DT != MTC_F32 || MT == 1) {
        if (a.rank <= 8) return launch<DT, 8, MT, BACK, true>(st, a, keep, none);
        if (a.rank <= 16) return launch<DT, 16, MT, BACK, true>(st, a, keep, none);
    }
    if (a.rank <= 32) return launch<DT, 32, MT, BACK, true>(st, a, keep, none);
    if (a.rank <= MOST) return launch<DT, MOST, MT, BACK, true>(st, a, keep, none);
    return launch<DT, MOST, 1, BACK, false>(st, a, keep, none);
}
// values one by one on one side or both: two sizes of the rank are enough
template <int DT, int MT, bool BACK, bool VIN, bool VOUT>
cudaError_t launch_values(cudaStream_t st, const LoraArgs &a, bool keep, bool none) {
    constexpr int MOST = DT == MTC_F32 ? 32 : 64;
    if constexpr (DT != MTC_F32 || MT == 1) {
        if (a.rank <= 16) return launch<DT, 16, MT, BACK, true, VIN, VOUT>(st, a, keep, none);
    }
    if (a.rank <= MOST) return launch<DT, MOST, MT, BACK, true, VIN, VOUT>(st, a, keep, none);
    return launch<DT, MOST, 1, BACK, false, false, false>(st, a, keep, none);
}
template <int DT, int MT, bool BACK>
cudaError_t launch_side(cudaStream_t st, const LoraArgs &a, bool keep, bool none) {
    const bool in = lora_pieces_in(a), out = lora_pieces_out(a);
    if (in && out) return launch_pieces<DT, MT, BACK>(st, a, keep, none);
    if (in) return launch_values<DT, MT, BACK, true, false>(st, a, keep, none);
    return out ? launch_values<DT, MT, BACK, false, true>(st, a, keep, none) : launch_values<DT, MT, BACK, false, false>(st, a, keep, none);
}

}  // namespace

template <int DT>
cudaError_t launch_lora_mma(cudaStream_t st, const LoraArgs &a, bool backward, bool keep, bool none) {
    // Tiles of 32 rows where those of 16 leave clusters too small or make a second wave (launch), and the registers of the form allow it.  us of 16 and 32 rows, 4096 x 4096: bf16 rank 16,
    // 1024 rows 10.5 and 11.6, 2048 18.8 and 18.4; f32 rank 32, 192 rows 14.0 and 19.2, 256 22.0 and 19.2, 384 23.8 and 19.9, 512 26.0 and 34.0, 640 48.2 and 35.5, 2048 94 and 70
    // (1024 x 1024: 384 rows 9.0 and 12.4, 640 13.7 and 12.4); f32 rank 16, 1024 rows 26 and 35, 4096 89 and 129
    const bool between = a.n_rows > 240 && a.n_rows <= 480 && lora_width(a) > 2048;
    const bool wide = DT != MTC_F32 ? a.n_rows > 1152 : a.rank > 16 && (a.n_rows > 576 || between);
    if (wide) return backward ? launch_side<DT, 2, true>(st, a, keep, none) : launch_side<DT, 2, false>(st, a, keep, none);
    return backward ? launch_side<DT, 1, true>(st, a, keep, none) : launch_side<DT, 1, false>(st, a, keep, none);
}

}  // namespace mtc
