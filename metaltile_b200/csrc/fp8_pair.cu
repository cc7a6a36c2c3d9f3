// Products of e4m3 codes with block scales on tcgen05, for many tokens (dense: fp8_mm; grouped by expert: fp8_gather_mm):
//
//   out[t, n] = sum_b xs[t, b] * ws[n / 128, b] * D_b[t, n],      D_b[t, n] = sum_{k in block b} x[t, k] * w[n, k]
//
// A pair of CTAs (a cluster of two SMs) owns a tile of 256 tokens x 256 weight rows: each SM holds 128 tokens of A and half of the weight rows of B, and the MMAs
// (cta_group::2, 256 x 128, kind::f8f6f4) read both.  A block of 128 codes is a chain of four of them for each half of the weight rows, into an accumulator of its own in
// tensor memory; a half is one block of scales.  The epilogue takes the accumulators out, multiplies by xs * ws, one number a thread (lane = token), and adds up in
// registers: 128 sums a thread, eight warps.
//
// Bound by what an SM can take in.  128 x 256 x 128 products take an SM 512 cycles at the dense rate, and a tile of 256 x 256 needs 32 KB a block on each SM of a
// pair: 64 bytes a cycle, as many as an SM gets from L2; one CTA by itself with 128 x 256 would need 96.  Out of tensor memory and into the sums is 256 cycles
// of the FMA pipes.  The four accumulators are all of the tensor memory, two blocks deep, so the MMAs of a block run while the one before is read.
//
//   warps 0-7    epilogue   warps 0-3 the first half of the weight rows, 4-7 the second
//   warps 8-9    scales     xs of 128 tokens, 16 blocks at a time, turned round into shared memory (a load of each lane's own row would cost
//                           the load pipe ten cycles a lane), and ws
//   warp 10      producer   TMA, both CTAs of a pair into their own memory, one barrier in the first
//   warp 11      MMA        issued by the first CTA
// A persistent pair walks the tiles, tokens fastest.  Every wait is bounded: on expiry the kernel records a code in the status word, the roles leave and what is in
// flight is awaited (bounded too).
#include <cstddef>

#include "fp8.cuh"
#include "tcgen05.cuh"

namespace mtc {
namespace {

using namespace fp8;

constexpr int kTokens = 256, kCols = 256;        // of a tile; a CTA of a pair has 128 of the tokens
constexpr int kABytes = 128 * kBlock, kBBytes = 64 * kBlock, kStage = kABytes + 2 * kBBytes;
constexpr int kStages = 6;
constexpr int kEpiWarps = 8, kScaleWarp0 = 8, kScaleWarps = 2, kLoadWarp = 10, kMmaWarp = 11, kThreads = 384;
constexpr int kHeld = 16, kPitch = 132;          // blocks whose scales are in shared memory, floats of a block's xs
constexpr int kScaleFloats = kHeld * kPitch + 2 * kHeld;
constexpr int kMaxExperts = 1024;

struct PArgs {
    const float *xs, *ws;
    const uint32_t *expert_offsets;              // nullptr: dense
    void *out;
    uint32_t *status;
    int M, N, nkb, n_experts;
    int col_tiles, row_blocks;                   // ceil(N / 256), ceil(N / 128)
    int out_dt;
    int wide;                                    // rows of the output can be stored 16 bytes at a time
};
struct PMaps {
    CUtensorMap x, w;
};
struct __align__(16) PCtrl {
    uint64_t full[kStages], empty[kStages], d_full[2][2], d_empty[2][2], s_full[2], s_empty[2], drained;
    uint32_t tmem_base, issued;
    volatile uint32_t abort;
    uint32_t n_chunks;
    uint32_t first_chunk[kMaxExperts + 1];       // grouped: chunks of 256 tokens of the experts before
    uint32_t offset[kMaxExperts + 1];            // and the clamped offsets
};
constexpr int kCtlBytes = (sizeof(PCtrl) + 1023) / 1024 * 1024;
constexpr int kScaleBytes = (2 * kScaleFloats * 4 + 1023) / 1024 * 1024;
constexpr int kSmemBytes = 1024 + kCtlBytes + kScaleBytes + kStages * kStage;
static_assert(kSmemBytes <= 227 * 1024, "shared memory");

__device__ __forceinline__ uint32_t on_cta(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// into this CTA's memory; the barrier may be the other CTA's
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap *map, int c0, int c1, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar) : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// arrives at the barrier of this offset in both CTAs when the MMAs so far are complete
__device__ __forceinline__ void commit_pair(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"(static_cast<uint16_t>(3)) : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// The chunks of the experts, by one warp: ceil(rows / 256) each.  Offsets that run backwards or past the rows are clamped and reported.
__device__ void count_chunks(PCtrl *ctl, const PArgs &a) {
    const int lane = threadIdx.x & 31;
    uint32_t before = 0;
    for (int e0 = 0; e0 < a.n_experts; e0 += 32) {
        const int e = e0 + lane;
        uint32_t lo = 0, hi = 0;
        if (e < a.n_experts) {
            const uint32_t p = a.expert_offsets[e], q = a.expert_offsets[e + 1], m = static_cast<uint32_t>(a.M);
            if (p > m || q > m || q < p) atomicCAS(a.status, 0u, 0x901u);
            lo = min(p, m);
            hi = max(lo, min(q, m));
        }
        const uint32_t np = (hi - lo + kTokens - 1) / kTokens;
        uint32_t upto = np;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += v;
        }
        if (e < a.n_experts) {
            ctl->first_chunk[e] = before + upto - np;
            ctl->offset[e] = lo;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) {
        ctl->first_chunk[a.n_experts] = before;
        ctl->n_chunks = before;
    }
}

struct Tile {
    int expert, tok0, ntok, n0;
};
__device__ __forceinline__ Tile tile_of(const PCtrl *ctl, const PArgs &a, int index) {
    const int chunks = static_cast<int>(ctl->n_chunks), c = index % chunks;
    Tile t;
    t.n0 = index / chunks * kCols;
    if (!a.expert_offsets) {
        t.expert = 0;
        t.tok0 = c * kTokens;
        t.ntok = min(kTokens, a.M - t.tok0);
        return t;
    }
    int lo = 0, hi = a.n_experts;                // the last expert whose first chunk is not behind c: it has chunk c
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (static_cast<int>(ctl->first_chunk[mid]) <= c) lo = mid;
        else hi = mid;
    }
    t.expert = lo;
    const int at = (c - static_cast<int>(ctl->first_chunk[lo])) * kTokens;
    t.tok0 = static_cast<int>(ctl->offset[lo]) + at;
    const uint32_t end = max(ctl->offset[lo], min(a.expert_offsets[lo + 1], static_cast<uint32_t>(a.M)));
    t.ntok = min(kTokens, static_cast<int>(end) - t.tok0);
    return t;
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (DT == MTC_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
__device__ __forceinline__ void store16(void *p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) { *static_cast<uint4 *>(p) = make_uint4(a, b, c, d); }

// Eight neighbouring results of a row
template <int DT>
__device__ __forceinline__ void store8(void *out, size_t at, const uint64_t (&acc)[64], int i) {
    float2 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = halves(acc[i + j]);
    if constexpr (DT == MTC_F32) {
        float *const p = static_cast<float *>(out) + at;
        *reinterpret_cast<float4 *>(p) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        *reinterpret_cast<float4 *>(p + 4) = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    } else {
        store16(static_cast<uint16_t *>(out) + at, pack2<DT>(v[0].x, v[0].y), pack2<DT>(v[1].x, v[1].y), pack2<DT>(v[2].x, v[2].y), pack2<DT>(v[3].x, v[3].y));
    }
}

__global__ void __launch_bounds__(kThreads, 1) fp8_pair_kernel(const __grid_constant__ PMaps maps, const __grid_constant__ PArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *const smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    PCtrl *const ctl = reinterpret_cast<PCtrl *>(smem);
    float *const scales = reinterpret_cast<float *>(smem + kCtlBytes);       // two of [kHeld][kPitch] of xs, [2][kHeld] of ws
    const uint32_t ring = smem_u32(smem) + kCtlBytes + kScaleBytes;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = static_cast<int>(blockIdx.x & 1), pair = static_cast<int>(blockIdx.x >> 1), pairs = static_cast<int>(gridDim.x >> 1);
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&ctl->full[s], 1);
            mbar_init(&ctl->empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            for (int h = 0; h < 2; ++h) {
                mbar_init(&ctl->d_full[h][i], 1);
                mbar_init(&ctl->d_empty[h][i], kEpiWarps);       // four warps of each CTA, in the first one's memory
            }
            mbar_init(&ctl->s_full[i], kScaleWarps);
            mbar_init(&ctl->s_empty[i], kEpiWarps);
        }
        mbar_init(&ctl->drained, 1);
        ctl->abort = 0;
        ctl->issued = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)), "n"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    pdl_enter();
    if (!a.expert_offsets) {
        if (threadIdx.x == 0) ctl->n_chunks = (a.M + kTokens - 1) / kTokens;
    } else if (warp == 0) {
        count_chunks(ctl, a);
    }
    tc_fence_before();
    cluster_sync();                              // both CTAs' barriers exist
    tc_fence_after();
    const uint32_t tmem = ctl->tmem_base;
    const int n_tiles = static_cast<int>(ctl->n_chunks) * a.col_tiles;

    if (warp == kLoadWarp) {
        if (lane == 0) {
            int s = 0;
            uint32_t phase = 1;
            bool go = true;
            for (int i = pair; go && i < n_tiles; i += pairs) {
                const Tile t = tile_of(ctl, a, i);
                const int row = static_cast<int>(static_cast<long long>(t.expert) * a.N) + t.n0 + rank * 64;
                for (int kb = 0; kb < a.nkb; ++kb) {
                    if (!mbar_wait(&ctl->empty[s], phase, &ctl->abort, a.status, 0xb11u)) {
                        go = false;
                        break;
                    }
                    const uint32_t at = ring + s * kStage, bar = on_cta(smem_u32(&ctl->full[s]), 0);
                    if (rank == 0) mbar_expect_tx(&ctl->full[s], 2 * kStage);
                    tma_load_pair(at, &maps.x, kb * kBlock, t.tok0 + rank * 128, bar);
                    tma_load_pair(at + kABytes, &maps.w, kb * kBlock, row, bar);
                    tma_load_pair(at + kABytes + kBBytes, &maps.w, kb * kBlock, row + 128, bar);
                    ++ctl->issued;
                    if (++s == kStages) s = 0, phase ^= 1;
                }
            }
        }
    } else if (warp == kMmaWarp) {
        if (rank == 0) {
            constexpr uint32_t idesc = 1u << 4 | (128u >> 3) << 17 | (256u >> 4) << 24;
            int s = 0, d = 0;
            uint32_t phase = 0, d_phase = 1;
            bool go = true;
            for (int i = pair; go && i < n_tiles; i += pairs)
                for (int kb = 0; go && kb < a.nkb; ++kb) {
                    if (!mbar_wait_vote(&ctl->full[s], phase, &ctl->abort, a.status, 0xb12u)) {
                        go = false;
                        break;
                    }
                    const uint64_t xd = make_desc_sw128(ring + s * kStage);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (!mbar_wait_vote(&ctl->d_empty[h][d], d_phase, &ctl->abort, a.status, 0xb13u)) {
                            go = false;
                            break;
                        }
                        tc_fence_after();
                        if (elect_one()) {
                            const uint64_t wd = make_desc_sw128(ring + s * kStage + kABytes + h * kBBytes);
#pragma unroll
                            for (int k = 0; k < 4; ++k) mma_pair(tmem + (2 * h + d) * 128, xd + 2 * k, wd + 2 * k, idesc, k > 0);
                            if (h == 1) commit_pair(&ctl->empty[s]);
                            commit_pair(&ctl->d_full[h][d]);
                        }
                        __syncwarp();
                    }
                    if (++s == kStages) s = 0, phase ^= 1;
                    if (d ^= 1; d == 0) d_phase ^= 1;
                }
        }
    } else if (warp >= kScaleWarp0) {
        const int half = warp - kScaleWarp0;     // of the CTA's 128 tokens
        int b = 0;
        uint32_t phase = 1;
        bool go = true;
        for (int i = pair; go && i < n_tiles; i += pairs) {
            const Tile t = tile_of(ctl, a, i);
            const int first = rank * 128 + half * 64;
            const float *const ws = a.ws + (static_cast<size_t>(t.expert) * a.row_blocks + t.n0 / kBlock) * a.nkb;
            for (int kb = 0; kb < a.nkb; kb += kHeld) {
                if (!mbar_wait_vote(&ctl->s_empty[b], phase, &ctl->abort, a.status, 0xb14u)) {
                    go = false;
                    break;
                }
                float *const to = scales + b * kScaleFloats;
                const int k = lane & (kHeld - 1), r0 = lane / kHeld;         // two tokens at a time, 16 blocks of each
                const bool have = kb + k < a.nkb;
#pragma unroll
                for (int r = 0; r < 64; r += 32) {
                    float v[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int tok = first + r + 2 * j + r0;
                        v[j] = have && tok < t.ntok ? a.xs[static_cast<size_t>(t.tok0 + tok) * a.nkb + kb + k] : 0.0f;
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) to[k * kPitch + half * 64 + r + 2 * j + r0] = v[j];
                }
                if (half == 0) {
                    const bool there = have && t.n0 / kBlock + r0 < a.row_blocks;
                    to[kHeld * kPitch + lane] = there ? __ldg(ws + static_cast<size_t>(r0) * a.nkb + kb + k) : 0.0f;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl->s_full[b]);
                if (b ^= 1; b == 0) phase ^= 1;
            }
        }
    } else {
        const int h = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21) + h * 256;
        const uint32_t freed = on_cta(smem_u32(&ctl->d_empty[h][0]), 0);
        int d = 0, b = 0;
        uint32_t phase = 0, s_phase = 0;
        for (int i = pair; i < n_tiles; i += pairs) {
            const Tile t = tile_of(ctl, a, i);
            uint64_t acc[64] = {};
            for (int kb = 0; kb < a.nkb; ++kb) {
                const int at = kb % kHeld;
                const float *const held = scales + b * kScaleFloats;
                if (at == 0) mbar_wait(&ctl->s_full[b], s_phase, &ctl->abort, a.status, 0xb15u);
                const float f = held[at * kPitch + r] * held[kHeld * kPitch + h * kHeld + at];
                mbar_wait(&ctl->d_full[h][d], phase, &ctl->abort, a.status, 0xb16u);
                __syncwarp();
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 128; c += 32) {
                    uint32_t v[32];
                    tmem_ld<32>(lanes + d * 128 + c, v);
                    tmem_wait_ld();
                    if (c == 96) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) arrive_at(freed + d * 8);
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 2) fma2(acc[(c + j) / 2], v[j], v[j + 1], f, f);
                }
                if (d ^= 1; d == 0) phase ^= 1;
                if (at == kHeld - 1 || kb == a.nkb - 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl->s_empty[b]);
                    if (b ^= 1; b == 0) s_phase ^= 1;
                }
            }
            const int tok = rank * 128 + r, n = t.n0 + h * 128;
            if (tok >= t.ntok || ctl->abort) continue;
            const size_t out = static_cast<size_t>(t.tok0 + tok) * a.N + n;
            if (a.wide) {
#pragma unroll
                for (int c = 0; c < 128; c += 8)
                    if (n + c < a.N) {           // (N is a multiple of eight)
                        if (a.out_dt == MTC_BF16) store8<MTC_BF16>(a.out, out + c, acc, c / 2);
                        else if (a.out_dt == MTC_F16) store8<MTC_F16>(a.out, out + c, acc, c / 2);
                        else store8<MTC_F32>(a.out, out + c, acc, c / 2);
                    }
            } else {
#pragma unroll
                for (int c = 0; c < 128; c += 2) {
                    const float2 v = halves(acc[c / 2]);
                    if (n + c < a.N) st_from_f32(a.out, out + c, v.x, a.out_dt);
                    if (n + c + 1 < a.N) st_from_f32(a.out, out + c + 1, v.y, a.out_dt);
                }
            }
        }
    }
    __syncthreads();
    if (ctl->abort) {                            // gave up: let what is on its way arrive (the first CTA's barriers count both CTAs' copies)
        if (warp == kMmaWarp && rank == 0 && elect_one()) {
            commit_pair(&ctl->drained);
            drain_ring(&ctl->drained, 1, 1);
        } else if (warp == kLoadWarp && rank == 0 && lane == 0) {
            drain_ring(ctl->full, ctl->issued, kStages);
        }
        __syncthreads();
    }
    tc_fence_before();
    cluster_sync();                              // nobody leaves while the other may still arrive at its barriers or read its memory
    tc_fence_after();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512));
}

}  // namespace

bool fp8_pair_supported(int M, int N, int K, int n_experts, const void *x, const void *w) {
    return fp8_tile_supported(M, N, K, x, w) && n_experts <= kMaxExperts && static_cast<long long>(blocks(M) + n_experts) * blocks(N) < 0x7FFFFFFF;
}

cudaError_t launch_fp8_pair(Ctx *ctx, cudaStream_t st, const uint8_t *x, const float *xs, const uint8_t *w, const float *ws, const uint32_t *expert_offsets, void *out,
                            int M, int N, int K, int n_experts, int out_dt, std::string *why) {
    PArgs a{};
    a.xs = xs;
    a.ws = ws;
    a.expert_offsets = expert_offsets;
    a.out = out;
    a.status = ctx->d_status;
    a.M = M;
    a.N = N;
    a.nkb = blocks(K);
    a.n_experts = n_experts;
    a.col_tiles = (N + kCols - 1) / kCols;
    a.row_blocks = blocks(N);
    a.out_dt = out_dt;
    a.wide = N % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    PMaps maps;
    cudaError_t e = make_map_2d(&maps.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, static_cast<long long>(n_experts) * N, K, 64, kBlock, why);
    if (e == cudaSuccess) e = make_map_2d(&maps.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, M, K, 128, kBlock, why);
    if (e != cudaSuccess) return e;
    static PerDeviceAttr attr;
    if ((e = attr.set(fp8_pair_kernel, kSmemBytes)) != cudaSuccess) return e;
    const long long chunks = expert_offsets ? static_cast<long long>(std::min(M, n_experts)) + M / kTokens : (M + kTokens - 1) / kTokens, tiles = chunks * a.col_tiles;
    const int pairs = static_cast<int>(std::min<long long>(ctx->sm_count / 2, tiles));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.stream = st;
    cudaLaunchAttribute la[2];
    la[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    la[0].val.programmaticStreamSerializationAllowed = 1;
    la[1].id = cudaLaunchAttributeClusterDimension;
    la[1].val.clusterDim.x = 2;
    la[1].val.clusterDim.y = la[1].val.clusterDim.z = 1;
    cfg.attrs = la;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, fp8_pair_kernel, maps, a);
}

}  // namespace mtc
