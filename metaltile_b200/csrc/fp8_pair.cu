// Products of e4m3 codes with block scales on tcgen05, for many tokens (dense: fp8_mm; grouped by expert: fp8_gather_mm):
//
//   out[t, n] = sum_b xs[t, b] * ws[n / 128, b] * D_b[t, n],      D_b[t, n] = sum_{k in block b} x[t, k] * w[n, k]
//
// A pair of CTAs (a cluster of two SMs) owns a tile of 256 tokens x 256 weight rows: each SM holds 128 tokens of A and half of the weight
// rows of B, and the MMAs (cta_group::2, 256 x 256, kind::f8f6f4) read both.  A block of 128 codes is a chain of four of them into an
// accumulator of its own in tensor memory.  The epilogue takes it out, multiplies by xs * ws, one number a thread (lane = token, and a
// warp's 128 columns share their ws), and adds up in registers: 128 sums a thread, eight warps.
//
// What bounds it.  128 x 256 x 128 products take an SM 512 cycles at the dense rate, and a tile of 256 x 256 needs 32 KB a block on each SM
// of a pair: 64 bytes a cycle, as many as an SM gets from L2; one CTA by itself with 128 x 256 would need 96.  Without the epilogue the
// ring and the MMAs run at 585 cycles a block.  With it a block takes 780 to 840, the MMA warp waiting for an accumulator: two are all of
// the tensor memory, so a block's MMAs (512), the way to the epilogue, its four loads of tensor memory in a row, the way back and the issue
// of the next are one chain for two blocks.  But no single link is the bound (1184 x 4096 x 28672, 838 cycles a block): handed back before
// it is read 822, one load of four 800, no additions 755, all three together 746; what takes the rest down to 585 is not known.  Waits that
// spin instead of sleeping slow the others' shared memory (2 to 8 % more).  A tile ends with 2300 cycles of stores (f32 4000) and 300 to
// 900 to find the next; MMAs of two blocks run beside that.  2048 x 28672 x 4096: 212 us, 2.27 PFLOP/s, in a graph of some ten calls at full
// clock; back to back for seconds, at the 1.49 GHz of the power limit, 248 us, 1.94 PFLOP/s.
//
// Steps on the way (us for that case at full clock): hand-offs that release at cluster scope 587, relaxed ones 348; one try in front of the
// polling loop, whose entry costs 200 cycles, and results out by TMA instead of a row a lane 303; the registers of the other roles for the
// epilogue, so that nothing spills, and the next columns loaded while the last are added 235; MMAs of 256 columns instead of two chains of
// 128, which read A twice, 226; 32-bit addresses and one plain loop over the blocks in the epilogue 214.  16 epilogue warps of 64 columns:
// 264 (96 registers each spill).
//
//   warps 0-7    epilogue   warps 0-3 the first half of the weight rows, 4-7 the second
//   warps 8-9    scales     xs of 128 tokens, 16 blocks at a time, and ws, by cp.async into shared memory (a load of each lane's own row would cost the load pipe ten
//                           cycles a lane)
//   warp 10      producer   TMA, both CTAs of a pair into their own memory, one barrier in the first
//   warp 11      MMA        issued by the first CTA
// A persistent pair walks the tiles, tokens fastest.  Every wait is bounded: on expiry the kernel records a code in the status word, the
// roles leave and what is in flight is awaited (bounded too).
#include <cstddef>

#include "fp8_tc.cuh"

namespace mtc {
namespace {

using namespace fp8;

constexpr int kTokens = 256, kCols = 256;        // of a tile; a CTA of a pair has 128 of the tokens
constexpr int kABytes = 128 * kBlock, kBBytes = 128 * kBlock, kStage = kABytes + kBBytes;
constexpr int kStages = 4;                       // (five: the same)
constexpr int kOutBytes = 4096;                  // of an epilogue warp: 32 rows x 128 bytes of results on their way out
constexpr int kEpiWarps = 8, kScaleWarp0 = 8, kScaleWarps = 2, kLoadWarp = 10, kMmaWarp = 11, kThreads = 384;
constexpr int kHeld = 16, kPitch = 20;           // blocks whose scales are in shared memory, floats of a row of xs
constexpr int kScaleFloats = 128 * kPitch + 2 * kHeld;
constexpr int kMaxExperts = 1024;

struct PArgs {
    const float *xs, *ws;
    const uint32_t *expert_offsets;              // nullptr: dense
    void *out;
    uint32_t *status;
    int M, N, nkb, n_experts;
    int chunks;                                  // of 256 tokens; grouped: the most that offsets in order make
    int col_tiles, row_blocks;                   // ceil(N / 256), ceil(N / 128)
    int out_dt;
    int wide;                                    // rows of the output are whole 16-byte pieces at 16-byte boundaries: `out` of the maps holds
};
struct PMaps {
    CUtensorMap x, w, out;
};
struct __align__(16) PCtrl {
    uint64_t full[kStages], empty[kStages], d_full[2], d_empty[2], s_full[2], s_empty[2], drained;
    uint32_t tmem_base, issued;
    volatile uint32_t abort;
    uint32_t n_chunks;
    uint32_t first_chunk[kMaxExperts + 1];       // grouped: chunks of 256 tokens of the experts before
    uint32_t offset[kMaxExperts + 1];            // and the clamped offsets
};
constexpr int kCtlBytes = (sizeof(PCtrl) + 1023) / 1024 * 1024;
constexpr int kScaleBytes = (2 * kScaleFloats * 4 + 1023) / 1024 * 1024;
constexpr int kSmemBytes = 1024 + kCtlBytes + kScaleBytes + 8 * kOutBytes + kStages * kStage;
static_assert(kSmemBytes <= 227 * 1024, "shared memory");
static_assert(kStages * kStage >= 128 * kCols * 4, "the sums of a slice go where the ring was");

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
// arrives at the barrier of this offset in both CTAs (a bit each of their rank in the cluster) when the MMAs so far are complete
__device__ __forceinline__ void commit_pair(uint64_t *bar, uint32_t both) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"(static_cast<uint16_t>(both)) : "memory");
}
// Relaxed: what it hands over is tensor memory, ordered by the tcgen05 fence in front.  (A release at cluster scope waits for everything
// the thread has in flight: 1150 cycles a block, 2048 x 28672 x 4096 in 587 us instead of 348.)
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// The chunks of the experts, by one warp: ceil(rows / 256) each.  Offsets that run backwards or past the rows are clamped and reported.
__device__ void count_chunks(PCtrl *ctl, const PArgs &a) {
    const int lane = threadIdx.x & 31;
    constexpr uint32_t kMany = 0x7FFFFFFFu;      // sums end there: offsets that run backwards may hold any number of rows
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
            if (lane >= d) upto = min(upto + v, kMany);
        }
        if (e < a.n_experts) {
            ctl->first_chunk[e] = min(before + (upto - np), kMany);
            ctl->offset[e] = lo;
        }
        before = min(before + __shfl_sync(0xffffffffu, upto, 31), kMany);
    }
    if (lane == 0) {
        ctl->first_chunk[a.n_experts] = before;
        ctl->n_chunks = min(before, static_cast<uint32_t>(a.chunks));
    }
}

// Waits of the epilogue by addresses: its registers are sums and values on their way, and a 64-bit pointer more makes them spill.  Not
// inlined: the way that rarely runs.
__device__ __noinline__ void wait_long(uint32_t bar, uint32_t parity, uint32_t abort, uint32_t *status, uint32_t code) {
    const uint32_t r = mbar_poll(bar, parity, abort);
    if (r != 1) mbar_gave_up(r, abort, status, code);
}
__device__ __forceinline__ void wait_at(uint32_t bar, uint32_t parity, uint32_t abort, uint32_t *status, uint32_t code) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (!ok) wait_long(bar, parity, abort, status, code);
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

// Sixteen bytes of neighbouring results from the sums acc[i] on: eight of 16 bits, four of 32
template <int DT, int N>
__device__ __forceinline__ uint4 piece(const uint64_t (&acc)[N], int i) {
    uint32_t w[4];
    if constexpr (DT == MTC_F32) {
        const float2 lo = halves(acc[i]), hi = halves(acc[i + 1]);
        return make_uint4(__float_as_uint(lo.x), __float_as_uint(lo.y), __float_as_uint(hi.x), __float_as_uint(hi.y));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 v = halves(acc[i + j]);
            if constexpr (DT == MTC_BF16) {
                const __nv_bfloat162 p = __floats2bfloat162_rn(v.x, v.y);
                w[j] = *reinterpret_cast<const uint32_t *>(&p);
            } else {
                const __half2 p = __floats2half2_rn(v.x, v.y);
                w[j] = *reinterpret_cast<const uint32_t *>(&p);
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// A warp's rows (32 at most) x NC columns, through shared memory, 128 bytes a row at a time: all 32 rows out by TMA, which goes on while
// the next tile's blocks are added; fewer, or rows that 16-byte pieces do not fit, by stores that run along the rows.  (A lane storing its
// own row costs the load pipe a cycle a row and store: 67 us of 330 for 2048 x 28672 x 4096 in 16-byte pieces, and 30 us for one tile of
// odd rows, element by element.)
template <int DT, int NC>
__device__ __forceinline__ void store_rows_as(const PMaps &maps, const PArgs &a, const uint64_t (&acc)[NC / 2], uint32_t staged, int row, int rows, int n) {
    constexpr int PER = DT == MTC_F32 ? 4 : 8;                       // results of a 16-byte piece
    constexpr int NP = NC < 8 * PER ? NC / PER : 8;                  // pieces of a row at a time
    const int lane = threadIdx.x & 31;
    const bool whole = NP == 8 && a.wide && rows >= 32;
#pragma unroll
    for (int c = 0; c < NC; c += NP * PER) {
        if (n + c >= a.N) break;
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            const uint4 v = piece<DT>(acc, (c + q * PER) / 2);
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(staged + lane * 128 + ((q ^ (lane & 7)) << 4)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
        }
        if (whole) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
                             ::"l"(reinterpret_cast<uint64_t>(&maps.out)), "r"(n + c), "r"(row), "r"(staged) : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
            continue;
        }
        __syncwarp();
        if (a.wide) {                            // NP lanes a row
            const int q = lane % NP;
            if (n + c + q * PER < a.N) {
                for (int i = lane / NP; i < min(rows, 32); i += 32 / NP) {
                    uint4 v;
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(staged + i * 128 + ((q ^ (i & 7)) << 4)));
                    *reinterpret_cast<uint4 *>(static_cast<char *>(a.out) + (static_cast<size_t>(row + i) * a.N + n + c + q * PER) * (16 / PER)) = v;
                }
            }
        } else {
            for (int i = 0; i < min(rows, 32); ++i)
#pragma unroll
                for (int e = lane; e < NP * PER; e += 32) {
                    if (n + c + e >= a.N) break;
                    const uint32_t from = staged + i * 128 + (((e / PER) ^ (i & 7)) << 4) + e % PER * (16 / PER);
                    const size_t to = static_cast<size_t>(row + i) * a.N + n + c + e;
                    if constexpr (DT == MTC_F32) {
                        uint32_t v;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(from));
                        static_cast<uint32_t *>(a.out)[to] = v;
                    } else {
                        uint16_t v;
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(from));
                        static_cast<uint16_t *>(a.out)[to] = v;
                    }
                }
        }
        __syncwarp();                            // read before the next piece is written
    }
}

template <int NC>
__device__ __forceinline__ void store_rows(const PMaps &maps, const PArgs &a, const uint64_t (&acc)[NC / 2], uint32_t staged, int row, int rows, int n) {
    if (rows <= 0 || n >= a.N) return;
    if (a.out_dt == MTC_BF16) store_rows_as<MTC_BF16, NC>(maps, a, acc, staged, row, rows, n);
    else if (a.out_dt == MTC_F16) store_rows_as<MTC_F16, NC>(maps, a, acc, staged, row, rows, n);
    else store_rows_as<MTC_F32, NC>(maps, a, acc, staged, row, rows, n);
}

// The sums of all S slices of this CTA's tokens, and out: a warp its 32 tokens x 128 / S columns, 32 at a time.  Sums lie as
// [column][token] where the ring was, in the CTAs of the same rank of each pair; they are added in the order of K.
template <int S>
__device__ __forceinline__ void join_slices(const PMaps &maps, const PArgs &a, uint32_t sums, uint32_t staged, int slice, int rank, int first, int rows, const Tile &t) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll 1
    for (int p = 0; p < 4 / S; ++p) {
        const int c0 = (warp >> 2) * 128 + (slice * (4 / S) + p) * 32;
        uint64_t acc[16];
#pragma unroll
        for (int c = 0; c < 32; c += 16) {       // sixteen columns in flight
            float v[S][16];
#pragma unroll
            for (int q = 0; q < S; ++q) {
                const uint32_t from = on_cta(sums + ((c0 + c) * 128 + (warp & 3) * 32 + lane) * 4, 2 * q + rank);
#pragma unroll
                for (int i = 0; i < 16; ++i) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[q][i]) : "r"(from + i * 512) : "memory");
            }
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                float lo = v[0][i], hi = v[0][i + 1];
#pragma unroll
                for (int q = 1; q < S; ++q) lo += v[q][i], hi += v[q][i + 1];
                asm("mov.b64 %0, {%1, %2};" : "=l"(acc[(c + i) / 2]) : "f"(lo), "f"(hi));
            }
        }
        store_rows<32>(maps, a, acc, staged + warp * kOutBytes, t.tok0 + first, rows, t.n0 + c0);
    }
}

// Registers: 384 threads start with 168, 256 of them go on with more and 128 with fewer.  What leaves the epilogue's loop without spills,
// or with the fewest.
template <int SLICES>
constexpr int kEpiRegs = SLICES == 4 ? 216 : 224;
template <int SLICES>
constexpr int kOtherRegs = 3 * 168 - 2 * kEpiRegs<SLICES>;

// SLICES of K: pairs of a cluster that own a tile together; 1: a pair walks tiles.
template <int SLICES>
__global__ void __launch_bounds__(kThreads, 1) fp8_pair_kernel(const __grid_constant__ PMaps maps, const __grid_constant__ PArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *const smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    PCtrl *const ctl = reinterpret_cast<PCtrl *>(smem);
    float *const scales = reinterpret_cast<float *>(smem + kCtlBytes);       // two of [128][kPitch] of xs, [2][kHeld] of ws
    const uint32_t staged = __shfl_sync(0xffffffffu, smem_u32(smem), 0) + kCtlBytes + kScaleBytes, ring = staged + kEpiWarps * kOutBytes;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int in_cluster = static_cast<int>(blockIdx.x) % (2 * SLICES), rank = in_cluster & 1, slice = in_cluster >> 1, leader = SLICES == 1 ? 0 : in_cluster & ~1;
    const int pair = static_cast<int>(blockIdx.x) / (2 * SLICES), pairs = static_cast<int>(gridDim.x) / (2 * SLICES);
    const int kb0 = SLICES == 1 ? 0 : static_cast<int>(static_cast<long long>(a.nkb) * slice / SLICES);
    const int kb1 = SLICES == 1 ? a.nkb : static_cast<int>(static_cast<long long>(a.nkb) * (slice + 1) / SLICES);
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&ctl->full[s], 1);
            mbar_init(&ctl->empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&ctl->d_full[i], 1);
            mbar_init(&ctl->d_empty[i], 2 * kEpiWarps);              // those of both CTAs, in the first one's memory
            mbar_init(&ctl->s_full[i], 32 * kScaleWarps);
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
        if (threadIdx.x == 0) ctl->n_chunks = a.chunks;
    } else if (warp == 0) {
        count_chunks(ctl, a);
    }
    tc_fence_before();
    cluster_sync();                              // both CTAs' barriers exist
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
    const int n_tiles = static_cast<int>(ctl->n_chunks) * a.col_tiles;

    if (warp == kLoadWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs<SLICES>));
        if (lane == 0) {
            int s = 0;
            uint32_t phase = 1;
            bool go = true;
            for (int i = pair; go && i < n_tiles; i += pairs) {
                const Tile t = tile_of(ctl, a, i);
                const int row = static_cast<int>(static_cast<long long>(t.expert) * a.N) + t.n0 + rank * 128;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!wait_soon(&ctl->empty[s], phase, &ctl->abort, a.status, 0xb11u)) {
                        go = false;
                        break;
                    }
                    const uint32_t at = ring + s * kStage, bar = on_cta(smem_u32(&ctl->full[s]), leader);
                    if (rank == 0) mbar_expect_tx(&ctl->full[s], 2 * kStage);
                    tma_load_pair(at, &maps.x, kb * kBlock, t.tok0 + rank * 128, bar);
                    tma_load_pair(at + kABytes, &maps.w, kb * kBlock, row, bar);
                    ++ctl->issued;
                    if (++s == kStages) s = 0, phase ^= 1;
                }
            }
            // The MMAs' arrivals at `empty` come through the cluster on their own: the last ones are awaited too, so that none reaches a
            // CTA that has left
            for (int i = 0; go && i < kStages; ++i) {
                go = wait_soon(&ctl->empty[s], phase, &ctl->abort, a.status, 0xb11u);
                if (++s == kStages) s = 0, phase ^= 1;
            }
        }
    } else if (warp == kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs<SLICES>));
        if (rank == 0) {                         // the whole warp walks the loop, so that the operands of the MMAs are uniform; one thread issues
            constexpr uint32_t idesc = 1u << 4 | (256u >> 3) << 17 | (256u >> 4) << 24;
            int s = 0, d = 0;
            uint32_t phase = 0, d_phase = 1;
            bool go = true;
            for (int i = pair; go && i < n_tiles; i += pairs)
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!wait_all(&ctl->full[s], phase, &ctl->abort, a.status, 0xb12u)) {
                        go = false;
                        break;
                    }
                    const uint64_t xd = make_desc_sw128(ring + s * kStage), wd = make_desc_sw128(ring + s * kStage + kABytes);
                    if (!wait_all(&ctl->d_empty[d], d_phase, &ctl->abort, a.status, 0xb13u)) {
                        go = false;
                        break;
                    }
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) mma_pair(tmem + d * 256, xd + 2 * k, wd + 2 * k, idesc, k > 0);
                        commit_pair(&ctl->d_full[d], 3u << leader);
                        commit_pair(&ctl->empty[s], 3u << leader);
                    }
                    __syncwarp();
                    if (++s == kStages) s = 0, phase ^= 1;
                    if (d ^= 1; d == 0) d_phase ^= 1;
                }
        }
    } else if (warp >= kScaleWarp0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs<SLICES>));
        const int half = warp - kScaleWarp0;     // of the CTA's 128 tokens
        const int k = lane & (kHeld - 1), r0 = lane / kHeld;
        int b = 0;
        uint32_t phase = 1;
        bool go = true;
        for (int i = pair; go && i < n_tiles; i += pairs) {
            const Tile t = tile_of(ctl, a, i);
            const int first = rank * 128 + half * 64;
            const float *const ws = a.ws + (static_cast<size_t>(t.expert) * a.row_blocks + t.n0 / kBlock) * a.nkb;
            for (int kb = kb0; kb < kb1; kb += kHeld) {
                if (!mbar_wait_vote(&ctl->s_empty[b], phase, &ctl->abort, a.status, 0xb14u)) {
                    go = false;
                    break;
                }
                // two tokens at a time, 16 blocks of each; what does not exist is filled with zeros
                const uint32_t to = smem_u32(scales) + (b * kScaleFloats + (half * 64 + r0) * kPitch + k) * 4;
                const float *const from = a.xs + static_cast<size_t>(t.tok0 + first + r0) * a.nkb + kb + k;
                const int last = kb + k < kb1 ? t.ntok - first - r0 : 0;
#pragma unroll 8
                for (int r = 0; r < 64; r += 2)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + r * kPitch * 4), "l"(r < last ? from + static_cast<size_t>(r) * a.nkb : a.xs), "r"(r < last ? 4 : 0) : "memory");
                if (half == 0) {
                    const bool there = kb + k < kb1 && t.n0 / kBlock + r0 < a.row_blocks;
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(scales) + (b * kScaleFloats + 128 * kPitch + lane) * 4),
                                 "l"(there ? ws + static_cast<size_t>(r0) * a.nkb + kb + k : a.ws), "r"(there ? 4 : 0) : "memory");
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&ctl->s_full[b])) : "memory");
                if (b ^= 1; b == 0) phase ^= 1;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs<SLICES>));
        const int h = warp >> 2;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21) + h * 128;
        const uint32_t bars = staged - kCtlBytes - kScaleBytes;                          // the control block
        const uint32_t freed = on_cta(bars + offsetof(PCtrl, d_empty), leader);
        const uint32_t xs_at = bars + kCtlBytes + ((warp & 3) * 32 + lane) * kPitch * 4, ws_at = bars + kCtlBytes + (128 * kPitch + h * kHeld) * 4;
        int d = 0, b = 0;
        uint32_t phase = 0, s_phase = 0;
        for (int i = pair; i < n_tiles; i += pairs) {
            uint64_t acc[64] = {};
            uint32_t v[2][32];                   // the next columns are on their way while these are added
#pragma unroll 1
            for (int kb = kb0; kb < kb1; ++kb) {
                const int at = (kb - kb0) % kHeld;
                if (at == 0) wait_at(bars + offsetof(PCtrl, s_full) + b * 8, s_phase, bars + offsetof(PCtrl, abort), a.status, 0xb15u);
                const float f = ld_shared(xs_at + (b * kScaleFloats + at) * 4) * ld_shared(ws_at + (b * kScaleFloats + at) * 4);
                wait_at(bars + offsetof(PCtrl, d_full) + d * 8, phase, bars + offsetof(PCtrl, abort), a.status, 0xb16u);
                __syncwarp();
                tc_fence_after();
                tmem_ld<32>(lanes + d * 256, v[0]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    tmem_wait_ld(v[c & 1]);
                    if (c < 3) {
                        tmem_ld<32>(lanes + d * 256 + (c + 1) * 32, v[~c & 1]);
                    } else {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) arrive_at(freed + d * 8);
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 2) fma2(acc[c * 16 + j / 2], v[c & 1][j], v[c & 1][j + 1], f, f);
                }
                if (d ^= 1; d == 0) phase ^= 1;
                if (at == kHeld - 1 || kb == kb1 - 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bars + offsetof(PCtrl, s_empty) + b * 8);
                    if (b ^= 1; b == 0) s_phase ^= 1;
                }
            }
            const Tile t = tile_of(ctl, a, i);
            if (ctl->abort) continue;
            if constexpr (SLICES == 1) {
                const int first = rank * 128 + (warp & 3) * 32;
                store_rows<128>(maps, a, acc, staged + warp * kOutBytes, t.tok0 + first, t.ntok - first, t.n0 + h * 128);
            } else {                             // the only tile of this cluster: its copies have all arrived, and its MMAs have read them
#pragma unroll
                for (int c = 0; c < 128; c += 2) {
                    const float2 v2 = halves(acc[c / 2]);
                    const uint32_t to = ring + ((h * 128 + c) * 128 + (warp & 3) * 32 + lane) * 4;
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(to), "f"(v2.x) : "memory");
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + 512), "f"(v2.y) : "memory");
                }
            }
        }
        if constexpr (SLICES > 1) {
            cluster_sync();                      // the sums of all slices are there
            if (pair < n_tiles && !ctl->abort) {
                const Tile t = tile_of(ctl, a, pair);
                const int first = rank * 128 + (warp & 3) * 32;
                join_slices<SLICES>(maps, a, ring, staged, slice, rank, first, t.ntok - first, t);
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    if (SLICES > 1 && warp >= kEpiWarps) {     // (the epilogue met this barrier above)
        __syncwarp();
        cluster_sync();
    }
    __syncthreads();
    if (ctl->abort) {                            // gave up: let what is on its way arrive (the first CTA's barriers count both CTAs' copies)
        if (warp == kMmaWarp && rank == 0 && elect_one()) {
            commit_pair(&ctl->drained, 1u << leader);            // (the other CTA does not wait for it)
            drain_ring(&ctl->drained, 1, 1);
        } else if (warp == kLoadWarp && rank == 0 && lane == 0) {
            drain_ring(ctl->full, ctl->issued, kStages);
        }
        __syncthreads();
    }
    tc_fence_before();
    cluster_sync();                              // nobody leaves while the other's threads may still arrive at its barriers or read its memory
    tc_fence_after();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512));
}

template <int S>
cudaError_t config(cudaLaunchConfig_t &cfg, cudaLaunchAttribute (&la)[2], cudaStream_t st, long long clusters) {
    static PerDeviceAttr attr;
    const cudaError_t e = attr.set(fp8_pair_kernel<S>, kSmemBytes);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3(static_cast<unsigned>(clusters * 2 * S));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.stream = st;
    la[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    la[0].val.programmaticStreamSerializationAllowed = 1;
    la[1].id = cudaLaunchAttributeClusterDimension;
    la[1].val.clusterDim.x = 2 * S;
    la[1].val.clusterDim.y = la[1].val.clusterDim.z = 1;
    cfg.attrs = la;
    cfg.numAttrs = 2;
    return cudaSuccess;
}
template <int S>
cudaError_t launch(cudaStream_t st, const PMaps &maps, const PArgs &a, long long clusters) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute la[2];
    const cudaError_t e = config<S>(cfg, la, st, clusters);
    return e != cudaSuccess ? e : cudaLaunchKernelEx(&cfg, fp8_pair_kernel<S>, maps, a);
}
// Clusters that the device runs at once: asked for once a device (clusters have to fit into groups of SMs of different sizes).  0 where it
// cannot be told.
template <int S>
int clusters_at_once() {
    static std::atomic<int> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    int n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute la[2];
        if (config<S>(cfg, la, nullptr, 1) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, fp8_pair_kernel<S>, &cfg) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            n = -1;
        }
        known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

}  // namespace

bool fp8_pair_supported(int M, int N, int K, int n_experts, const void *x, const void *w) {
    return fp8_tile_supported(M, N, K, n_experts, x, w) && n_experts <= kMaxExperts && static_cast<long long>(blocks(M) + n_experts) * blocks(N) < 0x7FFFFFFF;
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
    const int size = static_cast<int>(dtype_size(out_dt));
    a.wide = static_cast<long long>(N) * size % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    PMaps maps{};
    cudaError_t e = make_map_2d(&maps.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, static_cast<long long>(n_experts) * N, K, 128, kBlock, why);
    if (e == cudaSuccess) e = make_map_2d(&maps.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, M, K, 128, kBlock, why);
    if (e == cudaSuccess && a.wide)
        e = make_map_2d(&maps.out, size == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, size, out, M, N, 32, 128 / size, why);
    if (e != cudaSuccess) return e;
    const long long chunks = expert_offsets ? static_cast<long long>(std::min(M, n_experts)) + M / kTokens : (M + kTokens - 1) / kTokens, tiles = chunks * a.col_tiles;
    if (tiles > kMostSize) return cudaErrorInvalidConfiguration;
    a.chunks = static_cast<int>(chunks);
    // K slices where tiles would leave SMs without work, all clusters at once (15 of four pairs, 33 of two).  Joining them takes 3 us: 256
    // x 4096 x 4096 18.3 us, in two slices 16.2; x 14336 50.1 and 34.3; 256 x 1024 x 4096 17.7, in four 13.0; but x 2048 11.6 to 11.8 and
    // 12.1 to 12.4.
    if (!expert_offsets && a.nkb >= 24 && tiles <= clusters_at_once<4>()) return launch<4>(st, maps, a, tiles);
    if (!expert_offsets && a.nkb >= 24 && tiles <= clusters_at_once<2>()) return launch<2>(st, maps, a, tiles);
    return launch<1>(st, maps, a, std::min<long long>(ctx->sm_count / 2, tiles));
}

}  // namespace mtc
