// Products of e4m3 codes with block scales on tcgen05, for few tokens a tile (dense: fp8_mm; grouped by expert: fp8_gather_mm):
//
//   out[t, n] = sum_b xs[t, b] * ws[n / 128, b] * D_b[n, t],      D_b[n, t] = sum_{k in block b} w[n, k] * x[t, k]
//
// An item is 128 weight rows x up to TN tokens x a slice of K.  Its weight rows share ws, so a block of 128 codes is one MMA chain (four
// steps of K = 32, kind::f8f6f4) into an accumulator of its own in tensor memory, which the epilogue takes out, multiplies by xs * ws and
// adds up in registers: lane = weight row, register = token.  The products and block sums are the tensor core's (codes have 4 bits, their
// products are exact), the sums over blocks f32.
//
// Bound by reading the weights once: a block of an item is 16 KB of them, 700 cycles of an SM's share of the memory's rate, against 128
// cycles of MMAs.  Two CTAs an SM with some 100 KB of stages each walk the items, the copies running ahead from one to the next; with few
// items and no experts K is cut into up to 8 slices, the CTAs of a cluster, which add up through shared memory in the order of K.  What an
// item takes beside its bytes is the way through the hand-offs: a wait, a load of tensor memory and the sums were 470 cycles a block,
// whatever its columns, so two or four blocks make one hand-off.  Measured (graph, us): 1 x 4096 x 4096 7.3, 1 x 14336 x 4096 14 (58.7 MB;
// each further matrix of that size 9.4, the memory's rate).
//
//   warps 0-3  epilogue   accumulators out, scaled, added up, stored
//   warp 4     producer   TMA: 128 x 128 codes of the weights, TN x 128 of the tokens, a stage; by cp.async the scales of 16 blocks
//   warp 5     MMA        and the tensor memory's allocation
// Every wait is bounded: on expiry the kernel records a code in the status word, the roles leave, copies and MMAs in flight are awaited
// (bounded too).
#include <cstddef>

#include "fp8_tc.cuh"

namespace mtc {
namespace {

using namespace fp8;

constexpr int kRows = 128;                       // weight rows of an item: TMEM lanes, MMA M; they share their scales
constexpr int kWBytes = kRows * kBlock;          // of a stage
constexpr int kMaxStages = 8;
constexpr int kEpi = 128, kLoadWarp = 4, kMmaWarp = 5, kThreads = 192, kPerSM = 2;
constexpr int kSmemBytes = 113 * 1024;           // of one of the two CTAs of an SM
constexpr int kMaxSlices = 8;

// SLICED: slices of K meet in shared memory.  A token's sums go to the CTA of rank token % slices, one place a slice, by stores that nobody
// waits for before the barrier of the cluster: (a + i * slices) has i-th place.  Tiles of 64 tokens have no room beside the ring and are
// fetched from where it was, after the barrier.
template <int TN, bool SLICED>
struct Form {
    static constexpr int kTogether = TN == 64 ? 2 : 4;               // blocks of a hand-off to the epilogue
    static constexpr int kCols = 2 * kTogether * TN;                 // two hand-offs in tensor memory
    static constexpr int kStep = TN < 32 ? TN : 32, kLoads = 64 / kStep;      // columns of a load of tensor memory, loads at a time
    static constexpr int kHeld = 16;                                 // blocks whose scales are in shared memory, [block][token], twice
    static constexpr int kPitch = TN + 4;
    static constexpr int kStage = kWBytes + TN * kBlock;
    static constexpr int kScales = kHeld * (kPitch + 1);             // floats: xs, then ws of the blocks
    static constexpr bool kPush = SLICED && TN < 64;
    static constexpr int kJoin = 1024 + (2 * kScales * 4 + 1023) / 1024 * 1024;          // where the slices' sums come in
    static constexpr int kRing = kJoin + (kPush ? (TN + kMaxSlices) * kRows * 4 : 0);    // where the stages start
    static constexpr int kStages = (kSmemBytes - 1024 - kRing) / kStage;
    static_assert(kStages >= 2 && kStages <= kMaxStages, "stages");
    static_assert(kStages * kStage >= TN * kRows * 4, "the sums of a slice go where the ring was");
};

struct TArgs {
    const float *xs, *ws;
    const uint32_t *expert_offsets;              // nullptr: dense
    void *out;
    uint32_t *status;
    int M, N, nkb, n_experts;
    int tiles;                                   // of 128 weight rows
    int chunks;                                  // dense: of TN tokens; grouped: the most that offsets in order make
    int slices;
    int out_dt;
    int early;                                   // weights may be requested before the previous kernel is complete
};
struct TMaps {
    CUtensorMap w, x;
};

struct __align__(16) TCtrl {
    uint64_t full[kMaxStages], empty[kMaxStages], d_full[2], d_empty[2], s_full[2], s_empty[2], drained;
    uint32_t tmem_base, issued;
    volatile uint32_t abort;
    int chunk[2][3];                             // first token, tokens and tile of the item whose scales are in each half: the producer found them
    int n_chunks;                                // of all experts, or of the dense rows
};
static_assert(sizeof(TCtrl) <= 1024, "control block");

__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
    uint32_t there;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
    return v;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t rank, float v) {
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there), "f"(v) : "memory");
}
__device__ __forceinline__ void st_shared(uint32_t addr, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }

// Chunks of TN rows: expert e with r rows has ceil(r / TN).  By one warp, four experts a lane: how many there are in all (want < 0), or the
// one with index `want`.  Offsets that run backwards or past the rows are clamped, and reported by the block that is told to.  (A load and
// a scan for 128 experts; with one for 32 128 experts of 768 x 2048 and 32 rows in all 14.7 us for 13.1, 4096 rows 46.0 for 43.4, 512
// experts of 512 x 1024 and 512 rows 43.4 for 34.9.)
struct Chunk {
    int expert, tok0, ntok;
};
__device__ __forceinline__ int find_chunk(const uint32_t *offsets, int n_experts, int m_total, int TN, int want, uint32_t *status, Chunk &found) {
    constexpr uint32_t kMany = 0x7FFFFFFFu;      // sums end there: offsets that run backwards may hold any number of rows
    const int lane = threadIdx.x & 31;
    const uint32_t m = static_cast<uint32_t>(m_total);
    uint32_t before = 0;
    for (int e0 = 0; e0 < n_experts; e0 += 128) {
        uint32_t at[5];                          // (behind the last expert: its end, no rows)
#pragma unroll
        for (int i = 0; i < 5; ++i) at[i] = offsets[min(e0 + 4 * lane + i, n_experts)];
        bool wrong = at[0] > m;
        int lo[4], hi[4];
        uint32_t own = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            wrong |= at[i + 1] > m || at[i + 1] < at[i];
            lo[i] = static_cast<int>(min(at[i], m));
            hi[i] = max(lo[i], static_cast<int>(min(at[i + 1], m)));
            own += (hi[i] - lo[i] + TN - 1) / TN;
        }
        if (status && wrong) atomicCAS(status, 0u, 0x901u);
        uint32_t upto = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto = min(upto + v, kMany);
        }
        int mine = want - static_cast<int>(before) - static_cast<int>(upto - own);     // index of the wanted chunk among this lane's
        const uint32_t has = __ballot_sync(0xffffffffu, want >= 0 && mine >= 0 && mine < static_cast<int>(own));
        if (has) {
            int expert = 0, tok0 = 0, ntok = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int np = (hi[i] - lo[i] + TN - 1) / TN;
                if (mine >= 0 && mine < np) {
                    expert = e0 + 4 * lane + i;
                    tok0 = lo[i] + mine * TN;
                    ntok = min(TN, hi[i] - tok0);
                }
                mine -= np;
            }
            const int src = __ffs(has) - 1;
            found.expert = __shfl_sync(0xffffffffu, expert, src);
            found.tok0 = __shfl_sync(0xffffffffu, tok0, src);
            found.ntok = __shfl_sync(0xffffffffu, ntok, src);
            return want;
        }
        before = min(before + __shfl_sync(0xffffffffu, upto, 31), kMany);
    }
    return static_cast<int>(before);
}

// Giving up, once every role has ended: lets what is on its way arrive before the CTA tears down.
__device__ __noinline__ void rest(TCtrl *ctl, int stages) {
    const int warp = threadIdx.x >> 5;
    if (warp == kMmaWarp && elect_one()) {
        umma_commit(&ctl->drained);
        drain_ring(&ctl->drained, 1, 1);
    } else if (warp == kLoadWarp && (threadIdx.x & 31) == 0) {
        drain_ring(ctl->full, ctl->issued, stages);
    }
    __syncthreads();
}

template <int TN, bool SLICED>
__global__ void __launch_bounds__(kThreads, kPerSM) fp8_tile_kernel(const __grid_constant__ TMaps maps, const __grid_constant__ TArgs a) {
    using F = Form<TN, SLICED>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *const smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    TCtrl *const ctl = reinterpret_cast<TCtrl *>(smem);
    float *const scales = reinterpret_cast<float *>(smem + 1024);    // two of kScales
    const uint32_t ring = __shfl_sync(0xffffffffu, smem_u32(smem), 0) + F::kRing;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = static_cast<int>(blockIdx.x % a.slices), first = static_cast<int>(blockIdx.x / a.slices), step = static_cast<int>(gridDim.x / a.slices);
    const int kb0 = static_cast<int>(static_cast<long long>(a.nkb) * rank / a.slices), kb1 = static_cast<int>(static_cast<long long>(a.nkb) * (rank + 1) / a.slices);
    if (threadIdx.x == 0) {
        for (int s = 0; s < F::kStages; ++s) {
            mbar_init(&ctl->full[s], 1);
            mbar_init(&ctl->empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&ctl->d_full[s], 1);
            mbar_init(&ctl->d_empty[s], kEpi / 32);
            mbar_init(&ctl->s_full[s], 33);
            mbar_init(&ctl->s_empty[s], kEpi / 32);
        }
        mbar_init(&ctl->drained, 1);
        ctl->abort = 0;
        ctl->issued = 0;
        if (!a.expert_offsets) ctl->n_chunks = a.chunks;         // (grouped: the producer counts them, and nobody else stores there)
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)), "n"(F::kCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (a.expert_offsets) {
        pdl_enter();
        if (warp == kLoadWarp) {
            Chunk none;
            const int n = find_chunk(a.expert_offsets, a.n_experts, a.M, TN, -1, blockIdx.x == 0 ? a.status : nullptr, none);
            __syncwarp();
            if (lane == 0) ctl->n_chunks = min(n, a.chunks);         // offsets that run backwards may hold rows many times over
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
    const int units = ctl->n_chunks * a.tiles;
    if constexpr (SLICED) asm volatile("barrier.cluster.arrive.relaxed.aligned;");        // this CTA runs: awaited before anything is stored into another
    // grouped: the tiles of a chunk behind each other; dense: the chunks of a tile, which read the same weights
    auto tile_of = [&](int unit) { return a.expert_offsets ? unit % a.tiles : unit / a.chunks; };
    auto chunk_of = [&](int unit) {
        Chunk c{0, 0, 0};
        if (a.expert_offsets) {
            find_chunk(a.expert_offsets, a.n_experts, a.M, TN, unit / a.tiles, nullptr, c);
        } else {
            c.expert = 0;
            c.tok0 = unit % a.chunks * TN;
            c.ntok = min(TN, a.M - c.tok0);
        }
        return c;
    };

    if (warp == kLoadWarp) {
        int s = 0;
        uint32_t phase = 1, s_phase = 1;         // of `empty`: the first round passes
        int b = 0;
        bool go = true, ok = true;               // of the warp; of the lane that requests the codes, which the others hear of once per kHeld blocks
        if (!a.expert_offsets && !a.early) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("griddepcontrol.launch_dependents;");
        }
        for (int unit = first; go && unit < units; unit += step) {
            const Chunk c = chunk_of(unit);
            const int tile = tile_of(unit), row = static_cast<int>(static_cast<long long>(c.expert) * a.N) + tile * kRows;
            int ahead = 0;
            if (a.early && unit == first) {      // weights are constants: as many as the ring holds while the previous kernel ends
                if (lane == 0) {
                    asm volatile("griddepcontrol.launch_dependents;");
                    for (int i = 0; kb0 + i < kb1 && i < F::kStages; ++i) {
                        mbar_expect_tx(&ctl->full[i], F::kStage);
                        tma_load_2d(ring + i * F::kStage, &maps.w, (kb0 + i) * kBlock, row, &ctl->full[i]);
                    }
                }
                ahead = min(kb1 - kb0, F::kStages);
                asm volatile("griddepcontrol.wait;" ::: "memory");
            }
            const float *const xs = a.xs + static_cast<size_t>(c.tok0) * a.nkb;
            const float *const ws = a.ws + (static_cast<size_t>(c.expert) * a.tiles + tile) * a.nkb;
            for (int kb = kb0; go && kb < kb1; ++kb) {
                if ((kb - kb0) % F::kHeld == 0) {        // scales of the next blocks, on their way as the codes are: a lane a block, two tokens at a time
                    if (!wait_all(&ctl->s_empty[b], s_phase, &ctl->abort, a.status, 0xb05u)) {
                        go = false;
                        break;
                    }
                    const int k = lane % F::kHeld, t0 = lane / F::kHeld;
                    const uint32_t to = smem_u32(scales) + b * F::kScales * 4;
                    if (kb + k < kb1) {
                        for (int t = t0; t < c.ntok; t += 32 / F::kHeld)
                            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + (k * F::kPitch + t) * 4), "l"(xs + static_cast<size_t>(t) * a.nkb + kb + k) : "memory");
                        if (t0 == 0) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + (F::kHeld * F::kPitch + k) * 4), "l"(ws + kb + k) : "memory");
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&ctl->s_full[b])) : "memory");
                    if (lane == 0) {
                        ctl->chunk[b][0] = c.tok0;
                        ctl->chunk[b][1] = c.ntok;
                        ctl->chunk[b][2] = tile;
                        mbar_arrive(&ctl->s_full[b]);
                    }
                    if (b ^= 1; b == 0) s_phase ^= 1;
                }
                const bool requested = kb - kb0 < ahead;
                if (lane == 0 && ok) {
                    ok = requested || wait_soon(&ctl->empty[s], phase, &ctl->abort, a.status, 0xb01u);
                    if (ok) {
                        const uint32_t at = ring + s * F::kStage;
                        if (!requested) {
                            mbar_expect_tx(&ctl->full[s], F::kStage);
                            tma_load_2d(at, &maps.w, kb * kBlock, row, &ctl->full[s]);
                        }
                        tma_load_2d(at + kWBytes, &maps.x, kb * kBlock, c.tok0, &ctl->full[s]);
                        ++ctl->issued;
                    }
                }
                if (++s == F::kStages) s = 0, phase ^= 1;
                if ((kb + 1 - kb0) % F::kHeld == 0 || kb + 1 == kb1) go = __shfl_sync(0xffffffffu, ok, 0);
            }
        }
        for (int i = 0; lane == 0 && go && ok && i < F::kStages; ++i) {      // the MMAs' last arrivals at `empty`: none reaches a CTA that has left
            ok = wait_soon(&ctl->empty[s], phase, &ctl->abort, a.status, 0xb01u);
            if (++s == F::kStages) s = 0, phase ^= 1;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == kMmaWarp) {
        constexpr uint32_t idesc = 1u << 4 | static_cast<uint32_t>(TN >> 3) << 17 | static_cast<uint32_t>(kRows >> 4) << 24;
        int s = 0, d = 0;
        uint32_t phase = 0, d_phase = 1;
        bool go = true;
        // No stage is full before the previous kernels of the stream are complete (x is theirs): what they take does not count against the
        // limit of the waits
        if (!a.expert_offsets) asm volatile("griddepcontrol.wait;" ::: "memory");
        for (int unit = first; go && unit < units; unit += step)
            for (int kb = kb0; go && kb < kb1; kb += F::kTogether) {
                const int here = min(F::kTogether, kb1 - kb);
                go = wait_all(&ctl->d_empty[d], d_phase, &ctl->abort, a.status, 0xb02u);
                for (int g = 0; go && g < here; ++g) {
                    if (!wait_all(&ctl->full[s], phase, &ctl->abort, a.status, 0xb03u)) {
                        go = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t wd = make_desc_sw128(ring + s * F::kStage), xd = make_desc_sw128(ring + s * F::kStage + kWBytes);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) mma_f8(tmem + (d * F::kTogether + g) * TN, wd + 2 * k, xd + 2 * k, idesc, k > 0);
                        umma_commit(&ctl->empty[s]);
                        if (g == here - 1) umma_commit(&ctl->d_full[d]);
                    }
                    __syncwarp();
                    if (++s == F::kStages) s = 0, phase ^= 1;
                }
                if (d ^= 1; d == 0) d_phase ^= 1;
            }
    } else {
        if (!a.expert_offsets) asm volatile("griddepcontrol.wait;" ::: "memory");
        if constexpr (SLICED) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        const uint32_t lanes = tmem + (static_cast<uint32_t>(warp) << 21);              // lane 32 * warp in bits 16 and up
        const int r = threadIdx.x;
        int d = 0, b = 0;
        uint32_t phase = 0, s_phase = 0;
        for (int unit = first; unit < units; unit += step) {
            Chunk c{0, 0, 0};                    // with the scales, from the producer (found by every warp again: 128 experts of 2048 x 768, 4096 rows, 55.5 us for 48.4)
            int tile = 0;
            uint64_t acc[TN / 2] = {};
            for (int kb = kb0; kb < kb1; kb += F::kTogether) {
                const int at = (kb - kb0) % F::kHeld, here = min(F::kTogether, kb1 - kb);
                const float *const held = scales + b * F::kScales;
                if (at == 0) wait_soon(&ctl->s_full[b], s_phase, &ctl->abort, a.status, 0xb06u);
                wait_soon(&ctl->d_full[d], phase, &ctl->abort, a.status, 0xb04u);
                __syncwarp();
                tc_fence_after();
#pragma unroll
                for (int q = 0; q < F::kTogether * TN; q += F::kLoads * F::kStep) {     // 64 columns at a time: of four blocks, of two, or of one
                    uint32_t v[F::kLoads][F::kStep];
#pragma unroll
                    for (int l = 0; l < F::kLoads; ++l) tmem_ld<F::kStep>(lanes + d * F::kTogether * TN + q + l * F::kStep, v[l]);
#pragma unroll
                    for (int l = 0; l < F::kLoads; ++l) tmem_wait_ld(v[l]);
                    if (q + F::kLoads * F::kStep == F::kTogether * TN) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&ctl->d_empty[d]);
                    }
#pragma unroll
                    for (int l = 0; l < F::kLoads; ++l) {
                        const int g = (q + l * F::kStep) / TN, col = (q + l * F::kStep) % TN;
                        if (g >= here) break;
                        const float *const f = held + (at + g) * F::kPitch + col;
                        const float ws = held[F::kHeld * F::kPitch + at + g];
#pragma unroll
                        for (int i = 0; i < F::kStep; i += 4) {
                            const float4 w = *reinterpret_cast<const float4 *>(f + i);
                            fma2(acc[(col + i) / 2], v[l][i], v[l][i + 1], w.x * ws, w.y * ws);
                            fma2(acc[(col + i) / 2 + 1], v[l][i + 2], v[l][i + 3], w.z * ws, w.w * ws);
                        }
                    }
                }
                if (d ^= 1; d == 0) phase ^= 1;
                if (at + F::kTogether == F::kHeld || kb + F::kTogether >= kb1) {
                    c.tok0 = ctl->chunk[b][0];
                    c.ntok = ctl->chunk[b][1];
                    tile = ctl->chunk[b][2];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl->s_empty[b]);
                    if (b ^= 1; b == 0) s_phase ^= 1;
                }
            }
            const int n = tile * kRows + r;
            if constexpr (!SLICED) {
                if (n < a.N && !ctl->abort) {
#pragma unroll
                    for (int t = 0; t < TN; t += 2) {
                        const float2 v = halves(acc[t / 2]);
                        if (t < c.ntok) st_from_f32(a.out, static_cast<size_t>(c.tok0 + t) * a.N + n, v.x, a.out_dt);
                        if (t + 1 < c.ntok) st_from_f32(a.out, static_cast<size_t>(c.tok0 + t + 1) * a.N + n, v.y, a.out_dt);
                    }
                }
            } else {                             // one unit a cluster
                const uint32_t join = ring - F::kRing + F::kJoin;
                int owner = 0, at = rank;        // of token t: t % slices, t / slices * slices + rank
#pragma unroll
                for (int t = 0; t < TN; ++t) {
                    const float2 v = halves(acc[t / 2]);
                    if (t < c.ntok) {
                        if constexpr (F::kPush) st_cluster(join + (at * kRows + r) * 4, owner, t & 1 ? v.y : v.x);
                        else st_shared(ring + (t * kRows + r) * 4, t & 1 ? v.y : v.x);
                    }
                    if (++owner == a.slices) owner = 0, at += a.slices;
                }
            }
        }
    }
    if constexpr (SLICED) {
        __syncwarp();
        if (warp >= kLoadWarp) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        cluster_sync();
    } else {
        __syncthreads();
    }
    if (ctl->abort) rest(ctl, F::kStages);
    if constexpr (SLICED) {
        if (first < units && warp < kLoadWarp && !ctl->abort) {      // the tokens of this rank
            const Chunk c = chunk_of(first);
            const int r = threadIdx.x, n = tile_of(first) * kRows + r;
            const uint32_t join = ring - F::kRing + F::kJoin;
            for (int t0 = rank, at = 0; t0 < c.ntok && n < a.N; t0 += 4 * a.slices, at += 4 * a.slices) {
                float part[4][kMaxSlices];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int q = 0; q < kMaxSlices; ++q) {
                        const int t = t0 + i * a.slices;
                        if (q >= a.slices || t >= c.ntok) part[i][q] = 0.0f;
                        else if constexpr (F::kPush) part[i][q] = ld_shared(join + ((at + i * a.slices + q) * kRows + r) * 4);
                        else part[i][q] = ld_cluster(ring + (t * kRows + r) * 4, q);
                    }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = t0 + i * a.slices;
                    float sum = part[i][0];
#pragma unroll
                    for (int q = 1; q < kMaxSlices; ++q)
                        if (q < a.slices) sum += part[i][q];
                    if (t < c.ntok) st_from_f32(a.out, static_cast<size_t>(c.tok0 + t) * a.N + n, sum, a.out_dt);
                }
            }
        }
        if constexpr (!F::kPush) {
            __syncwarp();
            cluster_sync();                      // no CTA leaves while its sums are read
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(F::kCols));
}

template <int TN, bool SLICED>
cudaError_t launch_as(Ctx *ctx, cudaStream_t st, const uint8_t *x, const uint8_t *w, TArgs a, int K, std::string *why) {
    TMaps maps;
    cudaError_t e = make_map_2d(&maps.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, static_cast<long long>(a.n_experts) * a.N, K, kRows, kBlock, why);
    if (e == cudaSuccess) e = make_map_2d(&maps.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, a.M, K, TN, kBlock, why);
    if (e != cudaSuccess) return e;
    static PerDeviceAttr attr;
    if ((e = attr.set(fp8_tile_kernel<TN, SLICED>, kSmemBytes)) != cudaSuccess) return e;
    const long long units = static_cast<long long>(a.chunks) * a.tiles;
    if (units > kMostSize) return cudaErrorInvalidConfiguration;
    // slices: a cluster a unit; else no more CTAs than run at once, each with units in turn
    const long long ctas = a.slices > 1 ? units * a.slices : std::min<long long>(units, static_cast<long long>(kPerSM) * ctx->sm_count);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.stream = st;
    cudaLaunchAttribute la[2];
    la[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    la[0].val.programmaticStreamSerializationAllowed = 1;
    la[1].id = cudaLaunchAttributeClusterDimension;
    la[1].val.clusterDim.x = static_cast<unsigned>(a.slices);
    la[1].val.clusterDim.y = la[1].val.clusterDim.z = 1;
    cfg.attrs = la;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, fp8_tile_kernel<TN, SLICED>, maps, a);
}
template <int TN>
cudaError_t launch(Ctx *ctx, cudaStream_t st, const uint8_t *x, const uint8_t *w, const TArgs &a, int K, std::string *why) {
    return a.slices > 1 ? launch_as<TN, true>(ctx, st, x, w, a, K, why) : launch_as<TN, false>(ctx, st, x, w, a, K, why);
}

}  // namespace

// K slices: as many as fill the SMs' places once, at least four blocks each
static int slices_for(int sms, long long units, int nkb) {
    int s = 1;
    while (s < kMaxSlices && units * (s + 1) <= static_cast<long long>(kPerSM) * sms && nkb / (s + 1) >= 4) ++s;
    return s;
}

// (a copy of codes starts at rows of 16-byte pieces; rows of all experts are one coordinate)
bool fp8_tile_supported(int M, int N, int K, int n_experts, const void *x, const void *w) {
    return M > 0 && N > 0 && K % 16 == 0 && static_cast<long long>(n_experts) * N <= kMostSize && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
           reinterpret_cast<uintptr_t>(w) % 16 == 0;
}

cudaError_t launch_fp8_tile(Ctx *ctx, cudaStream_t st, const uint8_t *x, const float *xs, const uint8_t *w, const float *ws, const uint32_t *expert_offsets, void *out,
                            int M, int N, int K, int n_experts, int out_dt, std::string *why) {
    TArgs a{};
    a.xs = xs;
    a.ws = ws;
    a.expert_offsets = expert_offsets;
    a.out = out;
    a.status = ctx->d_status;
    a.M = M;
    a.N = N;
    a.nkb = blocks(K);
    a.n_experts = n_experts;
    a.tiles = blocks(N);
    a.out_dt = out_dt;
    // Tokens of a tile.  Dense: what holds them, but 64 as two of 32, whose epilogues share the work (64 x 4096 x 4096 10.0 us, in one of
    // 64 11.1).  Grouped: 16 below eight rows an expert on average (128 experts of 768 x 2048: 4 rows 26.0 us, with 32 29.6; 8 rows 32.9
    // and 31.6; 32 rows 47.0, with 64 50.4).  128 were slower than both this and pairs.
    const int rows = expert_offsets ? (M >= 8 * n_experts ? 32 : 16) : M;
    const int TN = rows <= 16 ? 16 : rows <= 64 ? 32 : 64;
    const long long chunks = expert_offsets ? static_cast<long long>(std::min(M, n_experts)) + M / TN : (M + TN - 1) / TN;
    if (chunks > kMostSize) return cudaErrorInvalidConfiguration;
    a.chunks = static_cast<int>(chunks);
    // An expert's tiles never make slices: what a cluster costs is more than it gives (32 experts of 1536 x 2048, 8 rows: 9.5 us, in slices 16.0)
    a.slices = expert_offsets ? 1 : slices_for(ctx->sm_count, static_cast<long long>(a.chunks) * a.tiles, a.nkb);
    a.early = expert_offsets ? 0 : early_weights(ctx, st);
    switch (TN) {
        case 16: return launch<16>(ctx, st, x, w, a, K, why);
        case 32: return launch<32>(ctx, st, x, w, a, K, why);
        default: return launch<64>(ctx, st, x, w, a, K, why);
    }
}

}  // namespace mtc
