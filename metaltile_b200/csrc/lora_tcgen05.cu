// Low-rank adapters on tcgen05, for tiles of up to 128 rows of one adapter: h = x A^T and out = base + scale h B^T (or, back, u = dy B, dx = base + scale u A).
//
// A cluster of eight CTAs has one tile.  Each CTA sums up its eighth of the long axis of the first product into tensor memory (128 rows x rank), the parts meet
// over distributed shared memory, a CTA adds up sixteen rows and hands them to all others as an operand, and each CTA multiplies them with its eighth of
// the columns of the second product.  x, base and out pass once, an adapter once a tile of 128 rows (the warp-level kernel: of 32).  Everything comes
// in by cp.async, many copies ahead, since rows are gathered; results and base go through shared memory so that rows are whole lines.  The tensor core does
// next to nothing, but neither does a warp for its sums: with warp-level MMAs at rank 64 the two pieces of h alone were half of the second product's time.
//
// Measured: 2048 x 4096 x 4096, rank 64, bf16 28.6 us (the warp-level kernel 32.8; the bytes need 8.5), 4096 rows, rank 16 27.4 forward (30.5; the bytes need 15.7: 3.8 TB/s).
// What bounds it is the chain of a tile, of which an SM holds two: of 42,000 cycles at rank 64 the start takes 3,800, the first product 9,500, the sums' way 7,800 and the second product 14,400;
// 16 clusters of eight at 2048 rows, where 15 fit at one CTA an SM, so the one that shares its SMs ends last.  Tried and not better: 512 copying threads (35 us), two warps
// for the weights (27.1), x asked into L2 from the start (the start grows by what the product gains), base likewise (28.3).
//
// h is held in two pieces of T: 17 bits of bf16, 16 and more of f16, which is divided by a power of two of its row (lora_mma.cuh).  Three would not fit beside the ring at rank 64.
//
// The parts meet without a barrier: a CTA stores its sums into the shared memory of the rows' owners as they leave tensor memory (st.async), an owner copies its rows of h
// into all others' (cp.async.bulk), and the receiving side's mbarriers count the bytes.
//
//   warps 0-7  first product's copies; then base in and results out, 64 columns a step: warps 0-3 have the even steps, 4-7 the odd ones, each 32 rows of whole lines
//   warp 8     MMAs, tensor memory        warp 9     the second product's weights
//   shared memory: the first product's ring of stages (128 rows x 64 values of x 16 KB, 64 of the weights of every rank 8 KB; rows 128 bytes apart with the 128-byte
//   swizzle) and what comes in of the sums; then, in their places, h (32 KB), two buffers of weights (8 KB) and four of base and results (16 KB)
#include <algorithm>
#include <cstddef>

#include "lora_mma.cuh"
#include "tcgen05.cuh"

namespace mtc {
namespace {

using namespace lora;

constexpr int kCopy = 256, kMmaWarp = 8, kLoadWarp = 9, kThreads = kCopy + 64, kCluster = 8, kRows = 128, kOwn = kRows / kCluster;
constexpr int kStage = 24 * 1024, kWeights = 16 * 1024;                              // of a stage: where the weights start
constexpr int kHeld = 0, kPiece = 16 * 1024, kColumns = 64;
constexpr int kSmem = 1024 + 112 * 1024;
constexpr uint32_t kTmem = 256, kSums = 0;           // columns of tensor memory: the first product's sums, later four steps of the second one (so that weights wait for no result)

// Ranks 64: the sums of eight CTAs for sixteen rows are 32 KB, a stage less.  Base of the first steps comes in before the sums do: only the last buffer takes their place.
template <int RB>
struct Room {
    static constexpr int kStages = RB == 64 ? 3 : 4, kFrom = kStages * kStage;       // where the others' sums come in
    static __device__ __forceinline__ int weights(int b) { return b == 0 ? 32 * 1024 : RB == 64 ? 104 * 1024 : 40 * 1024; }
    static __device__ __forceinline__ int base(int b) { return RB == 64 ? (b < 2 ? 40 + 16 * b : 72 + 16 * (b - 2)) * 1024 : (48 + 16 * b) * 1024; }
    static constexpr int kEarly = RB == 64 ? 2 : 3;                                  // buffers of base that are free before the sums are added up
};
static_assert(Room<64>::kFrom == 72 * 1024 && Room<32>::kFrom == 96 * 1024, "sums of eight CTAs behind the ring");

struct Ctrl {
    int row_of[kRows];
    uint8_t unit[kRows];                         // f16: exponent of what a row of h was divided by
    uint64_t full[4], empty[4], columns[2], out[4], free[4], done, sums, held;
    uint32_t tmem, abort;
};
static_assert(sizeof(Ctrl) <= 1024, "control block");

// 16 bytes, zeros where there is nothing to be read
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void to_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// row r, 16-byte unit u of a tile of rows of 128 bytes
__device__ __forceinline__ uint32_t tile_at(uint32_t tile, int r, int u) { return tile + r * 128 + ((u ^ (r & 7)) << 4); }

// rows of the operand are 64 values of k; or, where k runs along the rows (`across`), of 8 k's a group of 1024 bytes
__device__ __forceinline__ uint64_t desc_of(uint32_t tile) { return make_desc_sw128(tile); }
constexpr uint32_t idesc_of(int dt, int n, bool across) {
    const uint32_t type = dt == MTC_BF16 ? 1u : 0u;
    return 1u << 4 | type << 7 | type << 10 | (across ? 1u << 16 : 0u) | static_cast<uint32_t>(n / 8) << 17 | static_cast<uint32_t>(kRows / 16) << 24;
}
__device__ __forceinline__ void umma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ uint32_t on_cta(uint32_t at, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
    return r;
}
// sixteen bytes into another CTA's shared memory, counted by a barrier there
__device__ __forceinline__ void send16(uint32_t at, const uint32_t *v, uint32_t bar) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
                 ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(bar) : "memory");
}
__device__ __forceinline__ void send_bulk(uint32_t at, uint32_t from, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(at), "r"(from), "r"(bytes), "r"(bar) : "memory");
}

// into L2, 16-byte aligned
__device__ __forceinline__ void prefetch(const void *p, int bytes) { asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory"); }

// Units of a row of sums are moved about so that neighbouring rows do not meet in a bank
template <int RB>
__device__ __forceinline__ int sums_swizzle(int r) { return RB == 16 ? r >> 1 & 3 : r & 7; }

// RB: 16, 32 or 64 ranks (zeros behind the rank).  BACK as in the warp-level kernel.
template <int DT, int RB, bool BACK>
__global__ void __launch_bounds__(kThreads, 2) lora_tile_kernel(const LoraArgs a, bool keep, bool none) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    using At = Room<RB>;
    constexpr int UNITS = RB / 8, SUMS = RB / 4, kStages = At::kStages;              // 16-byte units of a row of ranks, of a row of sums
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Ctrl *const ctl = reinterpret_cast<Ctrl *>(smem_raw);
    uint8_t *const data = smem_raw + 1024;
    const uint32_t sm = __shfl_sync(0xffffffffu, smem_u32(data), 0);
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), cr = cluster_rank();
    if (blockIdx.x == 0)
        for (int e = tid; e < a.n_adapters; e += kThreads)
            if (a.offsets[e] > a.offsets[e + 1] || a.offsets[e + 1] > static_cast<uint32_t>(a.n_rows)) atomicCAS(a.status, 0u, 0x901u);
    const Tile tile = find_tile(a, blockIdx.x / kCluster, kRows, none);
    if (tile.e < 0) return;                                  // the whole cluster
    const int chunks = (a.c_in + 63) / 64;
    const int chunk0 = static_cast<int>(static_cast<long long>(chunks) * cr / kCluster), mine = static_cast<int>(static_cast<long long>(chunks) * (cr + 1) / kCluster) - chunk0;
    if (tid < kRows) {
        int row = -1;
        if (tid < static_cast<int>(tile.n)) {
            const uint32_t v = a.order[tile.p0 + tid];
            if (v < static_cast<uint32_t>(a.n_rows)) row = static_cast<int>(v);
            else atomicCAS(a.status, 0u, 0x908u);
        }
        ctl->row_of[tid] = row;
    }
    const int units = (a.c_out + kColumns - 1) / kColumns;
    const int step0 = static_cast<int>(static_cast<long long>(units) * cr / kCluster), steps = static_cast<int>(static_cast<long long>(units) * (cr + 1) / kCluster) - step0;
    const int c_end = std::min((step0 + steps) * kColumns, a.c_out);
    if (tile.e >= a.n_adapters) {
        __syncthreads();
        copy_rows<DT, kThreads>(a, ctl->row_of, static_cast<int>(tile.n), step0 * kColumns, c_end, keep, cr, kCluster);
        return;
    }
    // Tensor memory before the next kernel may start, which may want some too and then wait for this one; and not before the previous one is done.
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem)), "r"(kTmem));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(&ctl->full[i], kCopy), mbar_init(&ctl->empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&ctl->columns[i], 32);
        for (int i = 0; i < 4; ++i) mbar_init(&ctl->out[i], 1), mbar_init(&ctl->free[i], kCopy / 2);
        mbar_init(&ctl->done, 1), mbar_init(&ctl->sums, 1), mbar_init(&ctl->held, 1);
        ctl->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        mbar_expect_tx(&ctl->sums, kCluster * kOwn * RB * 4);
        mbar_expect_tx(&ctl->held, (kCluster - 1) * (2 * kOwn * 128 + (DT == MTC_F16 ? kOwn : 0)));
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    cluster_arrive();                                        // the barriers are there: waited for before anything is sent
    asm volatile("griddepcontrol.launch_dependents;");
    const uint32_t tmem = __shfl_sync(0xffffffffu, ctl->tmem, 0);
    if (warp == kMmaWarp) {
        // ---- products; the operands' addresses are the same for the whole warp
        for (int c = 0; c < mine; ++c) {
            const int s = c % kStages;
            mbar_wait_warp(&ctl->full[s], (c / kStages) & 1, &ctl->abort, a.status, 0xb21u);
            tc_fence_after();
            const uint64_t x = desc_of(sm + s * kStage), w = desc_of(sm + s * kStage + kWeights);
            if (elect_one()) {
#pragma unroll
                for (int q = 0; q < 4; ++q) umma_f16_ss(tmem + kSums, x + 2 * q, w + (BACK ? 128 : 2) * q, idesc_of(DT, RB, BACK), c || q ? 1u : 0u);
                umma_commit(&ctl->empty[s]);
                if (c + 1 == mine) umma_commit(&ctl->done);
            }
            __syncwarp();
        }
        cluster_wait();
        __syncthreads();                         // the ring is free
        __syncthreads();                         // this CTA's rows of h are there: they go to the others
        if (lane < kCluster && lane != cr) {
            const uint32_t bar = on_cta(smem_u32(&ctl->held), lane), at = sm + kHeld + cr * kOwn * 128;
#pragma unroll
            for (int p = 0; p < 2; ++p) send_bulk(on_cta(at + p * kPiece, lane), at + p * kPiece, kOwn * 128, bar);
            if (DT == MTC_F16) send_bulk(on_cta(smem_u32(&ctl->unit[cr * kOwn]), lane), smem_u32(&ctl->unit[cr * kOwn]), kOwn, bar);
        }
        __syncwarp();
        mbar_wait_warp(&ctl->held, 0, &ctl->abort, a.status, 0xb22u);
        cluster_arrive();                        // nobody leaves while it sends: waited for at the end
        for (int j = 0; j < steps; ++j) {
            mbar_wait_warp(&ctl->columns[j & 1], (j >> 1) & 1, &ctl->abort, a.status, 0xb23u);
            if (j >= 4) mbar_wait_warp(&ctl->free[j & 3], (j / 4 - 1) & 1, &ctl->abort, a.status, 0xb24u);
            tc_fence_after();
            const uint64_t w = desc_of(sm + At::weights(j & 1)), h = desc_of(sm + kHeld);
            if (elect_one()) {
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int q = 0; q < RB / 16; ++q)
                        umma_f16_ss(tmem + (j & 3) * kColumns, h + (p * kPiece >> 4) + 2 * q, w + (BACK ? 128 : 2) * q, idesc_of(DT, kColumns, BACK), p || q ? 1u : 0u);
                umma_commit(&ctl->out[j & 3]);
            }
            __syncwarp();
        }
    } else if (warp == kLoadWarp) {
        // ---- the second product's weights: 64 columns of every rank
        const uint16_t *const up = static_cast<const uint16_t *>(a.up) + static_cast<size_t>(tile.e) * a.rank * a.c_out;
        // into L2 while the first product runs: steps are read two ahead, which is less than the way to memory takes
        if (steps > 0) {
            const int c0 = step0 * kColumns;
            if constexpr (BACK) {
                for (int r = lane; r < a.rank; r += 32) prefetch(up + static_cast<size_t>(r) * a.c_out + c0, (c_end - c0) * 2);
            } else {
                const int bytes = (c_end - c0) * a.rank * 2;
                for (int i = lane * 4096; i < bytes; i += 32 * 4096) prefetch(up + static_cast<size_t>(c0) * a.rank + i / 2, std::min(4096, bytes - i));
            }
        }
        cluster_wait();
        __syncthreads();                         // the ring is free
        // a lane's unit stays, its rows (columns; BACK: ranks) are ROWS apart
        constexpr int WIDE = BACK ? 8 : UNITS, ROWS = 32 / WIDE, TURNS = (BACK ? RB : kColumns) / ROWS;
        const int r0 = lane / WIDE, u = lane % WIDE;
        auto request = [&](int step) {
            if (step < steps) {
                const int c0 = (step0 + step) * kColumns, last = BACK ? a.rank : a.c_out - c0;       // rows that exist
                const bool unit = BACK ? c0 + u * 8 < a.c_out : u * 8 < a.rank;
                const uint32_t at = sm + At::weights(step & 1) + r0 * 128;
                const uint16_t *const from = BACK ? up + static_cast<size_t>(r0) * a.c_out + c0 + u * 8 : up + static_cast<size_t>(c0 + r0) * a.rank + u * 8;
                const size_t apart = static_cast<size_t>(ROWS) * (BACK ? a.c_out : a.rank);
#pragma unroll
                for (int i = 0; i < TURNS; ++i) {
                    const bool ok = unit && r0 + i * ROWS < last;
                    copy16(at + i * ROWS * 128 + ((u ^ ((r0 + i * ROWS) & 7)) << 4), ok ? from + i * apart : up, ok);
                }
            }
            copy_commit();
        };
        request(0);
        request(1);
        __syncthreads();
        cluster_arrive();
        for (int j = 0; j < steps; ++j) {
            copy_wait<1>();
            to_async_proxy();
            mbar_arrive(&ctl->columns[j & 1]);
            mbar_wait_warp(&ctl->out[j & 3], (j >> 2) & 1, &ctl->abort, a.status, 0xb2au);       // step j is multiplied: its place is free
            request(j + 2);
        }
        copy_wait<0>();
    } else {
        const size_t expert = tile.e;
        const uint16_t *const in = static_cast<const uint16_t *>(a.in), *const base = static_cast<const uint16_t *>(a.base);
        const uint16_t *const down = static_cast<const uint16_t *>(a.down) + expert * a.rank * a.c_in;
        const int u8 = tid & 7, r32 = tid >> 3;              // the 16-byte unit and the first row (of every 32) that this thread copies

        // ---- the first product's operands
        constexpr int LAG = kStages - 1;
        {
            const uint16_t *from[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = ctl->row_of[r32 + 32 * q];
                from[q] = row >= 0 ? in + static_cast<size_t>(row) * a.c_in : nullptr;
            }
            for (int i = 0; i < mine + LAG; ++i) {
                if (i < mine) {
                    const int s = i % kStages;
                    if (i >= kStages) mbar_wait_warp(&ctl->empty[s], (i / kStages - 1) & 1, &ctl->abort, a.status, 0xb25u);
                    const uint32_t at = sm + s * kStage;
                    const int k = (chunk0 + i) * 64 + u8 * 8;
                    const bool there = k < a.c_in;
#pragma unroll
                    for (int q = 0; q < 4; ++q) copy16(tile_at(at, r32 + 32 * q, u8), there && from[q] ? from[q] + k : in, there && from[q]);
                    if constexpr (!BACK) {       // rows are ranks
#pragma unroll
                        for (int q = 0; q < (RB + 31) / 32; ++q) {
                            const int r = r32 + 32 * q;
                            const bool ok = there && r < a.rank;
                            if (RB >= 32 || r < RB) copy16(tile_at(at + kWeights, r, u8), ok ? down + static_cast<size_t>(r) * a.c_in + k : down, ok);
                        }
                    } else {                     // rows are k's
#pragma unroll
                        for (int q0 = 0; q0 < 64 * UNITS; q0 += kCopy) {
                            const int q = q0 + tid, r = q / UNITS, u = q % UNITS, kk = (chunk0 + i) * 64 + r;
                            const bool ok = kk < a.c_in && u * 8 < a.rank;
                            if (64 * UNITS >= kCopy || q < 64 * UNITS) copy16(tile_at(at + kWeights, r, u), ok ? down + static_cast<size_t>(kk) * a.rank + u * 8 : down, ok);
                        }
                    }
                }
                copy_commit();
                if (i >= LAG) {
                    copy_wait<LAG>();
                    to_async_proxy();
                    mbar_arrive(&ctl->full[(i - LAG) % kStages]);
                }
            }
        }
        if (mine) mbar_wait_warp(&ctl->done, 0, &ctl->abort, a.status, 0xb26u);
        tc_fence_after();

        // ---- the parts of the sums go to the rows' owners
        const int row = (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;                // of tensor memory: the warp's quarter
        cluster_wait();
        if (RB > 16 || warp < 4) {
            constexpr int COLS = RB == 16 ? 16 : RB / 2;
            const int first = RB == 16 ? 0 : (warp >> 2) * COLS;
            uint32_t v[COLS];
#pragma unroll
            for (int i = 0; i < COLS; ++i) v[i] = 0;
            if (mine) {
                tmem_ld<COLS>(tmem + kSums + first + lanes, v);
                tmem_wait_ld();
            }
            const uint32_t to = on_cta(sm + At::kFrom + (cr * kOwn + row % kOwn) * RB * 4, row / kOwn), bar = on_cta(smem_u32(&ctl->sums), row / kOwn);
#pragma unroll
            for (int i = 0; i < COLS / 4; ++i) send16(to + (((first / 4 + i) ^ sums_swizzle<RB>(row)) << 4), v + 4 * i, bar);
        }
        tc_fence_before();
        __syncthreads();                         // (the ring is free: everybody has seen `done`)

        // ---- base of this warp's rows, every second step
        const int group = warp >> 2, r8 = (warp & 3) * 32 + (lane >> 3);             // parity of the steps; this lane's row of every four
        long long at_row[8];                     // offsets of these rows in base and out, -1: none
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int to = ctl->row_of[r8 + 4 * i];
            at_row[i] = to < 0 ? -1 : static_cast<long long>(to) * a.c_out + u8 * 8;
        }
        auto request = [&](int step) {
            const int c0 = (step0 + step) * kColumns;
            if (a.base && step < steps && c0 + u8 * 8 < a.c_out) {
                const uint32_t to = sm + At::base(step & 3);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (at_row[i] >= 0) copy16(tile_at(to, r8 + 4 * i, u8), base + at_row[i] + c0, true);
            }
            copy_commit();
        };
        request(group);
        if (group + 2 < At::kEarly) request(group + 2);
        if (a.base && steps > At::kEarly && tid < static_cast<int>(tile.n) && ctl->row_of[tid] >= 0) {       // and the rest comes into L2 while the sums are on their way
            const int c0 = (step0 + At::kEarly) * kColumns;
            prefetch(base + static_cast<size_t>(ctl->row_of[tid]) * a.c_out + c0, (c_end - c0) * 2);
        }
        const float scale = a.scales ? a.scales[expert] : 1.0f;

        // ---- h: this CTA's sixteen rows, four ranks a thread
        mbar_wait_warp(&ctl->sums, 0, &ctl->abort, a.status, 0xb27u);
        if (tid < kOwn * SUMS) {
            const int r = cr * kOwn + tid / SUMS, u = tid % SUMS;
            float4 v[kCluster], s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int q = 0; q < kCluster; ++q) v[q] = *reinterpret_cast<const float4 *>(data + At::kFrom + (q * kOwn + r % kOwn) * RB * 4 + ((u ^ sums_swizzle<RB>(r)) << 4));
#pragma unroll
            for (int q = 0; q < kCluster; ++q) s.x += v[q].x, s.y += v[q].y, s.z += v[q].z, s.w += v[q].w;
            const int to = ctl->row_of[r];
            if (keep && to >= 0 && u * 4 < a.rank) *reinterpret_cast<float4 *>(a.low + static_cast<size_t>(to) * a.rank + u * 4) = s;
            s = ranks_of(s, u * 4, a.rank);
            float f = 1.0f;
            if constexpr (DT == MTC_F16) {
                float most = most_of(s);
#pragma unroll
                for (int o = SUMS / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o, SUMS));
                f = unit_of(most);
                if (u == 0) ctl->unit[r] = static_cast<uint8_t>(__float_as_uint(f) >> 23);
            }
            uint2 w[2];
            hold_pieces<DT>(s, f, w);
#pragma unroll
            for (int p = 0; p < 2; ++p) *reinterpret_cast<uint2 *>(data + (tile_at(kHeld + p * kPiece, r, u / 2) + (u & 1) * 8)) = w[p];
        }
        to_async_proxy();
        __syncthreads();
        if (DT == MTC_F16) mbar_wait_warp(&ctl->held, 0, &ctl->abort, a.status, 0xb28u);
        cluster_arrive();
        const float factor = DT == MTC_F16 ? scale * __uint_as_float(static_cast<uint32_t>(ctl->unit[row]) << 23) : scale;

        // ---- 64 columns at a time; warps do not wait for each other
        if (group + 2 >= At::kEarly) request(group + 2);
        for (int j = group; j < steps; j += 2) {
            copy_wait<1>();                      // base of this step
            __syncwarp();
            uint8_t *const tile_base = data + At::base(j & 3);
            uint4 *const line = reinterpret_cast<uint4 *>(tile_base + row * 128);
            mbar_wait_warp(&ctl->out[j & 3], (j >> 2) & 1, &ctl->abort, a.status, 0xb29u);
            tc_fence_after();
#pragma unroll
            for (int half = 0; half < 8; half += 4) {
                lora::Eight<DT> b[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint4 q = a.base ? line[(half + i) ^ (row & 7)] : make_uint4(0, 0, 0, 0);
                    b[i].w[0] = q.x, b[i].w[1] = q.y, b[i].w[2] = q.z, b[i].w[3] = q.w;
                }
                uint32_t v[32];
                tmem_ld<32>(tmem + (j & 3) * kColumns + half * 8 + lanes, v);
                tmem_wait_ld();
                if (half) {
                    tc_fence_before();
                    mbar_arrive(&ctl->free[j & 3]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float r[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) r[k] = fmaf(__uint_as_float(v[8 * i + k]), factor, b[i].value(k));
                    lora::Eight<DT>::put(&line[(half + i) ^ (row & 7)], 0, r);
                }
            }
            __syncwarp();
            uint4 q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = *reinterpret_cast<const uint4 *>(tile_base + (r8 + 4 * i) * 128 + ((u8 ^ ((r8 + 4 * i) & 7)) << 4));
            const int c0 = (step0 + j) * kColumns;
            if (c0 + u8 * 8 < a.c_out) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (at_row[i] >= 0) *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + at_row[i] + c0) = q[i];
            }
            __syncwarp();
            request(j + 4);                      // in this step's place
        }
        copy_wait<0>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (ctl->abort && tid == 0) {                // gave up: bounded waits for MMAs that may still be on their way
        drain_ring(ctl->empty, mine, kStages);
        drain_ring(ctl->out, steps, 4);
    }
    __syncthreads();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmem));
    cluster_wait();
}

template <int DT, int RB, bool BACK>
cudaError_t launch(cudaStream_t st, const LoraArgs &a, bool keep, bool none) {
    static PerDeviceAttr attr;
    const cudaError_t e = attr.set(lora_tile_kernel<DT, RB, BACK>, kSmem);
    if (e != cudaSuccess) return e;
    const long long tiles = most_tiles(a, kRows);
    if (tiles * kCluster > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    return launch_cluster(lora_tile_kernel<DT, RB, BACK>, static_cast<unsigned>(tiles * kCluster), kThreads, kCluster, kSmem, st, a, keep, none);
}
template <int DT>
cudaError_t launch(cudaStream_t st, const LoraArgs &a, bool backward, bool keep, bool none) {
    if (a.rank <= 16) return backward ? launch<DT, 16, true>(st, a, keep, none) : launch<DT, 16, false>(st, a, keep, none);
    if (a.rank <= 32) return backward ? launch<DT, 32, true>(st, a, keep, none) : launch<DT, 32, false>(st, a, keep, none);
    return backward ? launch<DT, 64, true>(st, a, keep, none) : launch<DT, 64, false>(st, a, keep, none);
}

}  // namespace

bool lora_tile_supported(const LoraArgs &a, bool keep, int dt) {
    return dt != MTC_F32 && a.rank % 8 == 0 && a.rank <= 64 && (!keep || reinterpret_cast<uintptr_t>(a.low) % 16 == 0);
}
cudaError_t launch_lora_tile(cudaStream_t st, const LoraArgs &a, bool backward, bool keep, bool none, int dt) {
    return dt == MTC_BF16 ? launch<MTC_BF16>(st, a, backward, keep, none) : launch<MTC_F16>(st, a, backward, keep, none);
}

}  // namespace mtc
