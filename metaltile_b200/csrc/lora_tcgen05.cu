// Low-rank adapters on tcgen05, for tiles of up to 128 rows of one adapter: h = x A^T and out = base + scale h B^T (or, back, u = dy B, dx = base + scale u A).
//
// A cluster of eight CTAs has one tile.  Each CTA sums up its eighth of the long axis of the first product into tensor memory (128 rows x rank), the parts meet
// over distributed shared memory, a CTA adds up sixteen rows and hands them to all others as an operand, and each CTA multiplies them with its eighth of
// the columns of the second product.  Bound by memory: x, base and out pass once, an adapter once a tile of 128 rows (the warp-level kernel: of 32).  Everything comes
// in by cp.async, many copies ahead, since rows are gathered; results and base go through shared memory so that rows are whole lines.  The tensor core does
// next to nothing, but neither does a warp for its sums: with warp-level MMAs at rank 64 the two pieces of h alone were half of the second product's time.
//
// h is held in two pieces of T (16 bits and more; f16 divided by the power of two of its row's largest value).
//
//   shared memory, 24 KB units: first product a ring of four stages (128 rows x 64 values of x, 64 of the weights of every rank), rows 128 bytes apart with the
//   128-byte swizzle; then the part of the sums (32 KB), h (32 KB), and three buffers of 64 columns (weights 8 KB, base and results 16 KB), the last one in place of the part
#include <algorithm>
#include <cstddef>

#include "lora_mma.cuh"
#include "tcgen05.cuh"

namespace mtc {
namespace {

using namespace lora;

constexpr int kThreads = 256, kCluster = 8, kRows = 128, kOwn = kRows / kCluster;
constexpr int kStages = 4, kStage = 24 * 1024, kWeights = 16 * 1024;                 // of a stage: where the weights start
constexpr int kPart = 0, kHeld = 32 * 1024, kPiece = 16 * 1024, kColumns = 64, kBase = 8 * 1024;      // of a buffer of columns: where base starts
constexpr int kSmem = 1024 + 112 * 1024;
constexpr uint32_t kTmem = 256, kSums = 0, kOut = 64;                                // columns of tensor memory

struct Ctrl {
    int row_of[kRows];
    uint8_t unit[kRows];                         // f16: exponent of what a row of h was divided by
    uint64_t full[kStages], empty[kStages], out[2], done;
    uint32_t tmem, abort;
};
static_assert(sizeof(Ctrl) <= 1024, "control block");

__device__ __forceinline__ int buffer_at(int step) { return step % 3 == 0 ? 64 * 1024 : step % 3 == 1 ? 88 * 1024 : 0; }

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
__device__ __forceinline__ float4 ld_far(uint32_t at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void st_far(uint32_t at, uint32_t x, uint32_t y) { asm volatile("st.shared::cluster.v2.u32 [%0], {%1,%2};" ::"r"(at), "r"(x), "r"(y) : "memory"); }
__device__ __forceinline__ void st_far(uint32_t at, uint8_t v) { asm volatile("st.shared::cluster.u8 [%0], %1;" ::"r"(at), "r"(static_cast<uint32_t>(v)) : "memory"); }

// RB: 16, 32 or 64 ranks (zeros behind the rank).  BACK as in the warp-level kernel.
template <int DT, int RB, bool BACK>
__global__ void __launch_bounds__(kThreads, 2) lora_tile_kernel(const LoraArgs a, bool keep, bool none) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int UNITS = RB / 8, SUMS = RB / 4;             // 16-byte units of a row of ranks, of a row of sums
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Ctrl *const ctl = reinterpret_cast<Ctrl *>(smem_raw);
    uint8_t *const data = smem_raw + 1024;
    const uint32_t sm = smem_u32(data);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cr = cluster_rank();
    if (blockIdx.x == 0)
        for (int e = tid; e < a.n_adapters; e += kThreads)
            if (a.offsets[e] > a.offsets[e + 1] || a.offsets[e + 1] > static_cast<uint32_t>(a.n_rows)) atomicCAS(a.status, 0u, 0x901u);
    const Tile tile = find_tile(a, blockIdx.x / kCluster, kRows, none);
    if (tile.e < 0) return;                                  // the whole cluster
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
    if (tile.e == a.n_adapters) {
        __syncthreads();
        copy_rows<DT, kThreads>(a, ctl->row_of, static_cast<int>(tile.n), step0 * kColumns, std::min((step0 + steps) * kColumns, a.c_out), keep, cr, kCluster);
        return;
    }
    // Tensor memory before the next kernel may start, which may want some too and then wait for this one; and not before the previous one is done.
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem)), "r"(kTmem));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (tid == 32) {
        for (int i = 0; i < kStages; ++i) mbar_init(&ctl->full[i], kThreads), mbar_init(&ctl->empty[i], 1);
        mbar_init(&ctl->out[0], 1), mbar_init(&ctl->out[1], 1), mbar_init(&ctl->done, 1);
        ctl->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    asm volatile("griddepcontrol.launch_dependents;");
    const uint32_t tmem = ctl->tmem;
    const size_t expert = tile.e;
    const uint16_t *const in = static_cast<const uint16_t *>(a.in), *const base = static_cast<const uint16_t *>(a.base);
    const uint16_t *const down = static_cast<const uint16_t *>(a.down) + expert * a.rank * a.c_in, *const up = static_cast<const uint16_t *>(a.up) + expert * a.rank * a.c_out;
    const int u8 = tid & 7, r32 = tid >> 3;                  // the 16-byte unit and the first row (of every 32) that this thread copies
    int rows[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) rows[i] = ctl->row_of[r32 + 32 * i];

    // ---- the first product
    const int chunks = (a.c_in + 63) / 64;
    const int chunk0 = static_cast<int>(static_cast<long long>(chunks) * cr / kCluster), mine = static_cast<int>(static_cast<long long>(chunks) * (cr + 1) / kCluster) - chunk0;
    constexpr int LAG = kStages - 1;
    for (int i = 0; i < mine + LAG; ++i) {
        if (i < mine) {
            const int s = i % kStages;
            if (i >= kStages) mbar_wait(&ctl->empty[s], (i / kStages - 1) & 1, &ctl->abort, a.status, 0xb21u);
            const uint32_t at = sm + s * kStage;
            const int k = (chunk0 + i) * 64 + u8 * 8;
            const bool there = k < a.c_in;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const bool row = there && rows[q] >= 0;
                copy16(tile_at(at, r32 + 32 * q, u8), row ? in + static_cast<size_t>(rows[q]) * a.c_in + k : in, row);
            }
            if constexpr (!BACK) {               // rows are ranks
#pragma unroll
                for (int q = 0; q < (RB + 31) / 32; ++q) {
                    const int r = r32 + 32 * q;
                    const bool ok = there && r < a.rank;
                    if (RB >= 32 || r < RB) copy16(tile_at(at + kWeights, r, u8), ok ? down + static_cast<size_t>(r) * a.c_in + k : down, ok);
                }
            } else {                             // rows are k's
#pragma unroll
                for (int q = tid; q < 64 * UNITS; q += kThreads) {
                    const int r = q / UNITS, u = q % UNITS, kk = (chunk0 + i) * 64 + r;
                    const bool ok = kk < a.c_in && u * 8 < a.rank;
                    copy16(tile_at(at + kWeights, r, u), ok ? down + static_cast<size_t>(kk) * a.rank + u * 8 : down, ok);
                }
            }
        }
        copy_commit();
        if (i >= LAG) {
            const int c = i - LAG, s = c % kStages;
            copy_wait<LAG>();
            to_async_proxy();
            mbar_arrive(&ctl->full[s]);
            if (warp == 0) {
                mbar_wait_warp(&ctl->full[s], (c / kStages) & 1, &ctl->abort, a.status, 0xb22u);
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t x = desc_of(sm + s * kStage), w = desc_of(sm + s * kStage + kWeights);
#pragma unroll
                    for (int q = 0; q < 4; ++q) umma_f16_ss(tmem + kSums, x + 2 * q, w + (BACK ? 128 : 2) * q, idesc_of(DT, RB, BACK), c || q ? 1u : 0u);
                    umma_commit(&ctl->empty[s]);
                    if (c + 1 == mine) umma_commit(&ctl->done);
                }
                __syncwarp();
            }
        }
    }
    if (mine) mbar_wait(&ctl->done, 0, &ctl->abort, a.status, 0xb23u);
    tc_fence_after();

    // ---- what the second product reads is on its way meanwhile
    auto request = [&](int step) {
        if (step < steps) {
            const uint32_t at = sm + buffer_at(step);
            const int c0 = (step0 + step) * kColumns, c = c0 + u8 * 8;
            if constexpr (!BACK) {               // rows are columns
                for (int q = tid; q < kColumns * UNITS; q += kThreads) {
                    const int r = q / UNITS, u = q % UNITS;
                    const bool ok = c0 + r < a.c_out && u * 8 < a.rank;
                    copy16(tile_at(at, r, u), ok ? up + static_cast<size_t>(c0 + r) * a.rank + u * 8 : up, ok);
                }
            } else {                             // rows are ranks
#pragma unroll
                for (int q = 0; q < (RB + 31) / 32; ++q) {
                    const int r = r32 + 32 * q;
                    const bool ok = r < a.rank && c < a.c_out;
                    if (RB >= 32 || r < RB) copy16(tile_at(at, r, u8), ok ? up + static_cast<size_t>(r) * a.c_out + c : up, ok);
                }
            }
            if (a.base) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const bool ok = c < a.c_out && rows[q] >= 0;
                    copy16(tile_at(at + kBase, r32 + 32 * q, u8), ok ? base + static_cast<size_t>(rows[q]) * a.c_out + c : base, ok);
                }
            }
        }
        copy_commit();
    };
    __syncthreads();                             // (the ring is free: every warp has seen `done`)
    request(0);
    request(1);

    // ---- the parts of the sums, rows of RB values, their units moved about so that neighbouring rows do not meet in a bank
    auto sums_at = [&](int r, int u) { return static_cast<uint32_t>(kPart + r * RB * 4 + ((u ^ (RB == 16 ? r >> 1 & 3 : r & 7)) << 4)); };
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;                    // of tensor memory: the warp's quarter
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
#pragma unroll
        for (int i = 0; i < COLS / 4; ++i)
            *reinterpret_cast<uint4 *>(data + sums_at(row, first / 4 + i)) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }
    tc_fence_before();
    cluster_arrive();
    cluster_wait();
    // this CTA's sixteen rows: four ranks a thread
    if (tid < kOwn * SUMS) {
        const int r = cr * kOwn + tid / SUMS, u = tid % SUMS;
        float4 v[kCluster], s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int q = 0; q < kCluster; ++q) v[q] = ld_far(on_cta(sm + sums_at(r, u), q));
#pragma unroll
        for (int q = 0; q < kCluster; ++q) s.x += v[q].x, s.y += v[q].y, s.z += v[q].z, s.w += v[q].w;
        const int to = ctl->row_of[r];
        if (keep && to >= 0 && u * 4 < a.rank) *reinterpret_cast<float4 *>(a.low + static_cast<size_t>(to) * a.rank + u * 4) = s;
        float f = 1.0f;
        if constexpr (DT == MTC_F16) {
            float most = fmaxf(fmaxf(fabsf(s.x), fabsf(s.y)), fmaxf(fabsf(s.z), fabsf(s.w)));
#pragma unroll
            for (int o = SUMS / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o, SUMS));
            f = unit_of(most);
        }
        uint2 w[2];
        hold_pieces<DT>(s, f, w);
#pragma unroll
        for (int q = 0; q < kCluster; ++q) {
            const uint32_t at = on_cta(sm + kHeld, q);
#pragma unroll
            for (int p = 0; p < 2; ++p) st_far(tile_at(at + p * kPiece, r, u / 2) + (u & 1) * 8, w[p].x, w[p].y);
            if (DT == MTC_F16 && u == 0) st_far(on_cta(smem_u32(&ctl->unit[r]), q), static_cast<uint8_t>(__float_as_uint(f) >> 23));
        }
    }
    asm volatile("fence.proxy.async;" ::: "memory");         // what was written to the others is their operand
    cluster_arrive();
    cluster_wait();
    asm volatile("fence.proxy.async;" ::: "memory");
    request(2);

    // ---- the second product, 64 columns at a time; the product of the next is under way while one goes out
    const float scale = a.scales ? a.scales[expert] : 1.0f;
    const float factor = DT == MTC_F16 ? scale * __uint_as_float(static_cast<uint32_t>(ctl->unit[row]) << 23) : scale;
    auto multiply = [&](int step) {              // by warp 0
        if (elect_one()) {
            const uint64_t w = desc_of(sm + buffer_at(step)), h = desc_of(sm + kHeld);
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int q = 0; q < RB / 16; ++q)
                    umma_f16_ss(tmem + kOut + (step & 1) * kColumns, h + (p * kPiece >> 4) + 2 * q, w + (BACK ? 128 : 2) * q, idesc_of(DT, kColumns, BACK), p || q ? 1u : 0u);
            umma_commit(&ctl->out[step & 1]);
        }
        __syncwarp();
    };
    if (steps > 0) {
        copy_wait<2>();
        to_async_proxy();
        __syncthreads();
        if (warp == 0) {
            tc_fence_after();
            multiply(0);
        }
    }
    for (int j = 0; j < steps; ++j) {
        copy_wait<1>();                          // the columns of step j + 1
        to_async_proxy();
        tc_fence_before();
        __syncthreads();
        if (warp == 0 && j + 1 < steps) {
            tc_fence_after();
            multiply(j + 1);
        }
        mbar_wait(&ctl->out[j & 1], (j >> 1) & 1, &ctl->abort, a.status, 0xb24u);
        tc_fence_after();
        uint32_t v[32];
        tmem_ld<32>(tmem + kOut + (j & 1) * kColumns + (warp >> 2) * 32 + lanes, v);
        tmem_wait_ld();
        uint8_t *const at = data + buffer_at(j) + kBase + row * 128;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint4 *const p = reinterpret_cast<uint4 *>(at + ((((warp >> 2) * 4 + i) ^ (row & 7)) << 4));
            lora::Eight<DT> b;
            const uint4 q = a.base ? *p : make_uint4(0, 0, 0, 0);
            b.w[0] = q.x, b.w[1] = q.y, b.w[2] = q.z, b.w[3] = q.w;
            float r[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) r[k] = fmaf(__uint_as_float(v[8 * i + k]), factor, b.value(k));
            lora::Eight<DT>::put(p, 0, r);
        }
        __syncthreads();
        const int c = (step0 + j) * kColumns + u8 * 8;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (rows[q] >= 0 && c < a.c_out)
                *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + static_cast<size_t>(rows[q]) * a.c_out + c) =
                    *reinterpret_cast<const uint4 *>(data + buffer_at(j) + kBase + (r32 + 32 * q) * 128 + ((u8 ^ (r32 & 7)) << 4));
        __syncthreads();
        request(j + 3);
    }
    copy_wait<0>();
    if (ctl->abort && tid == 0) {                // gave up: bounded waits for MMAs that may still be on their way
        drain_ring(ctl->empty, mine, kStages);
        for (int i = 0; i < 2 && i < steps; ++i) {
            const int last = steps - 1 - ((steps - 1 - i) & 1);                      // the last step of this buffer
            for (uint32_t n = 0; n < 1u << 16 && !mbar_try(&ctl->out[i], (last >> 1) & 1); ++n) {}
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmem));
}

template <int DT, int RB, bool BACK>
cudaError_t launch(cudaStream_t st, const LoraArgs &a, bool keep, bool none) {
    static PerDeviceAttr attr;
    const cudaError_t e = attr.set(lora_tile_kernel<DT, RB, BACK>, kSmem);
    if (e != cudaSuccess) return e;
    const long long tiles = std::min<long long>(a.n_rows, a.n_rows / kRows + a.n_adapters + 1ll);
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
