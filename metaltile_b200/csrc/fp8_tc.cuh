// What the tcgen05 kernels of the 8-bit float products share.
#pragma once

#include "fp8.cuh"
#include "tcgen05.cuh"

namespace mtc {
namespace fp8 {

// A wait that mostly finds its phase complete: one try, and only then the polling loop, whose entry alone costs a warp some 200 cycles (one
// block of 256 x 256 x 128 products took 1140 cycles with the loop at every hand-off, 610 so).
__device__ __forceinline__ bool wait_soon(uint64_t *bar, uint32_t parity, volatile uint32_t *abort, uint32_t *status, uint32_t code) {
    return mbar_try(bar, parity) || mbar_wait(bar, parity, abort, status, code);
}

// The same by a whole warp whose loop has to stay uniform (the operands of an MMA then come straight from uniform registers: with one
// thread in the loop four MMAs and their commits took 250 cycles to issue).
__device__ __forceinline__ bool wait_all(uint64_t *bar, uint32_t parity, volatile uint32_t *abort, uint32_t *status, uint32_t code) {
    return __all_sync(0xffffffffu, mbar_try(bar, parity)) || __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, status, code));
}

// The values of a load of tensor memory are there: they pass through, so that nothing that uses them moves in front.
__device__ __forceinline__ void tmem_wait_ld16(uint32_t *v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]),
                   "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 : : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[N]) {
    static_assert(N == 16 || N == 32, "columns of one load");
    tmem_wait_ld16(v);
    if constexpr (N == 32)
        asm volatile("" : "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]),
                     "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]));
}

// acc += d * f, both halves of a pair
__device__ __forceinline__ void fma2(uint64_t &acc, uint32_t d0, uint32_t d1, float f0, float f1) {
    uint64_t d, f;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(d0), "r"(d1));
    asm("mov.b64 %0, {%1, %2};" : "=l"(f) : "f"(f0), "f"(f1));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(d), "l"(f));
}
__device__ __forceinline__ float2 halves(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ float ld_shared(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

}  // namespace fp8
}  // namespace mtc
