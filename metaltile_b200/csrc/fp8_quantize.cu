// Float rows or matrices -> e4m3 codes with an f32 scale for each block of 128 (activations) or 128 x 128 (weights).
// The reference has no 8-bit float format; this stands next to its affine quantizer (crates/metaltile-std/src/mlx/quantized.rs:3629-3667).
//
//   s = max(max |x| / 448, 2^-90) over the finite values of the block (pow2: the least power of two that is not below)
//   code = x / s rounded to the nearest e4m3 value, ties to even; infinities and NaN become NaN
//
// Bound by memory: every value is read once and stays in registers between the maximum and the codes.
#include "fp8.cuh"

namespace mtc {
namespace {

using namespace fp8;

// eight consecutive values of a row; `n` of them exist
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const void *base, size_t at, int n, float (&v)[8]) {
    if constexpr (VEC) {
        if (n <= 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.0f;
            return;
        }
        if constexpr (DT == MTC_F32) {
            const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at);
            const float4 a = p[0], b = p[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 q = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(base) + at);
            const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (DT == MTC_BF16) {
                    v[2 * i] = __uint_as_float(u[i] << 16);
                    v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
                } else {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
                    v[2 * i] = f.x;
                    v[2 * i + 1] = f.y;
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? ld_written_as_f32(base, at + i, DT) : 0.0f;
    }
}

__device__ __forceinline__ float largest(const float (&v)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = fabsf(v[i]);
        m = fmaxf(m, a < INFINITY ? a : 0.0f);      // (a NaN compares false)
    }
    return m;
}

template <bool VEC>
__device__ __forceinline__ void store8(uint8_t *codes, size_t at, int n, const float (&v)[8], float s, float inv) {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = to_e4m3x2(code_quotient(v[2 * i], s, inv), code_quotient(v[2 * i + 1], s, inv));
    if constexpr (VEC) {
        if (n > 0) *reinterpret_cast<uint2 *>(codes + at) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) codes[at + i] = static_cast<uint8_t>(c[i / 2] >> (i & 1) * 8);
    }
}

// Blocks of 1 x 128: sixteen lanes a block, eight values a lane.
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const void *x, const uint32_t *rows, uint8_t *codes, float *scales, long long n_rows,
                                                            long long n_src_rows, int K, int pow2, uint32_t *status) {
    pdl_enter();
    const int kb = blocks(K), lane = threadIdx.x & 15;
    const long long total = n_rows * kb, step = static_cast<long long>(gridDim.x) * (blockDim.x / 16);
    // (both halves of a warp go round equally often: the shuffles below take all lanes)
    const long long first = static_cast<long long>(blockIdx.x) * (blockDim.x / 16) + threadIdx.x / 16, trips = (total - (first & ~1ll) + step - 1) / step;
    for (long long t = 0; t < trips; ++t) {
        const long long i = first + t * step;
        const bool have = i < total;
        const long long r = have ? i / kb : 0;
        const int b = static_cast<int>(have ? i - r * kb : 0), k0 = b * kBlock + lane * 8;
        long long src = r;
        if (rows && have) {
            const uint32_t id = rows[r];
            src = id;
            if (id >= n_src_rows) {
                if (lane == 0 && b == 0) atomicCAS(status, 0u, 0x906u);      // an index outside the tensor reads row 0
                src = 0;
            }
        }
        const int n = have ? K - k0 : 0;
        float v[8];
        load8<DT, VEC>(x, static_cast<size_t>(src) * K + k0, n, v);
        float m = largest(v);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float s = scale_of(m, pow2), inv = __frcp_rn(s);
        if (have && lane == 0) scales[i] = s;
        store8<VEC>(codes, static_cast<size_t>(r) * K + k0, n, v, s, inv);
    }
}

// Blocks of 128 x 128: a CTA a block; a warp two rows of 128 at a time, eight times.
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const void *x, uint8_t *codes, float *scales, long long n_rows, int K, int pow2) {
    pdl_enter();
    const int kb = blocks(K);
    const long long nb = (n_rows + kBlock - 1) / kBlock;
    const long long id = blockIdx.x;                          // (matrix, block of rows, block of columns)
    const int b = static_cast<int>(id % kb);
    const long long rb = id / kb % nb, mat = id / kb / nb;
    const int lane = threadIdx.x & 15, row = threadIdx.x / 16, k0 = b * kBlock + lane * 8;
    float v[8][8];
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long r = rb * kBlock + i * 16 + row;
        load8<DT, VEC>(x, static_cast<size_t>(mat * n_rows + r) * K + k0, r < n_rows ? K - k0 : 0, v[i]);
        m = fmaxf(m, largest(v[i]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    __shared__ float most[8];
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, most[i]);
    const float s = scale_of(m, pow2), inv = __frcp_rn(s);
    if (threadIdx.x == 0) scales[id] = s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long r = rb * kBlock + i * 16 + row;
        store8<VEC>(codes, static_cast<size_t>(mat * n_rows + r) * K + k0, r < n_rows ? K - k0 : 0, v[i], s, inv);
    }
}

template <int DT, bool VEC>
cudaError_t launch(Ctx *ctx, cudaStream_t st, const void *x, const uint32_t *rows, uint8_t *codes, float *scales, int n_mats, long long n_rows,
                   long long n_src_rows, int K, int block_rows, int pow2) {
    if (block_rows == 1) {
        const long long ctas = (n_rows * blocks(K) + 15) / 16;
        return launch_pdl(quantize_rows_kernel<DT, VEC>, static_cast<unsigned>(ctas < 1ll << 30 ? ctas : 1ll << 30), 256, 0, st, x, rows, codes, scales,
                          n_rows, n_src_rows, K, pow2, ctx->d_status);
    }
    const long long ctas = n_mats * ((n_rows + kBlock - 1) / kBlock) * blocks(K);
    if (ctas > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    return launch_pdl(quantize_blocks_kernel<DT, VEC>, static_cast<unsigned>(ctas), 256, 0, st, x, codes, scales, n_rows, K, pow2);
}

}  // namespace

cudaError_t launch_fp8_quantize(Ctx *ctx, cudaStream_t st, const void *x, const uint32_t *rows, uint8_t *codes, float *scales, int n_mats,
                                long long n_rows, long long n_src_rows, int K, int block_rows, int pow2, int dt) {
    const bool vec = K % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 8 == 0;
    auto *f = dt == MTC_F32    ? (vec ? launch<MTC_F32, true> : launch<MTC_F32, false>)
              : dt == MTC_BF16 ? (vec ? launch<MTC_BF16, true> : launch<MTC_BF16, false>)
                               : (vec ? launch<MTC_F16, true> : launch<MTC_F16, false>);
    return f(ctx, st, x, rows, codes, scales, n_mats, n_rows, n_src_rows, K, block_rows, pow2);
}

}  // namespace mtc
