// What the tensor-core kernels of low-rank adapters share: operands in pieces, fragments, and which rows and columns a lane holds.
//
// Operands.  Warp-level MMAs of 16-bit values with f32 sums.  f32 values are three bf16 pieces, each what is left rounded to 8 bits: 24 bits, exact.  A rest is at most 2^-8 of what was
// rounded, so the products of pieces that are left out (two small ones and the smallest; six of nine remain) are together at most 2^-24 of the whole, on either side of it.  (Pieces that are
// cut off leave rests of twice the size and of one sign: 2^-21.)  bf16 and f16 weights and activations are operands as they are.
//
// What lies between the two products, h or u, is an f32 sum.  Beside f32 weights it is an operand in three pieces, 24 bits.  Beside 16-bit weights it is held in two, which costs two MMAs a
// step of ranks: 17 bits of bf16 (2^-17 of each value; the result, rounded to 8 bits, is off by up to 2^-8), 16 and more of f16 (below).  What is kept for the backward pass is the f32 sum.
//
// Order of k.  A sum may run over k in any order as long as both operands have the same, so a lane takes what lies next to each other in memory: of
// 32 neighbours lane (g, t) = (lane / 4, lane % 4) has 8t .. 8t + 7, the first four of them in the first of two MMAs.  Where the other operand lies across (k along
// its rows), the lane loads eight such rows and pairs them up.
#pragma once

#include "lora.cuh"

namespace mtc {
namespace lora {

template <int DT>
constexpr int pieces = DT == MTC_F32 ? 3 : 1;    // of weights and activations

__device__ __forceinline__ uint32_t high_halves(uint32_t lo, uint32_t hi) { return __byte_perm(lo, hi, 0x7632); }
__device__ __forceinline__ uint32_t low_halves(uint32_t lo, uint32_t hi) { return __byte_perm(lo, hi, 0x5410); }

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// What is rounded for the first piece: within the largest of bf16, so that a f32 value above that does not become an infinity (one that is an infinity is left to the next piece)
__device__ __forceinline__ float first_piece(float v) {
    float r;
    asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(0x1.FEp127f));
    return r;
}

__device__ __forceinline__ float or_zero(float v) { return fabsf(v) < INFINITY ? v : 0.0f; }

// How f32 values are cut into pieces: without a look at them, where a value beyond the largest of bf16 leaves NaN in every sum that it goes into; with the first piece held back, where only
// infinities and NaN do; or with these in the last piece alone, which is multiplied with the others' first pieces only: these have the values' signs, and are zero where the values are.
enum class Care { none, large, all };

// W neighbouring values as operand pieces: pairs of 16-bit values (one value: the low half)
template <int DT, int W>
struct Vals {
    static constexpr int P = pieces<DT>, N = (W + 1) / 2;
    uint32_t w[P][N];

    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int i = 0; i < N; ++i) w[p][i] = 0;
    }
    // aligned to W values
    template <Care CARE>
    __device__ __forceinline__ void load(const void *base, size_t at, bool there) {
        zero();
        if (!there) return;
        if constexpr (DT != MTC_F32) {
            const uint16_t *const p = static_cast<const uint16_t *>(base) + at;
            if constexpr (W == 8) {
                const uint4 q = *reinterpret_cast<const uint4 *>(p);
                w[0][0] = q.x, w[0][1] = q.y, w[0][2] = q.z, w[0][3] = q.w;
            } else if constexpr (W == 4) {
                const uint2 q = *reinterpret_cast<const uint2 *>(p);
                w[0][0] = q.x, w[0][1] = q.y;
            } else if constexpr (W == 2) {
                w[0][0] = *reinterpret_cast<const uint32_t *>(p);
            } else {
                w[0][0] = *p;
            }
        } else {
            const float *const p = static_cast<const float *>(base) + at;
            float v[W];
            if constexpr (W >= 4) {
#pragma unroll
                for (int i = 0; i < W / 4; ++i) {
                    const float4 q = reinterpret_cast<const float4 *>(p)[i];
                    v[4 * i] = q.x, v[4 * i + 1] = q.y, v[4 * i + 2] = q.z, v[4 * i + 3] = q.w;
                }
            } else if constexpr (W == 2) {
                const float2 q = *reinterpret_cast<const float2 *>(p);
                v[0] = q.x, v[1] = q.y;
            } else {
                v[0] = *p;
            }
            split<CARE>(v);
        }
    }
    // n of them exist, any alignment
    template <Care CARE>
    __device__ __forceinline__ void load_any(const void *base, size_t at, int n) {
        if constexpr (DT == MTC_F32) {
            float v[W];
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = i < n ? static_cast<const float *>(base)[at + i] : 0.0f;
            split<CARE>(v);
        } else {
            zero();
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (i < n) w[0][i / 2] |= static_cast<uint32_t>(static_cast<const uint16_t *>(base)[at + i]) << (i & 1) * 16;
        }
    }
    template <Care CARE>
    __device__ __forceinline__ void split(float (&v)[W]) {
        auto piece_of = [](float x, int k) {
            if (CARE == Care::all && k + 1 < P) x = or_zero(x);
            return CARE != Care::none && k == 0 ? first_piece(x) : x;
        };
#pragma unroll
        for (int k = 0; k < P; ++k) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float lo = v[2 * i], hi = W == 1 ? 0.0f : v[W == 1 ? 0 : 2 * i + 1];
                const uint32_t u = w[k][i] = bf16_pair(piece_of(lo, k), piece_of(hi, k));
                v[2 * i] = lo - __uint_as_float(u << 16);
                if (W > 1) v[W == 1 ? 0 : 2 * i + 1] = hi - __uint_as_float(u & 0xFFFF0000u);
            }
        }
    }
    // value j of x with value j of y, as a pair
    static __device__ __forceinline__ uint32_t pair(const Vals &x, const Vals &y, int p, int j) {
        return j & 1 ? high_halves(x.w[p][j / 2], y.w[p][j / 2]) : low_halves(x.w[p][j / 2], y.w[p][j / 2]);
    }
};

// d += a b: 16 x 16 values of a, 16 x 8 of b
template <bool HALF>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (HALF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight results next to each other: + base, rounded, out
template <int DT>
struct Eight {
    uint32_t w[DT == MTC_F32 ? 8 : 4];
    __device__ __forceinline__ void load(const void *base, size_t at, bool there) {
        constexpr int W = DT == MTC_F32 ? 8 : 4;
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = 0;
        if (!there) return;
        const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const char *>(base) + at * (DT == MTC_F32 ? 4 : 2));
#pragma unroll
        for (int i = 0; i < W / 4; ++i) {
            const uint4 q = p[i];
            w[4 * i] = q.x, w[4 * i + 1] = q.y, w[4 * i + 2] = q.z, w[4 * i + 3] = q.w;
        }
    }
    __device__ __forceinline__ void load_any(const void *base, size_t at, int n) {
#pragma unroll
        for (int i = 0; i < (DT == MTC_F32 ? 8 : 4); ++i) w[i] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i >= n) break;
            if constexpr (DT == MTC_F32) w[i] = static_cast<const uint32_t *>(base)[at + i];
            else w[i / 2] |= static_cast<uint32_t>(static_cast<const uint16_t *>(base)[at + i]) << (i & 1) * 16;
        }
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (DT == MTC_F32) return __uint_as_float(w[i]);
        const uint32_t u = w[i / 2];
        if constexpr (DT == MTC_BF16) return __uint_as_float(i & 1 ? u & 0xFFFF0000u : u << 16);
        return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? u >> 16 : u)));
    }
    template <bool VEC = true>
    __device__ __forceinline__ void add_and_store(void *out, size_t at, const float (&v)[8], float factor, int n = 8) const {
        float r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = fmaf(v[i], factor, value(i));
        if constexpr (VEC) {
            put(out, at, r);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) st_from_f32(out, at + i, r[i], DT);
        }
    }
    static __device__ __forceinline__ void put(void *out, size_t at, const float (&r)[8]) {
        if constexpr (DT == MTC_F32) {
            float4 *p = reinterpret_cast<float4 *>(static_cast<float *>(out) + at);
            p[0] = make_float4(r[0], r[1], r[2], r[3]);
            p[1] = make_float4(r[4], r[5], r[6], r[7]);
        } else {
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (DT == MTC_BF16) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(r[2 * i], r[2 * i + 1]);
                    u[i] = *reinterpret_cast<const uint32_t *>(&h);
                } else {
                    const __half2 h = __floats2half2_rn(r[2 * i], r[2 * i + 1]);
                    u[i] = *reinterpret_cast<const uint32_t *>(&h);
                }
            }
            *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(out) + at) = make_uint4(u[0], u[1], u[2], u[3]);
        }
    }
};

struct Tile {
    int e;                                       // n_adapters and above: rows of none; -1: no such tile
    uint32_t p0, n;
};

// The tile of this cluster: tiles of `rows` places are dealt out adapter by adapter.  By every warp for itself.
__device__ __forceinline__ Tile find_tile(const LoraArgs &a, int id, int rows, bool none) {
    // the places behind the last adapter's, and those before the first one's, are of no adapter
    const int lane = threadIdx.x & 31, last = none ? a.n_adapters + 1 : a.n_adapters - 1;
    const uint32_t R = a.n_rows;
    long long before = 0;                        // offsets that run backwards may name more tiles than 32 bits hold
    for (int e0 = 0; e0 <= last; e0 += 32) {
        const int e = e0 + lane;
        uint32_t from = 0, to = 0;
        if (e <= last) {
            from = e <= a.n_adapters ? min(a.offsets[e], R) : 0;
            to = e < a.n_adapters ? min(a.offsets[e + 1], R) : e == a.n_adapters ? R : min(a.offsets[0], R);
        }
        const uint32_t n = to > from ? to - from : 0;
        const long long mine = (static_cast<long long>(n) + rows - 1) / rows;
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const long long first = before + upto - mine;
        const uint32_t hit = __ballot_sync(0xffffffffu, id >= first && id < first + mine);
        if (hit) {
            const uint32_t skip = static_cast<uint32_t>(id - first) * rows;
            const int src = __ffs(hit) - 1;
            return {e0 + src, __shfl_sync(0xffffffffu, from + skip, src), __shfl_sync(0xffffffffu, min(n - skip, static_cast<uint32_t>(rows)), src)};
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return {-1, 0, 0};
}

// f16: a power of two that brings a row's largest number to between 2^14 and 2^15, within what f32 can divide by.  So high that the least of a row keep their bits: two pieces of f16 reach
// down to 2^-24, 38 octaves below, and are 16 bits and more of every value down to 2^-22 of the largest.  (Products with f16 weights of 2^16 leave f32 sums room.)
__device__ __forceinline__ float unit_of(float most) { return __uint_as_float(static_cast<uint32_t>(max(static_cast<int>(__float_as_uint(most) >> 23) - 14, 1)) << 23); }
// (infinities and NaN are not counted: beside them all numbers of a row would be zeros or infinities)
__device__ __forceinline__ float most_of(float4 s) { return fmaxf(fmaxf(fabsf(or_zero(s.x)), fabsf(or_zero(s.y))), fmaxf(fabsf(or_zero(s.z)), fabsf(or_zero(s.w)))); }
// Four ranks' sums from rank r on: zeros behind the last rank, where an infinity in x or dy has met the zeros of weights that do not exist
__device__ __forceinline__ float4 ranks_of(float4 s, int r, int rank) {
    if (r + 4 > rank) {
        if (r >= rank) s.x = 0.0f;
        if (r + 1 >= rank) s.y = 0.0f;
        if (r + 2 >= rank) s.z = 0.0f;
        s.w = 0.0f;
    }
    return s;
}
// Four neighbours as operand pieces.  f16: divided by `unit`, since it has five bits of exponent.
template <int DT, Care CARE = Care::all>
__device__ __forceinline__ void hold_pieces(float4 s, float unit, uint2 *piece) {
    constexpr int H = DT == MTC_F32 ? 3 : 2;
    float v[4] = {s.x, s.y, s.z, s.w};
    if constexpr (DT == MTC_F16) {
        const float inv = 1.0f / unit;           // exact
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= inv;
    }
#pragma unroll
    for (int p = 0; p < H; ++p) {
        uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float &x = v[2 * i], &y = v[2 * i + 1];
            if constexpr (DT == MTC_F16) {
                const __half2 h = __floats2half2_rn(x, y);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
                const float2 f = __half22float2(h);
                x = fabsf(x) < INFINITY ? x - f.x : 0.0f, y = fabsf(y) < INFINITY ? y - f.y : 0.0f;
            } else {
                if (CARE == Care::all && H == 3 && p + 1 < H) w[i] = p == 0 ? bf16_pair(first_piece(or_zero(x)), first_piece(or_zero(y))) : bf16_pair(or_zero(x), or_zero(y));
                else w[i] = p == 0 ? bf16_pair(first_piece(x), first_piece(y)) : bf16_pair(x, y);
                x -= __uint_as_float(w[i] << 16), y -= __uint_as_float(w[i] & 0xFFFF0000u);
            }
        }
        piece[p] = make_uint2(w[0], w[1]);
    }
}
// ... each `apart` values behind the other
template <int DT>
__device__ __forceinline__ void hold(float4 s, float unit, uint16_t *at, int apart) {
    constexpr int H = DT == MTC_F32 ? 3 : 2;
    uint2 w[H];
    hold_pieces<DT>(s, unit, w);
#pragma unroll
    for (int p = 0; p < H; ++p) *reinterpret_cast<uint2 *>(at + p * apart) = w[p];
}

// Rows of no adapter, by the CTAs of a cluster: columns from .. to of this one; zeros of `low` where it is kept
template <int DT, int THREADS, bool VEC = true>
__device__ __forceinline__ void copy_rows(const LoraArgs &a, const int *row_of, int n, int from, int to, bool keep, int cr, int cs) {
    if (a.base != a.out) {
        for (int r = threadIdx.x >> 5; r < n; r += THREADS / 32) {
            const int row = row_of[r];
            if (row < 0) continue;
            for (int c = from + (threadIdx.x & 31) * 8; c < to; c += 256) {
                const size_t at = static_cast<size_t>(row) * a.c_out + c;
                Eight<DT> v;
                if constexpr (VEC) v.load(a.base, at, a.base != nullptr);
                else v.load_any(a.base, at, a.base ? to - c : 0);
                const float zero[8] = {};
                v.template add_and_store<VEC>(a.out, at, zero, 1.0f, to - c);
            }
        }
    }
    if (keep)
        for (int i = threadIdx.x + cr * THREADS; i < n * a.rank; i += THREADS * cs)
            if (row_of[i / a.rank] >= 0) a.low[static_cast<size_t>(row_of[i / a.rank]) * a.rank + i % a.rank] = 0.0f;
}

// Tiles of `rows` rows that there are at most: one of fewer rows for each adapter and on both sides of them
inline long long most_tiles(const LoraArgs &a, int rows) {
    const long long tiles = a.n_rows / rows + a.n_adapters + 2ll;
    return tiles < a.n_rows ? tiles : a.n_rows;
}

// Clusters
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }      // nothing was written
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float4 ld_cta(const float *p, uint32_t rank) {
    uint32_t at;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

template <typename... P, typename... A>
cudaError_t launch_cluster(void (*kern)(P...), unsigned ctas, int threads, int cluster, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute la[2];
    la[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    la[0].val.programmaticStreamSerializationAllowed = 1;
    la[1].id = cudaLaunchAttributeClusterDimension;
    la[1].val.clusterDim.x = cluster;
    la[1].val.clusterDim.y = la[1].val.clusterDim.z = 1;
    cfg.attrs = la;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
}

}  // namespace lora
}  // namespace mtc
