// Kernels of the 4-bit matrices: quantising, reading back and products with a few rows.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "launch_util.cuh"
#include "q4.h"

namespace t2sp {

namespace {

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T rounded(float v);
template <> __device__ __forceinline__ float rounded<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half rounded<__half>(float v) { return __float2half_rn(v); }

// Byte of (row pair g, g + 8; k) inside the packed matrices.
__device__ __forceinline__ long long q4_byte(int e, int strip, int g, int k, int kblocks, int strips) {
    const int kk = k & 63, j = kk & 3;
    return ((static_cast<long long>(e) * strips + strip) * kblocks + (k >> 6)) * 512 + (g * 4 + ((kk >> 2) & 3)) * 16 +
           (kk >> 4) * 4 + ((j & 1) << 1) + (j >> 1);
}

// The nearest of -7 .. 7 to v / scale, ties to even. The quotient of two 16-bit values cannot round onto a tie that
// the exact quotient does not hold: a tie (h + 1/2) * scale has at most 15 significant bits, so an unequal v differs
// from it by more than 2^-17 relative, far above the division's 2^-24.
__device__ __forceinline__ int q4_round(float v, float scale) {
    if (!(scale > 0.f)) return 0;
    const float q = rintf(__fdiv_rn(v, scale));
    return static_cast<int>(fminf(fmaxf(q, -7.f), 7.f));  // a NaN becomes -7; its scale is not a number either
}

// One thread for the row pair (g, g + 8) of a strip and one group of k.
template <class T>
__global__ void q4_pack_kernel(const Q4Params p) {
    const int kblocks = q4_kblocks(p.K), strips = q4_strips(p.N), groups = q4_groups(p.K, p.group);
    const long long idx = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    const int g = static_cast<int>(idx & 7);
    long long rest = idx >> 3;
    const int strip = static_cast<int>(rest % strips);
    rest /= strips;
    const int grp = static_cast<int>(rest % groups), e = static_cast<int>(rest / groups);
    if (e >= p.E) return;
    const T* w = static_cast<const T*>(p.w) + e * p.bs_w;
    auto load = [&](int n, long long k) {
        if (n >= p.N || k >= p.K) return 0.f;
        return to_f32(p.trans_b ? w[n * p.ldw + k] : w[k * p.ldw + n]);
    };
    const int k0 = grp * p.group, k1 = min(k0 + p.group, kblocks * 64);
    float scale[2];
    for (int h = 0; h < 2; ++h) {
        float m = 0.f;
        bool nan = false;
        for (int k = k0; k < k1; ++k) {
            const float v = fabsf(load(strip * 16 + g + 8 * h, k));
            nan = nan || v != v;
            m = fmaxf(m, v);
        }
        const T s = rounded<T>(nan ? __int_as_float(0x7fc00000) : __fdiv_rn(m, 7.f));
        scale[h] = to_f32(s);
        reinterpret_cast<T*>(p.s)[((static_cast<long long>(e) * strips + strip) * groups + grp) * 16 + g * 2 + h] = s;
    }
    for (int k = k0; k < k1; ++k) {
        const int lo = q4_round(load(strip * 16 + g, k), scale[0]) + 8, hi = q4_round(load(strip * 16 + g + 8, k), scale[1]) + 8;
        p.q[q4_byte(e, strip, g, k, kblocks, strips)] = static_cast<uint8_t>(lo | (hi << 4));
    }
}

__device__ __forceinline__ int q4_value(const Q4Params& p, int e, int n, int k, int kblocks, int strips) {
    const int row = n & 15;
    const int b = p.q[q4_byte(e, n >> 4, row & 7, k, kblocks, strips)];
    return ((row >> 3) ? b >> 4 : b & 15) - 8;
}
template <class T>
__device__ __forceinline__ float q4_scale(const Q4Params& p, int e, int n, int k, int strips, int groups) {
    const int row = n & 15;
    return to_f32(reinterpret_cast<const T*>(p.s)[((static_cast<long long>(e) * strips + (n >> 4)) * groups + k / p.group) * 16 +
                                                  (row & 7) * 2 + (row >> 3)]);
}

template <class T>
__global__ void q4_unpack_kernel(const Q4Params p) {
    const int kblocks = q4_kblocks(p.K), strips = q4_strips(p.N), groups = q4_groups(p.K, p.group);
    const long long idx = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    const int inner = p.trans_b ? p.K : p.N, outer = p.trans_b ? p.N : p.K;
    const int i = static_cast<int>(idx % inner);
    const long long rest = idx / inner;
    const int o = static_cast<int>(rest % outer), e = static_cast<int>(rest / outer);
    if (e >= p.E) return;
    const int n = p.trans_b ? o : i, k = p.trans_b ? i : o;
    const float v = q4_value(p, e, n, k, kblocks, strips) * q4_scale<T>(p, e, n, k, strips, groups);
    static_cast<T*>(p.wout)[e * p.bs_w + o * p.ldw + i] = rounded<T>(v);
}

// ---------------------------------------------------------------- products of a few rows
constexpr int kGemvWarps = 8;
constexpr int kGemvUnroll = 4;                                 // 64-k blocks a warp has in flight for each of its strips
constexpr int kGemvChunk = kGemvWarps * kGemvUnroll * 64;      // k values the CTA takes at a time
constexpr int kGemvStrips = 2;                                 // strips of 16 n a CTA computes

// Two 16-bit values q - 8 from the nibbles at bits 0..3 and 16..19 of `w`: the nibble becomes the low mantissa bits of
// 1024 (fp16) or 128 (bf16), where a unit is 1, and 1032 or 136 is subtracted; both steps are exact.
template <class T> __device__ __forceinline__ uint32_t q4_pair(uint32_t w);
template <> __device__ __forceinline__ uint32_t q4_pair<__half>(uint32_t w) {
    const uint32_t v = (w & 0x000f000fu) | 0x64006400u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408)));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <> __device__ __forceinline__ uint32_t q4_pair<__nv_bfloat16>(uint32_t w) {
    const uint32_t v = (w & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v),
                                     __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308)));
    return *reinterpret_cast<const uint32_t*>(&r);
}

template <class T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

template <class T> __device__ __forceinline__ float2 pair_f32(uint32_t w);
template <> __device__ __forceinline__ float2 pair_f32<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <> __device__ __forceinline__ float2 pair_f32<__nv_bfloat16>(uint32_t w) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}

template <int NT>
struct GemvShared {
    static constexpr int kPitch = kGemvChunk * 2 + 32;   // bytes of a staged row: rows 32 bytes apart modulo 128, so that a
                                                         // fragment load of 8 rows x 32 bytes meets every bank once
    uint8_t x[8 * NT * kPitch];
    float part[kGemvWarps][kGemvStrips * 16][8 * NT + 1];
    int rows[8 * NT];                                    // rows of y that this pass computes
    int count;
};

// Y[r] = X[r / per] x W[index[r]]. A CTA computes kGemvStrips strips of 16 n for the rows of one matrix: blockIdx.y is a row of y, and
// the CTA of the first row that names a matrix takes all rows that name it, so a matrix is read once however many
// rows share it (up to 8 NT rows at a time). The warps divide k; each turns 16-byte pieces of packed weights into A fragments of
// m16n8k16 (16 n x 16 k of integers, exact in 16 bits) against B fragments of x (8 rows), sums a group in the instruction's fp32
// accumulator, scales it in fp32 and adds it up; the eight partial sums meet in shared memory in a fixed order.
template <class T, class O, int NT, bool G32>
__global__ void __launch_bounds__(kGemvWarps * 32) q4_gemv_kernel(const Q4Params p) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    GemvShared<NT>& sh = *reinterpret_cast<GemvShared<NT>*>(smem_raw);
    const int kblocks = q4_kblocks(p.K), strips = q4_strips(p.N), groups = q4_groups(p.K, p.group);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int lead = blockIdx.y;
    int e = 0;
    if (p.index) {
        e = p.index[lead];
        if (e >= p.E) {
            if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(p.status, ST_BAD_INDEX);
            return;
        }
        if (e < 0) return;
        int earlier = 0;
        for (int r = threadIdx.x; r < lead; r += blockDim.x) earlier |= p.index[r] == e;
        if (__syncthreads_or(earlier)) return;
    }
    const int strip0 = blockIdx.x * kGemvStrips;
    const uint8_t* qbase = p.q + (static_cast<long long>(e) * strips + strip0) * kblocks * 512 + lane * 16;
    const T* sbase = reinterpret_cast<const T*>(p.s) + (static_cast<long long>(e) * strips + strip0) * groups * 16 + g * 2;
    const int nstrips = min(kGemvStrips, strips - strip0);
    const int chunks = (kblocks * 64 + kGemvChunk - 1) / kGemvChunk;
    const int gsh = p.group == 128 ? 1 : 0;

    uint4 q[kGemvStrips][kGemvUnroll];
    uint32_t sc[kGemvStrips][kGemvUnroll][G32 ? 2 : 1];
    auto fetch = [&](int chunk, int u) {
        const int kb = (chunk * kGemvWarps + warp) * kGemvUnroll + u;
#pragma unroll
        for (int i = 0; i < kGemvStrips; ++i) {
            q[i][u] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
#pragma unroll
            for (int h = 0; h < (G32 ? 2 : 1); ++h) sc[i][u][h] = 0;
            if (kb < kblocks && i < nstrips) {
                q[i][u] = load_stream(qbase + (static_cast<long long>(i) * kblocks + kb) * 512);
#pragma unroll
                for (int h = 0; h < (G32 ? 2 : 1); ++h)
                    sc[i][u][h] = *reinterpret_cast<const uint32_t*>(
                        sbase + (static_cast<long long>(i) * groups + (G32 ? kb * 2 + h : kb >> gsh)) * 16);
            }
        }
    };
    const bool x_aligned = (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && p.ldx % 8 == 0;

    for (int pass = 0;; ++pass) {
        // the rows of this pass
        if (warp == 0) {
            const int base = pass * 8 * NT;   // rows that earlier passes took
            int found;
            if (p.index) {
                int seen = 0;
                for (int r0 = lead; r0 < p.R && seen < base + 8 * NT; r0 += 32) {
                    const int r = r0 + lane;
                    const unsigned hit = __ballot_sync(0xffffffffu, r < p.R && p.index[r] == e);
                    const int slot = seen + __popc(hit & ((1u << lane) - 1)) - base;
                    if ((hit >> lane & 1) && slot >= 0 && slot < 8 * NT) sh.rows[slot] = r;
                    seen += __popc(hit);
                }
                found = max(0, min(8 * NT, seen - base));
            } else {
                found = max(0, min(8 * NT, p.R - base));
                for (int i = lane; i < found; i += 32) sh.rows[i] = base + i;
            }
            if (lane == 0) sh.count = found;
        }
        __syncthreads();
        const int count = sh.count;
        if (count == 0) return;
        float acc[kGemvStrips][NT][4] = {};
#pragma unroll
        for (int u = 0; u < kGemvUnroll; ++u) fetch(0, u);
        for (int chunk = 0; chunk < chunks; ++chunk) {
            // the chunk of x, zero beyond K
            for (int i = threadIdx.x; i < count * (kGemvChunk / 8); i += blockDim.x) {
                const int row = i / (kGemvChunk / 8), k8 = (i % (kGemvChunk / 8)) * 8;
                const long long k = chunk * static_cast<long long>(kGemvChunk) + k8;
                const uint16_t* src = static_cast<const uint16_t*>(p.x) + (sh.rows[row] / p.per) * p.ldx + k;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (x_aligned && k + 8 <= p.K) {
                    v = *reinterpret_cast<const uint4*>(src);
                } else {
                    uint32_t* w = &v.x;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (k + j < p.K) w[j >> 1] |= uint32_t(src[j]) << (16 * (j & 1));
                }
                *reinterpret_cast<uint4*>(sh.x + row * GemvShared<NT>::kPitch + k8 * 2) = v;
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < kGemvUnroll; ++u) {
                const int kk = (warp * kGemvUnroll + u) * 64;
                float c[kGemvStrips][NT][4] = {};
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    uint2 b[NT];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        b[n] = make_uint2(0, 0);
                        if (n * 8 + g < count) b[n] = *reinterpret_cast<const uint2*>(sh.x + (n * 8 + g) * GemvShared<NT>::kPitch + (kk + 16 * s + 4 * t) * 2);
                    }
#pragma unroll
                    for (int i = 0; i < kGemvStrips; ++i) {
                        const uint32_t w = (&q[i][u].x)[s];
                        const uint32_t a[4] = {q4_pair<T>(w), q4_pair<T>(w >> 4), q4_pair<T>(w >> 8), q4_pair<T>(w >> 12)};
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma_16816<T>(c[i][n], a, b[n].x, b[n].y);
                    }
                    if (s == 3 || (G32 && s == 1)) {
#pragma unroll
                        for (int i = 0; i < kGemvStrips; ++i) {
                            const float2 f = pair_f32<T>(sc[i][u][G32 ? s >> 1 : 0]);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                acc[i][n][0] += f.x * c[i][n][0];
                                acc[i][n][1] += f.x * c[i][n][1];
                                acc[i][n][2] += f.y * c[i][n][2];
                                acc[i][n][3] += f.y * c[i][n][3];
                                c[i][n][0] = c[i][n][1] = c[i][n][2] = c[i][n][3] = 0.f;
                            }
                        }
                    }
                }
                if (chunk + 1 < chunks) fetch(chunk + 1, u);
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < kGemvStrips; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) sh.part[warp][i * 16 + g + (j >> 1) * 8][n * 8 + 2 * t + (j & 1)] = acc[i][n][j];
        __syncthreads();
        for (int i = threadIdx.x; i < kGemvStrips * 16 * count; i += blockDim.x) {
            const int n = strip0 * 16 + i % (kGemvStrips * 16), row = i / (kGemvStrips * 16);
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kGemvWarps; ++w) v += sh.part[w][i % (kGemvStrips * 16)][row];
            if (n < p.N) static_cast<O*>(p.y)[sh.rows[row] * p.ldy + n] = rounded<O>(v);
        }
        __syncthreads();   // the next pass writes the shared rows
    }
}

template <class T, class O, int NT, bool G32>
cudaError_t gemv_launch(const Q4Params& p, cudaStream_t stream) {
    auto kern = q4_gemv_kernel<T, O, NT, G32>;
    static std::atomic<bool> configured[kMaxDev];
    if (cudaError_t e = allow_smem(kern, sizeof(GemvShared<NT>), configured)) return e;
    const dim3 grid((q4_strips(p.N) + kGemvStrips - 1) / kGemvStrips, p.index ? p.R : 1);
    kern<<<grid, kGemvWarps * 32, sizeof(GemvShared<NT>), stream>>>(p);
    return cudaGetLastError();
}

template <class T, class O>
cudaError_t gemv_typed(const Q4Params& p, cudaStream_t stream) {
    if (p.R <= 8) return p.group == 32 ? gemv_launch<T, O, 1, true>(p, stream) : gemv_launch<T, O, 1, false>(p, stream);
    return p.group == 32 ? gemv_launch<T, O, 2, true>(p, stream) : gemv_launch<T, O, 2, false>(p, stream);
}

unsigned blocks_for(long long work) { return static_cast<unsigned>((work + 127) / 128); }

}  // namespace

cudaError_t q4_pack_launch(const Q4Params& p, cudaStream_t stream) {
    const long long work = 8ll * q4_strips(p.N) * q4_groups(p.K, p.group) * p.E;
    if (p.bf16) q4_pack_kernel<__nv_bfloat16><<<blocks_for(work), 128, 0, stream>>>(p);
    else q4_pack_kernel<__half><<<blocks_for(work), 128, 0, stream>>>(p);
    return cudaGetLastError();
}

cudaError_t q4_unpack_launch(const Q4Params& p, cudaStream_t stream) {
    const long long work = static_cast<long long>(p.E) * p.K * p.N;
    if (p.bf16) q4_unpack_kernel<__nv_bfloat16><<<blocks_for(work), 128, 0, stream>>>(p);
    else q4_unpack_kernel<__half><<<blocks_for(work), 128, 0, stream>>>(p);
    return cudaGetLastError();
}

cudaError_t q4_gemv_launch(const Q4Params& p, cudaStream_t stream) {
    if (p.bf16) return p.out_f32 ? gemv_typed<__nv_bfloat16, float>(p, stream) : gemv_typed<__nv_bfloat16, __nv_bfloat16>(p, stream);
    return p.out_f32 ? gemv_typed<__half, float>(p, stream) : gemv_typed<__half, __half>(p, stream);
}

}  // namespace t2sp
