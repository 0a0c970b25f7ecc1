// Kernels of the 4-bit matrices: quantising, reading back and products with a few rows.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

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
    return ((static_cast<long long>(e) * strips + strip) * kblocks + (k >> 6)) * 512 + (g * 4 + (kk >> 4)) * 16 +
           ((kk >> 2) & 3) * 4 + ((j & 1) << 1) + (j >> 1);
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

template <class T, class O>
__global__ void q4_gemv_kernel(const Q4Params p) {
    const int kblocks = q4_kblocks(p.K), strips = q4_strips(p.N), groups = q4_groups(p.K, p.group);
    const int n = blockIdx.x * blockDim.x + threadIdx.x, r = blockIdx.y;
    const int e = p.index ? p.index[r] : 0;
    if (e >= p.E && threadIdx.x == 0 && blockIdx.x == 0) atomicOr(p.status, ST_BAD_INDEX);
    if (n >= p.N || e < 0 || e >= p.E) return;
    const T* x = static_cast<const T*>(p.x) + (r / p.per) * p.ldx;
    float acc = 0.f;
    for (int k0 = 0; k0 < p.K; k0 += p.group) {
        float part = 0.f;
        for (int k = k0; k < min(k0 + p.group, p.K); ++k) part += q4_value(p, e, n, k, kblocks, strips) * to_f32(x[k]);
        acc += part * q4_scale<T>(p, e, n, k0, strips, groups);
    }
    static_cast<O*>(p.y)[r * p.ldy + n] = rounded<O>(acc);
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
    const dim3 grid((p.N + 127) / 128, p.R);
    if (p.bf16) {
        if (p.out_f32) q4_gemv_kernel<__nv_bfloat16, float><<<grid, 128, 0, stream>>>(p);
        else q4_gemv_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, 128, 0, stream>>>(p);
    } else {
        if (p.out_f32) q4_gemv_kernel<__half, float><<<grid, 128, 0, stream>>>(p);
        else q4_gemv_kernel<__half, __half><<<grid, 128, 0, stream>>>(p);
    }
    return cudaGetLastError();
}

}  // namespace t2sp
