// Grouped products: C[t] = A[t] x B[e(t)] over rows sorted by group, and the gradient of B.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "grouped.h"

namespace t2sp {

namespace {

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f32(float v, float* p) { *p = v; }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16* p) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half* p) { *p = __float2half_rn(v); }

// True when the offsets do not decrease and stay inside the rows (checked by the whole block).
__device__ bool offsets_valid(const int* offsets, int E, int rows) {
    int bad = 0;
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
        const int lo = offsets[e], hi = offsets[e + 1];
        if (lo < 0 || hi < lo || hi > rows) bad = 1;
    }
    return __syncthreads_or(bad) == 0;
}

// 64 x 64 tiles of one group, 4 x 4 values a thread, fp32 sums.
template <class T, class O>
__global__ void __launch_bounds__(256) grouped_simple_kernel(const GroupedParams p) {
    __shared__ float sp[16][65], sq[16][65];
    if (!offsets_valid(p.offsets, p.E, p.rows)) {
        if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) atomicOr(p.status, ST_BAD_OFFSETS);
        return;
    }
    const int e = blockIdx.z;
    const int lo = p.offsets[e], hi = p.offsets[e + 1];
    const T* a = static_cast<const T*>(p.a);
    const T* b = static_cast<const T*>(p.b) + (p.grad ? 0 : e * p.bs_b);
    O* c = static_cast<O*>(p.c) + (p.grad ? e * p.bs_c : 0);
    const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
    const int r_begin = p.grad ? 0 : lo, r_end = p.grad ? p.K : hi;
    const int k_begin = p.grad ? lo : 0, k_end = p.grad ? hi : p.K;
    const int n0 = blockIdx.x * 64;
    for (int r0 = r_begin + blockIdx.y * 64; r0 < r_end; r0 += gridDim.y * 64) {
        float acc[4][4] = {};
        for (int k0 = k_begin; k0 < k_end; k0 += 16) {
            for (int i = threadIdx.x; i < 1024; i += 256) {
                const int x = i & 63, kk = i >> 6;
                const long long k = k0 + kk;
                const int r = r0 + x, n = n0 + x;
                float v = 0.f, w = 0.f;
                if (k < k_end && r < r_end) v = to_f32(p.grad ? a[k * p.lda + r] : a[r * p.lda + k]);
                if (k < k_end && n < p.N) w = to_f32(!p.grad && p.trans_b ? b[n * p.ldb + k] : b[k * p.ldb + n]);
                sp[kk][x] = v;
                sq[kk][x] = w;
            }
            __syncthreads();
            for (int kk = 0; kk < 16; ++kk)
                for (int i = 0; i < 4; ++i)
                    for (int j = 0; j < 4; ++j) acc[i][j] += sp[kk][tr * 4 + i] * sq[kk][tc + 16 * j];
            __syncthreads();
        }
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j) {
                const long long r = r0 + tr * 4 + i;
                const int n = n0 + tc + 16 * j;
                if (r < r_end && n < p.N) from_f32(acc[i][j], c + r * p.ldc + n);
            }
    }
}

template <class T>
void launch_typed(const GroupedParams& p, dim3 grid, cudaStream_t stream) {
    if (p.out_f32) grouped_simple_kernel<T, float><<<grid, 256, 0, stream>>>(p);
    else grouped_simple_kernel<T, T><<<grid, 256, 0, stream>>>(p);
}

}  // namespace

cudaError_t grouped_launch(const GroupedParams& p, cudaStream_t stream) {
    const int tiles = ((p.grad ? p.K : p.rows) + 63) / 64;
    const dim3 grid((p.N + 63) / 64, tiles < 64 ? tiles : 64, p.E);
    if (p.bf16) launch_typed<__nv_bfloat16>(p, grid, stream);
    else launch_typed<__half>(p, grid, stream);
    return cudaGetLastError();
}

}  // namespace t2sp
