// Eight 16-bit elements at a time of rows that start anywhere: the pieces that the copies and the quantising kernels move.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace t2sp {

// An ordinary load: some of the kernels that call this start while the kernel before still writes what they are about to read, and a load through the
// read-only path is defined only for memory that nobody writes while the kernel runs, from its start on.
__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// The eight elements from element m on (0 .. 7) of two aligned pieces.
__device__ __forceinline__ uint4 row16_cut(const uint4& a, const uint4& b, int m) {
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = m & 4 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = m & 2 ? w[i + 1] : w[i];
    const int bits = (m & 1) * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], bits);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Elements src[0 .. 7], zeros from src[left] on. A piece that does not start on 16 bytes is cut out of the two aligned pieces around it, where
// these lie within [begin, end), the operand's memory (eight 2-byte loads a thread kept a copy at a fifth of the memory's rate).
__device__ __forceinline__ uint4 row16_load(const uint16_t* src, int left, const uint16_t* begin, const uint16_t* end) {
    const int m = static_cast<int>(reinterpret_cast<uintptr_t>(src) & 15) >> 1;
    const uint16_t* base = src - m;
    if (left >= 8 && m == 0) return load16(src);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (left >= 8 && base >= begin && base + 16 <= end) {
        const uint4 a = load16(base), b = load16(base + 8);
        return row16_cut(a, b, m);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < left) (&v.x)[j >> 1] |= static_cast<uint32_t>(src[j]) << (16 * (j & 1));
    return v;
}

// dst[0 .. 7] = v, elements from dst[left] on are left alone.
__device__ __forceinline__ void row16_store(uint16_t* dst, uint4 v, int left) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(dst);
    if (left >= 8 && (at & 15) == 0) {
        *reinterpret_cast<uint4*>(dst) = v;
    } else if (left >= 8 && (at & 3) == 0) {
        uint32_t* d = reinterpret_cast<uint32_t*>(dst);
        d[0] = v.x; d[1] = v.y; d[2] = v.z; d[3] = v.w;
    } else if (left >= 8) {   // two bytes off a word
        uint32_t* d = reinterpret_cast<uint32_t*>(dst + 1);
        dst[0] = static_cast<uint16_t>(v.x);
        d[0] = __funnelshift_r(v.x, v.y, 16);
        d[1] = __funnelshift_r(v.y, v.z, 16);
        d[2] = __funnelshift_r(v.z, v.w, 16);
        dst[7] = static_cast<uint16_t>(v.w >> 16);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) dst[j] = static_cast<uint16_t>((&v.x)[j >> 1] >> (16 * (j & 1)));
    }
}

}  // namespace t2sp
