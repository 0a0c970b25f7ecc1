// Kernels of the 4-bit matrices: quantising, reading back and products with a few rows.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "launch_util.cuh"
#include "ptx.cuh"
#include "q4.h"
#include "row16.cuh"
#include "umma_core.cuh"
#include "umma_launch.h"

namespace t2sp {

namespace {

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T rounded(float v);
template <> __device__ __forceinline__ float rounded<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half rounded<__half>(float v) { return __float2half_rn(v); }

// The sixteen integers q - 8 of a lane's word as 16-bit floating-point A-fragment registers, exactly: the nibbles become low mantissa
// bits of a number whose last bit counts 1 (128 in bf16, 1024 in fp16; fp16 has room for the second nibble as it stands, counting
// 16), and one packed operation takes the constant off. (Leaving fp16 nibbles as subnormal numbers and the constant to the sums of x
// saves that operation, but the tensor core aligns a subnormal product by its exponent field and drops seven to ten bits of it.)
template <class T> struct Q4Frag;
template <> struct Q4Frag<__half> {
    static __device__ __forceinline__ uint32_t low(uint32_t w) {
        const uint32_t v = (w & 0x000f000fu) | 0x64006400u, o = 0x64086408u;   // 1024 + q, 1032
        const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&o));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static __device__ __forceinline__ uint32_t high(uint32_t w) {
        const uint32_t v = (w & 0x00f000f0u) | 0x64006400u, m = 0x2c002c00u, o = 0xd480d480u;   // 1024 + 16 q, 1 / 16, -72
        const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&m), *reinterpret_cast<const __half2*>(&o));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static __device__ __forceinline__ void expand(uint32_t w, uint32_t (&a)[4]) {
        a[0] = low(w);
        a[1] = high(w);
        a[2] = low(w >> 8);
        a[3] = high(w >> 8);
    }
};
template <> struct Q4Frag<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t low(uint32_t w) {
        const uint32_t v = (w & 0x000f000fu) | 0x43004300u, o = 0x43084308u;   // 128 + q, 136
        const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&o));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static __device__ __forceinline__ void expand(uint32_t w, uint32_t (&a)[4]) {
        a[0] = low(w);
        a[1] = low(w >> 4);
        a[2] = low(w >> 8);
        a[3] = low(w >> 12);
    }
};

template <class T> __device__ __forceinline__ float2 pair_f32(uint32_t w);
template <> __device__ __forceinline__ float2 pair_f32<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <> __device__ __forceinline__ float2 pair_f32<__nv_bfloat16>(uint32_t w) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}

// ---------------------------------------------------------------- quantising and reading back
// Both kernels pass tiles of 128 k x 128 n through shared memory: whole rows of W on the one side, a warp's strip of 16 n with its
// 16 bytes a lane on the other. They are bound by memory: 2 bytes a weight, and 0.5 + 2 / group.
constexpr int kTile = 128;
template <bool TRANS>
struct Q4Tile {
    // pitch in bytes, so that a strip's accesses (eight n, four k apart) meet different banks.
    // [pair of k][n]: a 32-bit word holds k and k + 1 of one n; two rows of pairs are 32 bytes apart modulo 128
    // TRANS, [n][k]: accesses of four k, rows 32 bytes apart
    static constexpr int kPitch = TRANS ? kTile * 2 + 32 : (kTile + 4) * 4;
    static constexpr int kBytes = (TRANS ? kTile : kTile / 2) * kPitch;
};

// Rows of W between global memory and the tile. Outside the matrix the tile holds zeros. Each thread moves eight pieces of eight elements:
// two at a time, of rows k and k + 1 (TRANS: n and n + 1).
template <bool TRANS, bool STORE>
__device__ __forceinline__ void tile_rows(const Q4Params& p, uint16_t* w, uint8_t* tile, int n0, int k0) {
    const int inner = TRANS ? p.K : p.N, outer = TRANS ? p.N : p.K, i0 = TRANS ? k0 : n0, o0 = TRANS ? n0 : k0;
    constexpr int kSteps = kTile / 2 * 16 / 256;
    const int pair = threadIdx.x >> 4, c = threadIdx.x & 15;      // pair of rows, piece of the row
    const int left = inner - i0 - c * 8;
    uint16_t* at = w + (o0 + 2 * pair) * p.ldw + i0 + c * 8;
    const long long next = 32 * p.ldw;
    uint4 v[kSteps][2];
    if constexpr (!STORE) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                v[s][h] = row16_load(at + s * next + h * p.ldw, o0 + 2 * pair + 32 * s + h < outer ? left : 0, static_cast<const uint16_t*>(p.w), p.w_end);
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        if constexpr (TRANS) {
            uint8_t* m = tile + (2 * pair + 32 * s) * Q4Tile<TRANS>::kPitch + c * 16;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint4* x = reinterpret_cast<uint4*>(m + h * Q4Tile<TRANS>::kPitch);
                if constexpr (!STORE) *x = v[s][h];
                else v[s][h] = *x;
            }
        } else {
            uint4* x = reinterpret_cast<uint4*>(tile + (pair + 16 * s) * Q4Tile<TRANS>::kPitch + c * 32);
            if constexpr (!STORE) {
                const uint4 a = v[s][0], b = v[s][1];
                x[0] = make_uint4(__byte_perm(a.x, b.x, 0x5410), __byte_perm(a.x, b.x, 0x7632), __byte_perm(a.y, b.y, 0x5410), __byte_perm(a.y, b.y, 0x7632));
                x[1] = make_uint4(__byte_perm(a.z, b.z, 0x5410), __byte_perm(a.z, b.z, 0x7632), __byte_perm(a.w, b.w, 0x5410), __byte_perm(a.w, b.w, 0x7632));
            } else {
                const uint4 a = x[0], b = x[1];
                v[s][0] = make_uint4(__byte_perm(a.x, a.y, 0x5410), __byte_perm(a.z, a.w, 0x5410), __byte_perm(b.x, b.y, 0x5410), __byte_perm(b.z, b.w, 0x5410));
                v[s][1] = make_uint4(__byte_perm(a.x, a.y, 0x7632), __byte_perm(a.z, a.w, 0x7632), __byte_perm(b.x, b.y, 0x7632), __byte_perm(b.z, b.w, 0x7632));
            }
        }
        if constexpr (STORE) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                row16_store(at + s * next + h * p.ldw, v[s][h], o0 + 2 * pair + 32 * s + h < outer ? left : 0);
        }
    }
}

// Four consecutive k of row n of the tile, as two packed pairs.
template <bool TRANS>
__device__ __forceinline__ uint2 tile_get(const uint8_t* tile, int n, int k) {
    if constexpr (TRANS) return *reinterpret_cast<const uint2*>(tile + n * Q4Tile<TRANS>::kPitch + k * 2);
    const uint8_t* c = tile + (k >> 1) * Q4Tile<TRANS>::kPitch + n * 4;
    return make_uint2(*reinterpret_cast<const uint32_t*>(c), *reinterpret_cast<const uint32_t*>(c + Q4Tile<TRANS>::kPitch));
}
template <bool TRANS>
__device__ __forceinline__ void tile_put(uint8_t* tile, int n, int k, uint2 v) {
    if constexpr (TRANS) {
        *reinterpret_cast<uint2*>(tile + n * Q4Tile<TRANS>::kPitch + k * 2) = v;
    } else {
        uint8_t* c = tile + (k >> 1) * Q4Tile<TRANS>::kPitch + n * 4;
        *reinterpret_cast<uint32_t*>(c) = v.x;
        *reinterpret_cast<uint32_t*>(c + Q4Tile<TRANS>::kPitch) = v.y;
    }
}

template <class T> struct Pair16;
template <> struct Pair16<__half> { using type = __half2; };
template <> struct Pair16<__nv_bfloat16> { using type = __nv_bfloat162; };
template <class T>
__device__ __forceinline__ uint32_t max_abs2(uint32_t m, uint32_t v) {   // of each 16-bit half; a NaN stays
    using P = typename Pair16<T>::type;
    const P r = __hmax2_nan(*reinterpret_cast<const P*>(&m), __habs2(*reinterpret_cast<const P*>(&v)));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// v / scale rounded to the nearest integer, ties to even, plus kNibble0, as the bits of a float: the integer is in the last bits. `inv` = 1 / scale,
// or 0 for a scale of 0. v * inv is off the quotient by less than 2^-19, and a quotient that is no tie is at
// least 2^-12 away from one: v and scale are integers a, b < 2^11 times powers of two, |v / scale - (h + 1/2)| = |2 v - (2 h + 1) scale| / (2
// scale), and the numerator is a multiple of the scale's last bit. So the product rounded to a multiple of 2^-14 (by the first sum, whose last
// bit that is) is a tie exactly where the quotient is one. A normal scale is at least (1 - 2^-8) max / 7, so the integer is within
// -7 .. 7; subnormal scales, those whose inverse leaves fp32 and those that
// are not finite take the division.
constexpr uint32_t kNibble0 = 0x4b400008u;   // 1.5 * 2^23 + 8
__device__ __forceinline__ uint32_t q4_nibble(float v, float inv) {
    return __float_as_uint(__fadd_rn(__fmaf_rn(v, inv, 768.f), 12582920.f - 768.f));
}
__device__ __noinline__ uint32_t q4_nibble_any(float v, float scale) {
    if (!(scale > 0.f) || scale == __int_as_float(0x7f800000)) return kNibble0;
    const float r = fminf(fmaxf(rintf(__fdiv_rn(v, scale)), -7.f), 7.f);   // the quotient of 16-bit values cannot round onto a tie, see above
    return __float_as_uint(__fadd_rn(r, 12582920.f));
}

template <class T, bool TRANS, int G>
__global__ void __launch_bounds__(256) q4_pack_kernel(const Q4Params p) {
    __shared__ __align__(16) uint8_t tile[Q4Tile<TRANS>::kBytes];
    const int kblocks = q4_kblocks(p.K), strips = q4_strips(p.N), groups = q4_groups(p.K, G);
    const int ntiles = (strips + 7) / 8, ktiles = (kblocks + 1) / 2;
    // tiles along W's rows run fastest
    const int x = blockIdx.x % (TRANS ? ktiles : ntiles), y = blockIdx.x / (TRANS ? ktiles : ntiles);
    const int kt = TRANS ? x : y % ktiles, nt = TRANS ? y % ntiles : x, e = y / (TRANS ? ntiles : ktiles);
    tile_rows<TRANS, false>(p, const_cast<uint16_t*>(static_cast<const uint16_t*>(p.w)) + e * p.bs_w, tile, nt * kTile, kt * kTile);
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int strip = nt * 8 + warp;
    if (strip >= strips) return;
    uint2 v[2][4][2];          // [block][word][row g, g + 8]: four k
    uint32_t top[2][2][2];     // [block][half of the block][row]: largest magnitude in either half of the word
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                uint32_t m = 0;
#pragma unroll
                for (int w = 2 * h; w < 2 * h + 2; ++w) {
                    v[b][w][r] = tile_get<TRANS>(tile, warp * 16 + g + 8 * r, b * 64 + 16 * w + 4 * t);
                    m = max_abs2<T>(max_abs2<T>(m, v[b][w][r].x), v[b][w][r].y);
                }
                m = max_abs2<T>(m, __byte_perm(m, m, 0x1032));
                m = max_abs2<T>(m, __shfl_xor_sync(0xffffffffu, m, 1));
                top[b][h][r] = max_abs2<T>(m, __shfl_xor_sync(0xffffffffu, m, 2));
            }
    uint8_t* q = p.q + ((static_cast<long long>(e) * strips + strip) * kblocks + kt * 2) * 512 + lane * 16;
    uint16_t* s = p.s + (static_cast<long long>(e) * strips + strip) * groups * 16;
    // [group of the tile's 128 k][row]. max / 7 in 16 bits: the fp32 product with 1 / 7 is off by 2^-23, and a quotient by 7 of a 16-bit number
    // is at least 1 / 14 of a last place (2^-15 relative) away from where its rounding to 16 bits would change.
    constexpr int kGroups = 128 / G;
    float inv[kGroups][2], scale[kGroups][2];
    bool any = false;   // a scale that needs the division
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        uint32_t word = 0;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            uint32_t m = G == 32 ? top[i >> 1][i & 1][r] : max_abs2<T>(top[i % 2][0][r], top[i % 2][1][r]);
            if (G == 128) m = max_abs2<T>(max_abs2<T>(m, top[1][0][r]), top[1][1][r]);
            const T sc = rounded<T>(pair_f32<T>(m).x * (1.f / 7.f));
            word |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&sc)) << (16 * r);
            const float f = to_f32(sc);
            any = any || !(f < __int_as_float(0x7f800000)) || (f > 0.f && f < (std::is_same<T, __half>::value ? 0x1p-14f : 0x1p-100f));
            inv[i][r] = f > 0.f ? __fdividef(1.f, f) : 0.f;
            scale[i][r] = f;
        }
        if (t == 0 && kt * kGroups + i < groups) *reinterpret_cast<uint32_t*>(s + (kt * kGroups + i) * 16 + g * 2) = word;
    }
    any = __any_sync(0xffffffffu, any);
    // the words: integers shifted into place and added up, with the constant part of their bits taken off
    auto words = [&](auto nibble, int b) {
        uint4 out;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint32_t word = 0;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float2 lo = pair_f32<T>(v[b][w][r].x), hi = pair_f32<T>(v[b][w][r].y);
                const float f[4] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
                for (int j = 0; j < 4; ++j) word += (nibble(f[j], G == 32 ? b * 2 + (w >> 1) : (G == 64 ? b : 0), r) - (kNibble0 & ~15u)) << (8 * j + 4 * r);
            }
            (&out.x)[w] = word;
        }
        *reinterpret_cast<uint4*>(q + b * 512) = out;
    };
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        if (kt * 2 + b >= kblocks) break;
        if (!any) words([&](float f, int i, int r) { return q4_nibble(f, inv[i][r]); }, b);
        else words([&](float f, int i, int r) { return q4_nibble_any(f, scale[i][r]); }, b);
    }
}

template <class T, bool TRANS>
__global__ void __launch_bounds__(256) q4_unpack_kernel(const Q4Params p) {
    using P = typename Pair16<T>::type;
    __shared__ __align__(16) uint8_t tile[Q4Tile<TRANS>::kBytes];
    const int kblocks = q4_kblocks(p.K), strips = q4_strips(p.N), groups = q4_groups(p.K, p.group);
    const int ntiles = (strips + 7) / 8, ktiles = (kblocks + 1) / 2;
    const int x = blockIdx.x % (TRANS ? ktiles : ntiles), y = blockIdx.x / (TRANS ? ktiles : ntiles);
    const int kt = TRANS ? x : y % ktiles, nt = TRANS ? y % ntiles : x, e = y / (TRANS ? ntiles : ktiles);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int strip = nt * 8 + warp;
    if (strip < strips) {
        const uint8_t* q = p.q + ((static_cast<long long>(e) * strips + strip) * kblocks + kt * 2) * 512 + lane * 16;
        const uint16_t* s = p.s + (static_cast<long long>(e) * strips + strip) * groups * 16 + g * 2;
        uint4 v[2];
        uint32_t sc[2][2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            if (kt * 2 + b >= kblocks) break;
            v[b] = *reinterpret_cast<const uint4*>(q + b * 512);
#pragma unroll
            for (int h = 0; h < 2; ++h) sc[b][h] = *reinterpret_cast<const uint32_t*>(s + (kt * 128 + b * 64 + h * 32) / p.group * 16);
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            if (kt * 2 + b >= kblocks) break;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t a[4];   // rows g, g + 8 with k = 0, 2 and 1, 3 of the four
                Q4Frag<T>::expand((&v[b].x)[w], a);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    // an integer of three bits times a 16-bit scale, rounded once
                    const uint32_t f = __byte_perm(sc[b][w >> 1], 0, r ? 0x3232 : 0x1010);
                    const P lo = __hmul2(*reinterpret_cast<const P*>(&a[r]), *reinterpret_cast<const P*>(&f));
                    const P hi = __hmul2(*reinterpret_cast<const P*>(&a[2 + r]), *reinterpret_cast<const P*>(&f));
                    const uint32_t l = *reinterpret_cast<const uint32_t*>(&lo), h = *reinterpret_cast<const uint32_t*>(&hi);
                    tile_put<TRANS>(tile, warp * 16 + g + 8 * r, b * 64 + 16 * w + 4 * t,
                                    make_uint2(__byte_perm(l, h, 0x5410), __byte_perm(l, h, 0x7632)));
                }
            }
        }
    }
    __syncthreads();
    tile_rows<TRANS, true>(p, static_cast<uint16_t*>(p.wout) + e * p.bs_w, tile, nt * kTile, kt * kTile);
}

// ---------------------------------------------------------------- products of a few rows
constexpr int kGemvWarps = 16;                        // that compute
constexpr int kGemvCopiers = 4;                       // more, that bring the weights: one thread of one warp took longer to issue a
                                                      // slot's copies, between the other warps' instructions, than the copies (4.0 TB/s)
constexpr int kGemvThreads = (kGemvWarps + kGemvCopiers) * 32;
constexpr int kGemvBlocks = 4;                        // blocks of 64 k that a warp computes at a time
constexpr int kGemvSlot = kGemvBlocks * (512 + 64);   // a warp's share of a slot: its blocks, and up to two groups' scales for each
constexpr int kGemvMaxShared = 227 << 10;

// Integers: sixteen k of unsigned nibbles against signed bytes of x, exact in 32 bits.
__device__ __forceinline__ void mma_16832(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <class T>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}


// Two ways to multiply, by the number of rows that share a pass over the weights.
//   INT  a few rows: the weights stay unsigned nibbles, whose offset 8 the sum of x over the group takes out, and a row of x is written
//        as 32-bit integers times one power of two, in four signed bytes; each byte is a column of m16n8k32. Two operations turn a word of weights into
//        operands, half as many instructions as with 16-bit products, and the sums of a group are exact. A row that these integers do not hold
//        exactly (gemv_wide: a spread of more than about 2^22 in bf16, or values that are not finite) stays in 16 bits instead, and its columns are
//        computed as below beside the integers of the unit's other rows (1 row x 8192 x 32768, groups of 128, f16: 27.6 us as integers, 39.6 in 16 bits).
//   else x stays in 16 bits, one column of m16n8k16 a row, with the nibbles as 16-bit numbers (Q4Frag).
template <int NT, bool INT>
struct GemvShape {
    static constexpr int kCols = 8 * NT;
    static constexpr int kPerRow = INT ? 4 : 1;                 // columns of a row
    static constexpr int kRows = kCols / kPerRow;               // rows of a pass
    static constexpr int kBlockBytes = INT ? 64 : 128;          // of a column, for 64 k
    static constexpr int kFlush = INT ? 4 : 1;                  // strips whose partial sums meet at a time
    static constexpr int kPartPitch = INT ? kRows : kCols + 1;  // floats of an n of them
};

// Shared memory of q4_gemv_kernel. A staged column of x holds, for each block of 64 k and each t = 0 .. 3, the bytes that lanes 4 g + t
// of the B fragments take: one 16-byte load (INT; pitch 64 modulo 128) or two (pitch 16 modulo 128), where eight
// lanes of a load (two columns, four t) meet every bank once.
template <int NT, bool INT>
struct GemvLayout {
    int pitch, xi, part, ring, bars, rows, units, idx, bytes;   // byte offsets
    __host__ __device__ GemvLayout(int kblocks, int groups, int unit_rows, int depth, int R, bool indexed) {
        using S = GemvShape<NT, INT>;
        pitch = INT ? (kblocks | 1) * 64 : kblocks * 128 + 16;
        xi = (unit_rows * S::kPerRow * pitch + 15) & ~15;
        part = (xi + (INT ? groups * S::kCols * 4 : 0) + 15) & ~15;
        ring = (part + 2 * S::kFlush * kGemvWarps * 16 * S::kPartPitch * 4 + 127) & ~127;
        bars = ring + kGemvWarps * depth * kGemvSlot;
        rows = bars + kGemvWarps * depth * 16;
        units = rows + 2 * S::kCols * 4 + 16;
        idx = units + (indexed ? R * 4 : 0);
        bytes = idx + (indexed ? R * 4 : 0);
    }
};

// What an integer sum of a group starts from, beside -8 times the sum of x's bytes: as the bits of a float this is 1.5 * 2^23, and an integer
// within 2^22 added to the bits is one added to the number, so one multiply-add turns the sum into a float of x's own size (sums in x's integers,
// scaled back at the end, would leave fp32's range 2^31 before the results do).
constexpr int kGemvZero = 0x4b400000;
__device__ __forceinline__ float gemv_power(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }   // 2^e, of a normal number

// The exponent of the largest power of two that keeps a row whose largest magnitude has the bits `top` (finite) within four signed bytes, at most
// 127 * 16843009 in magnitude: of the 16-bit types' numbers those below 1.9921875 * 2^30. Subnormal numbers are taken for 2^-126, where nothing of a
// 16-bit type needs more.
__device__ __forceinline__ int gemv_exponent(uint32_t top) {
    return 30 - max(static_cast<int>(top >> 23) - 127, -126) - ((top & 0x7fffffu) >= 0x7f0000u ? 1 : 0);
}
// 2 to that exponent as two factors: the power itself may leave fp32's range.
__device__ __forceinline__ void gemv_scale(uint32_t top, float& f1, float& f2) {
    const int up = gemv_exponent(top), up1 = up >> 1;
    f1 = __uint_as_float(static_cast<uint32_t>(up1 + 127) << 23);
    f2 = __uint_as_float(static_cast<uint32_t>(up - up1 + 127) << 23);
}
// The exponent of what a row's integers count on the way to the result, which is scaled by the rest: so that what a sum starts from stays in fp32's range.
__device__ __forceinline__ int gemv_unit(uint32_t top) { return max(-100, min(-gemv_exponent(top), 86)); }
// Whether a row holds a value that is no integer times that power, or that is not finite. `low`: the smallest magnitude of the row that is not 0, as the
// type's bits less one (0xffff: there is none). A value's last bit counts 2^(its exponent - mantissa bits), and less only in smaller values.
template <class T>
__device__ __forceinline__ bool gemv_wide(uint32_t top, uint32_t low) {
    constexpr int kBits = std::is_same<T, __half>::value ? 10 : 7, kBias = std::is_same<T, __half>::value ? 15 : 127;
    if (top >= 0x7f800000u) return true;
    const int last = max(static_cast<int>((low + 1) >> kBits), 1) - kBias - kBits;
    return low < 0xffffu && last + gemv_exponent(top) < 0;
}

// `nb` blocks of a slot from block kb0 of the strip on, for rows that stay in 16 bits: row g of the unit is column g of the instruction.
template <class T, int G>
__device__ __forceinline__ void gemv_wide_slot(float (&acc)[4], const uint8_t* x, const uint8_t* blocks, const uint8_t* scales, int kb0, int nb) {
    float c[4];
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < kGemvBlocks; ++u) {
        if (u >= nb) break;
        const uint4 q = *reinterpret_cast<const uint4*>(blocks + u * 512);
        const uint4 b[2] = {*reinterpret_cast<const uint4*>(x + (kb0 + u) * 128), *reinterpret_cast<const uint4*>(x + (kb0 + u) * 128 + 16)};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            uint32_t a[4];
            Q4Frag<T>::expand((&q.x)[s], a);
            const uint32_t b0 = (&b[s >> 1].x)[2 * (s & 1)], b1 = (&b[s >> 1].x)[2 * (s & 1) + 1];
            if ((s == 0 && (G != 128 || u % 2 == 0)) || (G == 32 && s == 2)) mma_16816<T>(c, a, b0, b1, zero);
            else mma_16816<T>(c, a, b0, b1, c);
            if ((s == 3 && (G != 128 || u % 2 == 1 || u + 1 == nb)) || (G == 32 && s == 1)) {
                const float2 f = pair_f32<T>(*reinterpret_cast<const uint32_t*>(scales + (G == 32 ? u * 2 + (s >> 1) : (G == 64 ? u : u >> 1)) * 32));
                acc[0] += f.x * c[0];
                acc[1] += f.x * c[1];
                acc[2] += f.y * c[2];
                acc[3] += f.y * c[3];
            }
        }
    }
}

// Y[r] = X[r / per] x W[index[r]]. Work items are (unit, strip of 16 n), where a unit is up to `unit_rows` rows that name one matrix:
// a matrix is read once for all of them. Every CTA takes an equal run of consecutive items, stages a unit's rows of x in shared memory once, with
// the sums of x over each group of k, and lets groups of `gs` warps compute a strip each. Other warps
// bring packed weights and scales with bulk copies, gs * kGemvBlocks blocks of a strip at a time into a ring of `depth` slots for each
// group, and run ahead over strip and unit ends. A computing warp turns 16 bytes a lane into A fragments, sums a group of k in the
// instruction's accumulators, and adds the scaled sum in fp32. The gs partial sums of a strip meet in shared memory in a fixed order.
template <class T, int NT, int G, bool INT>
__global__ void __launch_bounds__(kGemvThreads, 1) q4_gemv_kernel(const Q4Params p, int gs, int unit_rows, int depth) {
    using S = GemvShape<NT, INT>;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    constexpr int kCols = S::kCols;
    const int kblocks = q4_kblocks(p.K), strips = q4_strips(p.N), groups = q4_groups(p.K, G);
    const GemvLayout<NT, INT> lay(kblocks, groups, unit_rows, depth, p.R, p.index != nullptr);
    int* xi = reinterpret_cast<int*>(smem_raw + lay.xi);        // INT, [group][column]: see kGemvZero
    float* part = reinterpret_cast<float*>(smem_raw + lay.part);
    int* rows = reinterpret_cast<int*>(smem_raw + lay.rows);
    int* units = reinterpret_cast<int*>(smem_raw + lay.units);
    int* idx = reinterpret_cast<int*>(smem_raw + lay.idx);
    uint32_t* top = reinterpret_cast<uint32_t*>(rows + kCols);  // INT: the largest magnitude of each row, as the bits of a float, ...
    uint32_t* low = top + S::kRows;                             // ... then the smallest that is not 0, as the type's bits less one
    int* count_slot = rows + 2 * kCols;                         // two words, then the CTA's abort flag
    uint32_t* abort_slot = reinterpret_cast<uint32_t*>(count_slot + 2);
    const AbortCtx ab{abort_slot, p.status, p.wait_cycles > 0 ? p.wait_cycles : kWaitTimeoutCycles};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = warp / gs, wig = warp % gs, num_groups = kGemvWarps / gs;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem_raw + lay.bars);   // [group][depth] filled, then [group][depth] free
    const int slot_bytes = gs * kGemvSlot;
    if (threadIdx.x == 0) {
        for (int i = 0; i < num_groups * depth; ++i) {
            ptx::mbar_init(&bars[i], 1);
            ptx::mbar_init(&bars[num_groups * depth + i], gs);
        }
        ptx::fence_mbar_init();
        *abort_slot = 0u;
    }
    ptx::grid_dep_launch();
    ptx::grid_dep_wait();

    // units: the rows whose number among the rows of their matrix is a multiple of unit_rows start one
    int num_units;
    if (p.index) {
        for (int r = threadIdx.x; r < p.R; r += blockDim.x) idx[r] = p.index[r];
        __syncthreads();
        for (int r = threadIdx.x; r < p.R; r += blockDim.x) {
            const int e = idx[r];
            int before = 0;
            for (int i = 0; i < r; ++i) before += idx[i] == e;
            units[r] = e >= 0 && e < p.E && before % unit_rows == 0;
            if (e >= p.E && blockIdx.x == 0) atomicOr(p.status, ST_BAD_INDEX);
        }
        __syncthreads();
        if (warp == 0) {   // the marks become the list of rows, in place: its end never passes the marks still to be read
            int n = 0;
            for (int r0 = 0; r0 < p.R; r0 += 32) {
                const unsigned starts = __ballot_sync(0xffffffffu, r0 + lane < p.R && units[r0 + lane]);
                if (starts >> lane & 1) units[n + __popc(starts & ((1u << lane) - 1))] = r0 + lane;
                n += __popc(starts);
                __syncwarp();
            }
            if (lane == 0) count_slot[1] = n;   // a word of its own: the other one is written again while the copying warps read this
        }
        __syncthreads();
        num_units = count_slot[1];
    } else {
        num_units = (p.R + unit_rows - 1) / unit_rows;
        __syncthreads();
    }

    const long long items = static_cast<long long>(num_units) * strips;
    long long item = items * blockIdx.x / gridDim.x;
    const long long item_end = items * (blockIdx.x + 1) / gridDim.x;
    const int chunk = gs * kGemvBlocks;                         // blocks of a slot
    const int chunks = (kblocks + chunk - 1) / chunk;           // slots of a strip

    if (warp >= kGemvWarps) {
        // ------------------------------------------------------------ copying warps: each takes every `share`-th slot of one group
        if (!ptx::elect_one()) return;
        // a slot stays with one of them (`share` divides `depth`): a wait on the parity of its barrier must not miss a phase
        const int gr = (warp - kGemvWarps) % num_groups, mine = (warp - kGemvWarps) / num_groups;
        int share = kGemvCopiers / num_groups;
        while (depth % share) --share;
        if (mine >= share) return;
        uint64_t* full = bars + gr * depth;
        uint64_t* freed = full + num_groups * depth;
        uint8_t* ring = smem_raw + lay.ring + gr * depth * slot_bytes;
        const int q_full = chunk * 512, q_last = (kblocks - (chunks - 1) * chunk) * 512;
        const int s_full = chunk * 64 / G * 32, s_last = groups * 32 - (chunks - 1) * s_full;
        int turn = 0, slot = 0;          // slots of the group so far, modulo `share` and `depth`
        uint32_t phase = 1;              // the first round finds every slot free
        int left_out = p.skip_stage;
        bool ok = true;
        while (ok && item < item_end) {
            const int unit = static_cast<int>(item / strips);
            const int s_begin = static_cast<int>(item % strips);
            const int s_end = static_cast<int>(min(static_cast<long long>(strips), s_begin + (item_end - item)));
            item += s_end - s_begin;
            const int e = p.index ? idx[units[unit]] : 0;
            for (int strip = s_begin + gr; ok && strip < s_end; strip += num_groups) {
                const long long at = static_cast<long long>(e) * strips + strip;
                const uint8_t* q = p.q + at * kblocks * 512;
                const uint8_t* s = reinterpret_cast<const uint8_t*>(p.s) + at * groups * 32;
                for (int c = 1; c <= chunks; ++c, q += q_full, s += s_full) {
                    // once a role has given up nothing more is brought: the slots may still be read
                    if (turn == mine && !(ok = bounded_wait(&freed[slot], phase, ab, ST_TIMEOUT_PRODUCER) && *ab.flag == 0u)) break;
                    if (--left_out != 0 && turn == mine) {
                        const int qb = c == chunks ? q_last : q_full, sb = c == chunks ? s_last : s_full;
                        uint8_t* dst = ring + slot * slot_bytes;
                        ptx::mbar_expect_tx(&full[slot], qb + sb);
                        ptx::bulk_load(dst, q, qb, &full[slot]);
                        ptx::bulk_load(dst + q_full, s, sb, &full[slot]);
                    }
                    if (++turn == share) turn = 0;
                    if (++slot == depth) { slot = 0; phase ^= 1u; }
                }
            }
        }
        if (*ab.flag) __nanosleep(200000);   // for the copies on their way: the block's memory is given back when its last thread ends
        return;
    }

    // ---------------------------------------------------------------- computing warps
    const uint8_t* ring = smem_raw + lay.ring + group * depth * slot_bytes;
    uint64_t* full = bars + group * depth;
    uint64_t* freed = full + num_groups * depth;
    int flip = 0, held = 0;
    bool live = true;        // false once a wait has run out: it is reported, and the others test once only (the call's results are lost)
    int c_slot = 0;          // next slot to read
    uint32_t c_phase = 0;

    while (item < item_end) {
        const int unit = static_cast<int>(item / strips);
        const int s_begin = static_cast<int>(item % strips);
        const int s_end = static_cast<int>(min(static_cast<long long>(strips), s_begin + (item_end - item)));
        item += s_end - s_begin;
        const int lead = p.index ? units[unit] : unit * unit_rows;
        const int e = p.index ? idx[lead] : 0;

        // the rows of the unit, their x and its sums
        ptx::bar_sync(15, kGemvWarps * 32);   // the previous unit's x and rows have been read
        if (warp == 0) {
            int found = 0;
            if (p.index) {
                for (int r0 = lead; r0 < p.R && found < unit_rows; r0 += 32) {
                    const int r = r0 + lane;
                    const unsigned hit = __ballot_sync(0xffffffffu, r < p.R && idx[r] == e);
                    const int slot = found + __popc(hit & ((1u << lane) - 1));
                    if ((hit >> lane & 1) && slot < unit_rows) rows[slot] = r;
                    found = min(unit_rows, found + __popc(hit));
                }
            } else {
                found = min(unit_rows, p.R - lead);
                for (int i = lane; i < found; i += 32) rows[i] = lead + i;
            }
            if (lane == 0) *count_slot = found;
            if (lane < kCols) top[lane] = lane < S::kRows ? 0u : 0xffffu;
        }
        ptx::bar_sync(15, kGemvWarps * 32);
        const int count = *count_slot;
        // x in pieces of 8 k, a warp's 32 pieces of one row at a time; the first ones stay in registers between the two looks at them
        const int pieces = kblocks * 8, runs = max(1, (pieces + 31) / 32), total = count * runs;   // of no k: one run without pieces
        constexpr int kLanes = G / 8;                                   // lanes that hold a group
        constexpr int kKeep = INT ? 4 : 8;
        auto piece = [&](int i) -> uint4 {
            const int row = i / runs, k8 = (i - row * runs) * 32 + lane;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (i < total && k8 < pieces) {
                const long long k = k8 * 8ll;
                const uint16_t* src = static_cast<const uint16_t*>(p.x) + (rows[row] / p.per) * p.ldx + k;
                v = row16_load(src, static_cast<int>(min(8ll, p.K - k)), static_cast<const uint16_t*>(p.x), p.x_end);
            }
            return v;
        };
        uint4 kept[kKeep];
#pragma unroll
        for (int n = 0; n < kKeep; ++n) kept[n] = piece(warp + n * kGemvWarps);
        // the others, as many at a time: the loads of a batch are on their way together
        auto rest = [&](auto f) {
            for (int i = warp + kKeep * kGemvWarps; i < total; i += kKeep * kGemvWarps) {
                uint4 v[kKeep];
#pragma unroll
                for (int n = 0; n < kKeep; ++n) v[n] = piece(i + n * kGemvWarps);
#pragma unroll
                for (int n = 0; n < kKeep; ++n)
                    if (i + n * kGemvWarps < total) f(i + n * kGemvWarps, v[n]);
            }
        };
        if constexpr (INT) {
            auto look = [&](int i, const uint4& v) {
                uint32_t m = max_abs2<T>(max_abs2<T>(max_abs2<T>(max_abs2<T>(0u, v.x), v.y), v.z), v.w);
                const float2 f = pair_f32<T>(max_abs2<T>(m, __byte_perm(m, m, 0x1032)));
                const uint32_t b = __reduce_max_sync(0xffffffffu, __float_as_uint(f.x) & 0x7fffffffu);   // a NaN's bits are above infinity's
                uint32_t l = 0xffffffffu;   // of each half the magnitude less one, of a zero 0xffff
#pragma unroll
                for (int j = 0; j < 4; ++j) l = __vminu2(l, (((&v.x)[j] & 0x7fff7fffu) + 0x7fff7fffu) ^ 0x80008000u);
                l = __reduce_min_sync(0xffffffffu, min(l & 0xffffu, l >> 16));
                if (lane == 0) {
                    atomicMax(&top[i / runs], b);
                    atomicMin(&low[i / runs], l);
                }
            };
#pragma unroll
            for (int n = 0; n < kKeep; ++n)
                if (warp + n * kGemvWarps < total) look(warp + n * kGemvWarps, kept[n]);
            rest(look);
            ptx::bar_sync(15, kGemvWarps * 32);
        }
        uint32_t wide = 0;   // INT: rows that stay in 16 bits
        if constexpr (INT)
#pragma unroll
            for (int r = 0; r < S::kRows; ++r) wide |= static_cast<uint32_t>(gemv_wide<T>(top[r], low[r])) << r;   // not of a row that is not there
        auto halves = [&](uint8_t* column, int k8, const uint4& v) {   // in the order j = 0, 2, 1, 3 of the weights' pairs
            uint8_t* dst = column + (k8 >> 3) * 128 + (k8 & 1) * 64 + ((k8 >> 1) & 3) * 8;
            *reinterpret_cast<uint2*>(dst) = make_uint2(__byte_perm(v.x, v.y, 0x5410), __byte_perm(v.x, v.y, 0x7632));
            *reinterpret_cast<uint2*>(dst + 32) = make_uint2(__byte_perm(v.z, v.w, 0x5410), __byte_perm(v.z, v.w, 0x7632));
        };
        auto place = [&](int i, const uint4& v) {
            const int row = i / runs, k8 = (i - row * runs) * 32 + lane;
            const bool real = k8 < pieces;
            // k = 16 w + 4 t + j of block k8 / 8: w = (k8 % 8) / 2, t = 2 (k8 % 2) and the next
            if constexpr (INT) {
                if (wide >> row & 1) {   // in the place of its four columns of bytes
                    if (real) halves(smem_raw + row * 4 * lay.pitch, k8, v);
                    return;
                }
                float f1, f2;
                gemv_scale(top[row], f1, f2);
                const float2 a = pair_f32<T>(v.x), b = pair_f32<T>(v.y), c = pair_f32<T>(v.z), d = pair_f32<T>(v.w);
                const float f[8] = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
                // x + 0x80808080 as an unsigned number: its bytes less 128 are the signed bytes
                uint32_t u[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) u[j] = static_cast<uint32_t>(__float2int_rn(f[j] * f1 * f2)) + 0x80808080u;
                int sums[4];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const uint32_t sel = n | ((4 + n) << 4);
                    uint32_t digits[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        digits[h] = __byte_perm(__byte_perm(u[4 * h], u[4 * h + 1], sel), __byte_perm(u[4 * h + 2], u[4 * h + 3], sel), 0x5410) ^ 0x80808080u;
                    sums[n] = __dp4a(static_cast<int>(digits[0]), 0x01010101, __dp4a(static_cast<int>(digits[1]), 0x01010101, 0));
                    if (real) {
                        uint8_t* dst = smem_raw + (row * 4 + n) * lay.pitch + (k8 >> 3) * 64 + (k8 & 1) * 32 + ((k8 >> 1) & 3) * 4;
                        *reinterpret_cast<uint32_t*>(dst) = digits[0];
                        *reinterpret_cast<uint32_t*>(dst + 16) = digits[1];
                    }
                }
                // two sums to a word on the way over the group's lanes: each stays within 2^14
                int lo = sums[0] + sums[1] * 65536, hi = sums[2] + sums[3] * 65536;
#pragma unroll
                for (int m = 1; m < kLanes; m <<= 1) {
                    lo += __shfl_xor_sync(0xffffffffu, lo, m);
                    hi += __shfl_xor_sync(0xffffffffu, hi, m);
                }
                if (real && k8 % kLanes == 0) {
                    const int s0 = static_cast<int16_t>(lo & 0xffff), s2 = static_cast<int16_t>(hi & 0xffff);
                    *reinterpret_cast<int4*>(xi + (k8 / kLanes) * kCols + row * 4) =
                        make_int4(kGemvZero - 8 * s0, kGemvZero - 8 * ((lo - s0) >> 16), kGemvZero - 8 * s2, kGemvZero - 8 * ((hi - s2) >> 16));
                }
            } else if (real) {
                halves(smem_raw + row * lay.pitch, k8, v);
            }
        };
#pragma unroll
        for (int n = 0; n < kKeep; ++n)
            if (warp + n * kGemvWarps < total) place(warp + n * kGemvWarps, kept[n]);
        rest(place);
        ptx::bar_sync(15, kGemvWarps * 32);

        // lanes of columns without a row read column 0 of x: what they compute is in columns that are not stored
        const uint8_t* xlane[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n)
            xlane[n] = smem_raw + (n * 8 + g < count * S::kPerRow ? n * 8 + g : 0) * lay.pitch + t * (S::kBlockBytes / 4);
        // INT, of the row whose columns 2 t and 2 t + 1 are: what the lower one's byte counts, and that times what the sums start from
        float unit_of[NT], zero_of[NT];
        if constexpr (INT)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                unit_of[n] = gemv_power(gemv_unit(top[n * 2 + (t >> 1)]) + 16 * (t & 1));
                zero_of[n] = -__int_as_float(kGemvZero) * unit_of[n];
            }
        float acc[NT][4];
        // the warp's blocks of one slot, kGemvBlocks of them or `nb` at the strip's end
        auto compute = [&](auto full_slot, const uint8_t* blocks, const uint8_t* scales, int kb0, int nb) {
            float c[NT][4] = {};
            int ci[NT][4] = {};
            const int at0 = kb0 * 64 / G * kCols + 2 * t;
#pragma unroll
            for (int u = 0; u < kGemvBlocks; ++u) {
                if (!full_slot.value && u >= nb) break;
                const uint4 q = *reinterpret_cast<const uint4*>(blocks + u * 512);
                uint4 b[NT][INT ? 1 : 2];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int h = 0; h < (INT ? 1 : 2); ++h)
                        b[n][h] = *reinterpret_cast<const uint4*>(xlane[n] + (kb0 + u) * S::kBlockBytes + h * 16);
                const float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < 4; ++s) {   // 16 k each
                    const bool begins = (s == 0 && (G != 128 || u % 2 == 0)) || (G == 32 && s == 2);
                    const bool ends = (s == 3 && (G != 128 || u % 2 == 1 || (!full_slot.value && u + 1 == nb))) || (G == 32 && s == 1);
                    const int in_slot = G == 32 ? u * 2 + (s >> 1) : (G == 64 ? u : u >> 1);
                    if constexpr (INT) {
                        if (begins)
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const int2 o = *reinterpret_cast<const int2*>(xi + at0 + in_slot * kCols + n * 8);
                                ci[n][0] = ci[n][2] = o.x;
                                ci[n][1] = ci[n][3] = o.y;
                            }
                        if (s % 2 == 0) {
                            const uint32_t w0 = (&q.x)[s], w1 = (&q.x)[s + 1];
                            const uint32_t a[4] = {w0 & 0x0f0f0f0fu, (w0 >> 4) & 0x0f0f0f0fu, w1 & 0x0f0f0f0fu, (w1 >> 4) & 0x0f0f0f0fu};
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma_16832(ci[n], a, (&b[n][0].x)[s], (&b[n][0].x)[s + 1]);
                        }
                    } else {
                        uint32_t a[4];
                        Q4Frag<T>::expand((&q.x)[s], a);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const uint32_t b0 = (&b[n][s >> 1].x)[2 * (s & 1)], b1 = (&b[n][s >> 1].x)[2 * (s & 1) + 1];
                            if (begins) mma_16816<T>(c[n], a, b0, b1, zero);
                            else mma_16816<T>(c[n], a, b0, b1, c[n]);
                        }
                    }
                    if (ends) {
                        const float2 f = pair_f32<T>(*reinterpret_cast<const uint32_t*>(scales + in_slot * 32));
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if constexpr (INT) {
                                acc[n][0] += f.x * __fmaf_rn(__int_as_float(ci[n][0]), unit_of[n], zero_of[n]);
                                acc[n][1] += f.x * __fmaf_rn(__int_as_float(ci[n][1]), unit_of[n], zero_of[n]);
                                acc[n][2] += f.y * __fmaf_rn(__int_as_float(ci[n][2]), unit_of[n], zero_of[n]);
                                acc[n][3] += f.y * __fmaf_rn(__int_as_float(ci[n][3]), unit_of[n], zero_of[n]);
                            } else {
                                acc[n][0] += f.x * c[n][0];
                                acc[n][1] += f.x * c[n][1];
                                acc[n][2] += f.y * c[n][2];
                                acc[n][3] += f.y * c[n][3];
                            }
                        }
                    }
                }
            }
        };
        // the unit's strips; `mixed`: some of its rows stay in 16 bits (a loop of its own: tests and a call in the other one cost it 1 to 4 %)
        auto strips_of_unit = [&](auto mixed) {
            for (int strip = s_begin + group; strip < s_end; strip += num_groups) {
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
                float wide_acc[4];   // of rows 2 t and 2 t + 1
                if constexpr (mixed.value) wide_acc[0] = wide_acc[1] = wide_acc[2] = wide_acc[3] = 0.f;
                for (int kb0 = wig * kGemvBlocks; kb0 < chunks * chunk; kb0 += chunk) {
                    if (!ptx::mbar_try_wait(&full[c_slot], c_phase) && live) live = bounded_wait(&full[c_slot], c_phase, ab, ST_TIMEOUT_MMA);
                    __syncwarp();
                    const uint8_t* slot = ring + c_slot * slot_bytes;
                    const uint8_t* blocks = slot + wig * (kGemvBlocks * 512) + lane * 16;
                    const uint8_t* scales = slot + chunk * 512 + wig * (kGemvBlocks * 64 / G * 32) + g * 4;
                    const bool any = !mixed.value || wide != (1u << count) - 1u;   // a row of integers
                    if (any && kb0 + kGemvBlocks <= kblocks) compute(std::true_type(), blocks, scales, kb0, kGemvBlocks);
                    else if (any && kb0 < kblocks) compute(std::false_type(), blocks, scales, kb0, kblocks - kb0);
                    if constexpr (mixed.value)
                        if (kb0 < kblocks)
                            gemv_wide_slot<T, G>(wide_acc, smem_raw + (g < count ? g : 0) * 4 * lay.pitch + t * 32, blocks, scales, kb0, min(kGemvBlocks, kblocks - kb0));
                    __syncwarp();   // every lane has read the slot
                    if (lane == 0) ptx::mbar_arrive(&freed[c_slot]);
                    if (++c_slot == depth) { c_slot = 0; c_phase ^= 1u; }
                }
                float* mine = part + ((flip * S::kFlush + held) * kGemvWarps + warp) * 16 * S::kPartPitch;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if constexpr (INT) {
                        // bytes 0, 1 of a row in the lanes with even t, bytes 2, 3 in the next lanes
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float v = acc[n][2 * h] + 256.f * acc[n][2 * h + 1];
                            const float v2 = __shfl_xor_sync(0xffffffffu, v, 1);
                            if (t % 2 == 0 && !(mixed.value && (wide >> (n * 2 + (t >> 1)) & 1))) mine[(g + 8 * h) * S::kPartPitch + n * 2 + (t >> 1)] = v + v2;
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) mine[(g + (j >> 1) * 8) * S::kPartPitch + n * 8 + 2 * t + (j & 1)] = acc[n][j];
                    }
                }
                if constexpr (mixed.value)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (wide >> (2 * t + (j & 1)) & 1) mine[(g + 8 * (j >> 1)) * S::kPartPitch + 2 * t + (j & 1)] = wide_acc[j];
                if (++held < S::kFlush && strip + num_groups < s_end) continue;
                ptx::bar_sync(1 + group, gs * 32);
                // two buffers in turn: this one is written again only after the barrier of the next flush
                for (int i = wig * 32 + lane; i < held * 16 * count; i += gs * 32) {
                    const int n = i & 15, col = (i >> 4) % count, f = (i >> 4) / count;
                    const float* from = part + ((flip * S::kFlush + f) * kGemvWarps + group * gs) * 16 * S::kPartPitch + n * S::kPartPitch + col;
                    float v = 0.f;
#pragma unroll 4
                    for (int w = 0; w < gs; ++w) v += from[w * 16 * S::kPartPitch];
                    if constexpr (INT)
                        if (!(mixed.value && (wide >> col & 1))) v *= gemv_power(-gemv_exponent(top[col]) - gemv_unit(top[col]));
                    const int n_at = (strip - (held - 1 - f) * num_groups) * 16 + n;
                    if (n_at < p.N) {
                        const long long at = rows[col] * p.ldy + n_at;
                        if (p.out_f32) static_cast<float*>(p.y)[at] = v;
                        else static_cast<T*>(p.y)[at] = rounded<T>(v);
                    }
                }
                flip ^= 1;
                held = 0;
            }
        };
        if constexpr (INT) {
            if (wide) strips_of_unit(std::true_type());
            else strips_of_unit(std::false_type());
        } else {
            strips_of_unit(std::false_type());
        }
    }
    if (*ab.flag) __nanosleep(200000);   // as the copying lanes do
}

// How a call is cut: rows of x that a CTA stages at a time (as many as the instruction's columns and shared memory take; 0 when
// not one fits) and slots of the warps' rings.
struct GemvPlan {
    int unit_rows, depth, bytes;
};
template <int NT, bool INT>
GemvPlan gemv_plan(int K, int group, int R, bool indexed) {
    constexpr int most = GemvShape<NT, INT>::kRows;
    GemvPlan plan = {R < most ? R : most, 0, 0};
    for (; plan.unit_rows > 0; --plan.unit_rows)
        for (plan.depth = 4; plan.depth >= 2; --plan.depth) {
            plan.bytes = GemvLayout<NT, INT>(q4_kblocks(K), q4_groups(K, group), plan.unit_rows, plan.depth, R, indexed).bytes;
            if (plan.bytes <= kGemvMaxShared) return plan;
        }
    return plan;
}

template <class T, int NT, int G, bool INT>
cudaError_t gemv_launch(const Q4Params& p, cudaStream_t stream) {
    auto kern = q4_gemv_kernel<T, NT, G, INT>;
    static std::atomic<bool> configured[kMaxDev];
    if (cudaError_t e = allow_smem(kern, kGemvMaxShared, configured)) return e;
    const GemvPlan plan = gemv_plan<NT, INT>(p.K, G, p.R, p.index != nullptr);
    if (plan.unit_rows <= 0) return cudaErrorInvalidValue;   // the entry point has checked q4_gemv_fits
    const int sms = core_sm_count(), kblocks = q4_kblocks(p.K);
    const long long matrices = p.index && p.E > 0 ? (p.R < p.E ? p.R : p.E) : 1, share = (p.R + matrices - 1) / matrices;
    const long long units = matrices * ((share + plan.unit_rows - 1) / plan.unit_rows);   // as if the rows were spread evenly
    const long long items = units * q4_strips(p.N);
    const int grid = static_cast<int>(items < 1 ? 1 : (items < sms ? items : sms));
    // Warps to a strip: the number that needs the fewest slot times, where the groups of a CTA share its strips and a strip's end costs about
    // half a slot (8192 x 32768, 14 strips a CTA: 4 groups take 4 strips one after another, 2 groups 7 of half the length).
    const long long per_cta = (items + grid - 1) / grid;
    int gs = 16;
    long long best = 0;
    for (int n = 16; n >= 4; n /= 2) {
        const long long cost = (per_cta * n + 15) / 16 * (2 * ((kblocks + n * kGemvBlocks - 1) / (n * kGemvBlocks)) + 1);
        if (n == 16 || cost < best) { best = cost; gs = n; }
    }
    return launch_behind(kern, grid, kGemvThreads, plan.bytes, stream, p, gs, plan.unit_rows, plan.depth);
}

template <class T, int NT, bool INT>
cudaError_t gemv_group(const Q4Params& p, cudaStream_t stream) {
    if (p.group == 32) return gemv_launch<T, NT, 32, INT>(p, stream);
    return p.group == 64 ? gemv_launch<T, NT, 64, INT>(p, stream) : gemv_launch<T, NT, 128, INT>(p, stream);
}

template <class T>
cudaError_t gemv_typed(const Q4Params& p, cudaStream_t stream) {
    const bool indexed = p.index != nullptr;
    // rows that may be expected to share a matrix: with an index the mean over the matrices
    const int rows = indexed && p.E > 0 ? (p.R + p.E - 1) / p.E : p.R;
    if (rows <= 2 && gemv_plan<1, true>(p.K, p.group, p.R, indexed).unit_rows >= rows) return gemv_group<T, 1, true>(p, stream);
    if (rows <= 4 && gemv_plan<2, true>(p.K, p.group, p.R, indexed).unit_rows >= rows) return gemv_group<T, 2, true>(p, stream);
    // 16 rows at a time where all of them fit: 13 and 3 take longer than 8 and 8 (16 rows x 4096 x 32768: 52 us against 40)
    const bool two = rows > 8 && gemv_plan<2, false>(p.K, p.group, p.R, indexed).unit_rows >= (rows < 16 ? rows : 16);
    return two ? gemv_group<T, 2, false>(p, stream) : gemv_group<T, 1, false>(p, stream);
}

unsigned tiles_for(const Q4Params& p) {
    return static_cast<unsigned>(static_cast<long long>((q4_strips(p.N) + 7) / 8) * ((q4_kblocks(p.K) + 1) / 2) * p.E);
}

template <class T, bool TRANS>
cudaError_t pack_group(const Q4Params& p, cudaStream_t stream) {
    const unsigned grid = tiles_for(p);
    if (p.group == 32) q4_pack_kernel<T, TRANS, 32><<<grid, 256, 0, stream>>>(p);
    else if (p.group == 64) q4_pack_kernel<T, TRANS, 64><<<grid, 256, 0, stream>>>(p);
    else q4_pack_kernel<T, TRANS, 128><<<grid, 256, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t q4_pack_launch(const Q4Params& p, cudaStream_t stream) {
    if (p.bf16) return p.trans_b ? pack_group<__nv_bfloat16, true>(p, stream) : pack_group<__nv_bfloat16, false>(p, stream);
    return p.trans_b ? pack_group<__half, true>(p, stream) : pack_group<__half, false>(p, stream);
}

cudaError_t q4_unpack_launch(const Q4Params& p, cudaStream_t stream) {
    const unsigned grid = tiles_for(p);
    if (p.bf16) {
        if (p.trans_b) q4_unpack_kernel<__nv_bfloat16, true><<<grid, 256, 0, stream>>>(p);
        else q4_unpack_kernel<__nv_bfloat16, false><<<grid, 256, 0, stream>>>(p);
    } else {
        if (p.trans_b) q4_unpack_kernel<__half, true><<<grid, 256, 0, stream>>>(p);
        else q4_unpack_kernel<__half, false><<<grid, 256, 0, stream>>>(p);
    }
    return cudaGetLastError();
}

bool q4_gemv_fits(int K, int group, int R, bool indexed) { return gemv_plan<1, false>(K, group, R, indexed).unit_rows > 0; }

cudaError_t q4_gemv_launch(const Q4Params& p, cudaStream_t stream) {
    return p.bf16 ? gemv_typed<__nv_bfloat16>(p, stream) : gemv_typed<__half>(p, stream);
}

}  // namespace t2sp
