// Grouped products on the tensor cores. The operands are exchanged against the other GEMM kernels: the 256 rows of an
// MMA are columns n of the output and the MMA's columns are rows t of the group (forward) or indices k (gradient of B), so
// that a group's ragged end costs an MMA of fewer columns (any multiple of 16, of a pair 32) instead of rows computed in vain, and a
// weight tile that meets a handful of rows is still fetched at full width.
//
//   forward   D[n][t] = sum_k B[e][k][n] A[t][k]       tiles of up to 256 n x up to 256 rows of one group
//   gradient  D[n][k] = sum_t D[t][n] A[t][k]          tiles of up to 256 n x up to 256 k of one group's matrix; the contraction
//                                                      runs over the group's rows, whose last block is ragged
//
// The group boundaries are read here, on the device: every CTA loads the offsets, checks them and builds the table of
// first tiles in its prologue. Roles per CTA as in umma_pair.cuh (warp 0 producer, 1 MMA, 2-9 epilogue); the gradient has one more
// warp that clears the rows behind the group's end in its last block, in both operands (they belong to other groups or to nobody and may
// hold anything), before the MMA reads it.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "grouped.h"
#include "row16.cuh"
#include "umma_core.cuh"

namespace t2sp {

// Tile variants: 128 n x 128 columns by one CTA, 256 x 256 by a CTA pair (grouped_launch says when each is taken).
template <int MODE, int VAR>
struct GroupedCfg {
    static constexpr bool kGrad = MODE == GR_GRAD;
    static constexpr bool kPMn = MODE != GR_FWD_K;           // the MMA's A operand (n) is MN-major
    static constexpr bool kWarps = VAR == GR_TILE_WARPS;
    static constexpr int kPair = VAR == GR_TILE_128 || VAR == GR_TILE_32 || kWarps ? 1 : 2;  // CTAs of a tile
    static constexpr int kTileN = 128 * kPair;
    static constexpr int kTileC = VAR == GR_TILE_32 ? 32 : 128 * kPair;
    // columns come in steps that both CTAs' parts can take: 16 rows of a K-major operand, 64 (a swizzle atom) of an MN-major one
    static constexpr int kColStep = (kGrad ? 64 : 16) * kPair;
    static constexpr int kAccs = 2;                           // accumulators of kTileC columns, for two tiles in turn
    static constexpr int kStages = 6;
    static constexpr int kPBytes = 128 * 128;                 // 128 n x 64 k
    static constexpr int kQBytes = 128 * 128;                 // up to 128 columns x 64 k of one CTA
    static constexpr int kStageBytes = kPBytes + kQBytes;
    static constexpr int kEpiWarps = 8;                       // two for each quarter of the tensor memory's lanes
    static constexpr int kLoadWarps = kWarps ? 2 * kStages : 0;   // two for each stage
    static constexpr int kThreads = (2 + kEpiWarps + (kGrad ? 1 : 0) + kLoadWarps) * 32;
    static constexpr int kTmemCols = kAccs * kTileC;
    static constexpr int kNumBars = 4 * kStages + 4;
    static constexpr int kOutBytes = kEpiWarps * 2048;        // a 64 x 32 tile of 16-bit results for two epilogue warps
    static constexpr int kTableBytes = 2 * (kMaxGroups + 4) * 4 + 16;  // offsets, first tile of each group
    static constexpr int kSmemBytes = kStages * kStageBytes + kOutBytes + kTableBytes + 2048 + kNumBars * 8 + 16 + 1024;
    static_assert(kSmemBytes <= 232448, "shared memory budget exceeded");
};

// One tile of the output and its contraction.
struct __align__(16) GroupedTile {
    int e, n0, c0;      // group, first n, first column (row t of the group in the forward, k in the gradient)
    int cols;           // columns that exist
    int ncols;          // columns the MMA computes
    int num_kb;         // k-blocks, 0: the result is zero
    int row0, tail;     // gradient: first row of the group; rows in its last block (64: not ragged)
};

// n / d and n % d for 0 <= n, 0 < d, through a reciprocal (the compiler's division takes several times as long, and every role
// goes through a handful for each tile): up to quotients of 2^21 the product is off by less than one, beyond by a few.
__device__ __forceinline__ int quick_div(int n, int d, int& rest) {
    int q = static_cast<int>(__fdividef(static_cast<float>(n), static_cast<float>(d)));
    rest = n - q * d;
    while (rest < 0) { --q; rest += d; }
    while (rest >= d) { ++q; rest -= d; }
    return q;
}
// tile_coords of umma_core.cuh: groups of G row-blocks sweep all column-blocks, rows fastest inside a group.
__device__ __forceinline__ void quick_coords(int t, int tiles_m, int tiles_n, int G, int& mb, int& nb) {
    int r;
    const int g = quick_div(t, G * tiles_n, r);
    nb = quick_div(r, min(G, tiles_m - g * G), mb);
    mb += g * G;
}

// Blocks of `tile` that are dealt out first; a last block of at most half a tile is left for the end of the call, so that no CTA has full ones only.
__device__ __forceinline__ int main_blocks(int extent, int tile) {
    const int full = extent / tile, rest = extent - full * tile;
    return full + (rest > tile / 2 ? 1 : 0);
}

// The t-th tile of the call; false when there are no more. Every worker takes every num_workers-th tile.
// (Gradient of 24 empty groups, 776 x 1416, where some workers had eight full tiles and others five: 17.8 -> 14.9 us, 0.6 of it by the list below.)
//   forward   the groups in turn, each with its main blocks of n; then the narrow last blocks of all groups
//   gradient  long groups (grouped_tables) with all their tiles; then the main blocks of the others, their narrow blocks of n, those of k
template <int MODE, int VAR>
__device__ bool grouped_tile(const GroupedParams& p, const int* off, const int* first, int t, GroupedTile& g) {
    using Cfg = GroupedCfg<MODE, VAR>;
    constexpr int kRaster = 2048 / Cfg::kTileN;   // n-blocks that are swept together: 2048 n
    const int nblk = (p.N + Cfg::kTileN - 1) / Cfg::kTileN, nmain = main_blocks(p.N, Cfg::kTileN);
    if constexpr (MODE == GR_GRAD) {
        const int kblk = (p.K + Cfg::kTileC - 1) / Cfg::kTileC, kmain = main_blocks(p.K, Cfg::kTileC), per = nblk * kblk;
        if (t >= per * p.E) return false;
        const int heavy = first[p.E], light = p.E - heavy;
        int mb, kb, rest, place;   // place in the order of the groups
        if (t < heavy * per) {
            place = quick_div(t, per, rest);
            quick_coords(rest, nblk, kblk, kRaster, mb, kb);
        } else if ((t -= heavy * per) < light * nmain * kmain) {
            place = heavy + quick_div(t, nmain * kmain, rest);
            quick_coords(rest, nmain, kmain, kRaster, mb, kb);
        } else if ((t -= light * nmain * kmain) < light * (nblk - nmain) * kmain) {
            place = heavy + quick_div(t, kmain, kb);
            mb = nmain;
        } else {
            t -= light * (nblk - nmain) * kmain;
            place = heavy + quick_div(t, nblk, mb);
            kb = kmain;
        }
        g.e = first[place];
        g.n0 = mb * Cfg::kTileN;
        g.c0 = kb * Cfg::kTileC;
        g.cols = min(Cfg::kTileC, p.K - g.c0);
        g.row0 = off[g.e];
        const int rows = off[g.e + 1] - g.row0;
        g.num_kb = (rows + 63) >> 6;
        g.tail = rows - (g.num_kb - 1) * 64;
    } else {
        const int last = first[p.E] * nmain;   // the first of the narrow tiles
        if (t >= first[p.E] * nblk) return false;
        int mb, tb, e = 0;
        const bool narrow = t >= last;
        if (narrow) t -= last;
        const int each = narrow ? 1 : nmain;
        for (int step = 1 << (31 - __clz(p.E)); step > 0; step >>= 1)   // the last group whose tiles do not begin behind t
            if (e + step < p.E && first[e + step] * each <= t) e += step;
        g.e = e;
        const int lo = off[e], rows = off[e + 1] - lo;
        const int tiles = (rows + Cfg::kTileC - 1) / Cfg::kTileC;
        if (narrow) { mb = nmain; tb = t - first[e]; }
        else quick_coords(t - first[e] * nmain, nmain, tiles, kRaster, mb, tb);
        int rest;
        const int per = quick_div(rows + tiles * Cfg::kColStep - 1, tiles * Cfg::kColStep, rest) * Cfg::kColStep;   // near-equal tiles
        g.n0 = mb * Cfg::kTileN;
        g.c0 = lo + tb * per;
        g.cols = max(0, min(per, lo + rows - g.c0));
        g.num_kb = (p.K + 63) >> 6;
        g.row0 = 0;
        g.tail = 64;
    }
    g.ncols = max(Cfg::kColStep, (g.cols + Cfg::kColStep - 1) / Cfg::kColStep * Cfg::kColStep);
    return true;
}

// The first kListed tiles of a worker, prepared by as many threads at the start: every role goes through the same tiles, and working one out
// takes 0.2 us (gradient of 64 groups of 128 rows, 2048 x 1024: 86 -> 67 us).
constexpr int kListed = 64;
constexpr int kListBytes = kListed * static_cast<int>(sizeof(GroupedTile));
template <int MODE, int VAR>
__device__ __forceinline__ void grouped_list(const GroupedParams& p, const int* off, const int* first, GroupedTile* list, int worker, int num_workers) {
    if (threadIdx.x < kListed) {
        GroupedTile g;
        g.e = -1;
        const long long t = worker + static_cast<long long>(threadIdx.x) * num_workers;
        if (t > 0x7fffffff || !grouped_tile<MODE, VAR>(p, off, first, static_cast<int>(t), g)) g.e = -1;
        list[threadIdx.x] = g;
    }
}
// What a role needs to go through a worker's tiles: for (i = 0; tiles.get(i, g); ++i).
template <int MODE, int VAR>
struct GroupedTiles {
    const GroupedParams& p;
    const int *off, *first;
    const GroupedTile* list;
    int worker, num_workers;
    __device__ __forceinline__ bool get(int i, GroupedTile& g) const {
        if (i < kListed) {
            g = list[i];
            return g.e >= 0;
        }
        const long long t = worker + static_cast<long long>(i) * num_workers;
        return t <= 0x7fffffff && grouped_tile<MODE, VAR>(p, off, first, static_cast<int>(t), g);
    }
};

// Offsets into shared memory, checked, and the number of tiles of rows before every group (forward) or the order of the groups
// and how many are long (gradient). Returns false when the
// offsets decrease or leave the rows; every thread of the CTA gets the verdict.
template <int MODE, int VAR>
__device__ __forceinline__ bool grouped_tables(const GroupedParams& p, int* off, int* first) {
    using Cfg = GroupedCfg<MODE, VAR>;
    int bad = 0;
    for (int e = threadIdx.x; e <= p.E; e += blockDim.x) off[e] = p.offsets[e];
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) bad |= off[e] < 0 || off[e + 1] < off[e] || off[e + 1] > p.rows;
    if (__syncthreads_or(bad)) return false;
    if (MODE != GR_GRAD) {
        if (threadIdx.x < 32) {
            const int lane = threadIdx.x;
            int base = 0;
            for (int e0 = 0; e0 < p.E; e0 += 32) {
                const int e = e0 + lane;
                int v = e < p.E ? (off[e + 1] - off[e] + Cfg::kTileC - 1) / Cfg::kTileC : 0;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int u = __shfl_up_sync(0xffffffffu, v, d);
                    if (lane >= d) v += u;
                }
                if (e < p.E) first[e + 1] = base + v;
                base += __shfl_sync(0xffffffffu, v, 31);
            }
            if (lane == 0) first[0] = 0;
        }
    }
    if (MODE == GR_GRAD) {
        // The gradient's tiles take as long as their group has rows, and every worker takes every num_workers-th tile: the largest groups
        // come first, so that what is left to even out at the end is small (5 groups of 2560 uneven rows: 79 -> 69 us with
        // both gradients). Many groups are taken as they come: ordering them would cost more than it evens out.
        const bool sorted = p.E <= 128;
        const int mean = (off[p.E] - off[0]) / max(1, p.E);
        int longer = 0;
        for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
            const int rows = off[e + 1] - off[e];
            longer += sorted && rows > 2 * mean + 64;
            int place = sorted ? 0 : e;
            for (int i = 0; i < (sorted ? p.E : 0); ++i) {
                const int other = off[i + 1] - off[i];
                place += other > rows || (other == rows && i < e);
            }
            first[place] = e;
        }
        longer = __reduce_add_sync(0xffffffffu, longer);
        if (threadIdx.x == 0) first[p.E] = 0;
        __syncthreads();
        if (sorted && (threadIdx.x & 31) == 0 && longer) atomicAdd(&first[p.E], longer);
    }
    return true;   // the caller synchronises the CTA before the tables are used
}

template <class O> __device__ __forceinline__ O grouped_round(float v);
template <> __device__ __forceinline__ float grouped_round<float>(float v) { return v; }
template <> __device__ __forceinline__ __half grouped_round<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 grouped_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <class O> __device__ __forceinline__ uint32_t pack16(uint32_t lo, uint32_t hi);
template <> __device__ __forceinline__ uint32_t pack16<__half>(uint32_t lo, uint32_t hi) {
    const __half2 v = __floats2half2_rn(__uint_as_float(lo), __uint_as_float(hi));
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(uint32_t lo, uint32_t hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(lo), __uint_as_float(hi));
    return *reinterpret_cast<const uint32_t*>(&v);
}

// 16-bit results of 64 n x 32 columns, by two warps with 32 n each, through a transposed tile in shared memory ([column][n], 128 bytes a column,
// 16-byte pieces at piece ^ (column % 8)): each warp writes its half of every column with four instructions, then takes 16 columns out,
// whole 128-byte lines and 16 bytes a lane. (One 2-byte store a column and lane: a gradient tile of 256 x 256 with little to add up
// took 5 us to leave, a multiple of its products; 64-byte pieces of one warp: 15 bytes a cycle of the 32 that an SM can write.)
// UNROLL: rows at a time that are not all aligned; one where such rows are the rule (5 groups of 13 rows, 7552 x 7923, B by warps: 301 -> 272 us).
// `half`: which warp of the two; `n_left`, `cols`: what exists of the 64 n and of the columns.
// `ok`: whether this warp's accumulator is complete. Each warp waits for it by itself, and one may give up where the other still succeeds: false in
// both where it is false in either, so that they leave together and neither meets the barriers alone.
template <class O, int UNROLL>
__device__ __forceinline__ bool grouped_put(bool ok, uint32_t taddr, bool zero, uint8_t* tile, O* dst, long long ld, int n_left, int cols, int lane,
                                            int half, int barrier) {
    uint32_t r[2][16];
    if (!zero) {
        ptx::tmem_ld_16x256b_x4(taddr, r[0]);
        ptx::tmem_ld_16x256b_x4(taddr + (16u << 16), r[1]);
        ptx::tmem_ld_wait();
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) r[0][j] = r[1][j] = 0u;
    }
    if (!ptx::bar_and(barrier, 64, ok)) return false;   // the tile's previous content has been read
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int piece = half * 4 + 2 * h + ((lane >> 3) & 1);
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const int col = 8 * (i + (lane >> 4)) + (lane & 7);
            ptx::stmatrix_x4_trans(ptx::smem_u32(tile) + col * 128 + ((piece ^ (lane & 7)) << 4), pack16<O>(r[h][4 * i], r[h][4 * i + 1]),
                                   pack16<O>(r[h][4 * i + 2], r[h][4 * i + 3]), pack16<O>(r[h][4 * i + 4], r[h][4 * i + 5]),
                                   pack16<O>(r[h][4 * i + 6], r[h][4 * i + 7]));
        }
    }
    ptx::bar_sync(barrier, 64);
    const int piece = lane & 7;
    dst += piece * 8;
    // every row's pieces on 16 bytes, and all of them there: nothing to look at for each (gradient of 64 groups of 8 rows, 2048 x 1024: 63.4 -> 58.8 us)
    const bool plain = n_left >= 64 && !((reinterpret_cast<uintptr_t>(dst) | static_cast<uintptr_t>(ld * 2)) & 15);
    if (plain && cols >= 32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = 16 * half + 4 * i + (lane >> 3);
            *reinterpret_cast<uint4*>(dst + col * ld) = *reinterpret_cast<const uint4*>(tile + col * 128 + ((piece ^ (col & 7)) << 4));
        }
        return true;
    }
#pragma unroll(UNROLL)
    for (int i = 0; i < 4; ++i) {
        const int col = 16 * half + 4 * i + (lane >> 3);
        const uint4 v = *reinterpret_cast<const uint4*>(tile + col * 128 + ((piece ^ (col & 7)) << 4));
        if (col < cols && piece * 8 < n_left) row16_store(reinterpret_cast<uint16_t*>(dst + col * ld), v, n_left - piece * 8);
    }
    return true;
}

// Writes 32 columns of results from fp32 sums: lane = n, one output row (or k) for each column. Each store instruction writes 32 consecutive n.
template <class O>
__device__ __forceinline__ void grouped_store(O* dst, long long ld, int cols, const float (&r)[32]) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
        if (j < cols) dst[j * ld] = grouped_round<O>(r[j]);
}

// The blocks of a B whose rows do not start on 16 bytes, brought by two warps for each stage of the ring (a stage stays with its warps: a wait on
// the parity of its barrier must not miss a phase). A block is 1024 pieces of eight elements, cut out of the aligned pieces around them and written
// where TMA's 128-byte swizzle would put them (piece ^ row % 8); a lane has the loads of eight pieces on their way together.
// (Copying B into padded memory first moves it three times, once as writes that take nearly twice as long as reads; see
// grouped_warps_worthwhile for what was measured.)
template <int MODE, int VAR>
__device__ __forceinline__ void grouped_load(const GroupedParams& p, const GroupedTiles<MODE, VAR>& tiles, uint8_t* smem, uint64_t* full_bar,
                                             uint64_t* empty_bar, const AbortCtx& ab) {
    using Cfg = GroupedCfg<MODE, VAR>;
    constexpr bool kMn = MODE == GR_FWD_MN;
    constexpr int kBatch = 8;
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) - (2 + Cfg::kEpiWarps), mine = warp >> 1, id = (warp & 1) * 32 + lane;
    // n innermost: 64 k x 16 pieces of 8 n; k innermost: 128 n x 8 pieces of 8 k. This lane's piece of a row, its first row and the step to the next
    constexpr int kPieces = kMn ? 16 : 8, kStep = 64 / kPieces;
    const int c = id % kPieces, r0 = id / kPieces;
    int it = 0;
    GroupedTile g;
    for (int i_tile = 0; tiles.get(i_tile, g); ++i_tile) {
        const uint16_t* b = p.b_src + g.e * p.b_bs;
        for (int kb = 0; kb < g.num_kb; ++kb, ++it) {
            const int s = it % Cfg::kStages;
            if (s != mine) continue;
            uint8_t* slot = smem + s * Cfg::kStageBytes;
            constexpr int kRows = kMn ? 64 : 128, kCols = kMn ? 128 : 64;
            const int row0 = kMn ? kb * 64 : g.n0, col0 = kMn ? g.n0 : kb * 64;
            const int rows = min(kRows, (kMn ? p.K : p.N) - row0), cols = min(kCols, (kMn ? p.N : p.K) - col0);   // that exist
            const uint16_t* block = b + row0 * p.b_ld + col0;
            // Pieces outside the matrix are loaded as if they were its last row's or the row's first one. What they hold does not matter
            // beyond N, whose results are not stored; beyond K it is cleared.
            const uint16_t* src = block + (c * 8 < cols ? c * 8 : 0);
            // the aligned pieces around the first and the last piece lie inside the operand's memory (not at its very ends)
            const bool inside = block - 7 >= p.b_src && block + (rows - 1) * p.b_ld + ((cols - 1) & ~7) + 16 <= p.b_end;
#pragma unroll 1
            for (int i = 0; i < kRows / kStep; i += kBatch) {
                uint4 v[kBatch];
                if (inside) {
                    uint4 lo[kBatch], hi[kBatch];
#pragma unroll
                    for (int j = 0; j < kBatch; ++j) {
                        const uint16_t* at = src + min(r0 + (i + j) * kStep, rows - 1) * p.b_ld;
                        const uint16_t* base = reinterpret_cast<const uint16_t*>(reinterpret_cast<uintptr_t>(at) & ~uintptr_t(15));
                        lo[j] = load16(base);
                        hi[j] = load16(base + 8);
                    }
#pragma unroll
                    for (int j = 0; j < kBatch; ++j) {
                        const uint16_t* at = src + min(r0 + (i + j) * kStep, rows - 1) * p.b_ld;
                        v[j] = row16_cut(lo[j], hi[j], static_cast<int>(reinterpret_cast<uintptr_t>(at) & 15) >> 1);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < kBatch; ++j)
                        v[j] = row16_load(src + min(r0 + (i + j) * kStep, rows - 1) * p.b_ld, min(8, cols - (c * 8 < cols ? c * 8 : 0)), p.b_src, p.b_end);
                }
                if (kb * 64 + 64 > p.K) {
#pragma unroll
                    for (int j = 0; j < kBatch; ++j) {
                        const int left = kMn ? (r0 + (i + j) * kStep < rows ? 8 : 0) : cols - c * 8;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (2 * k + 1 >= left) (&v[j].x)[k] = 2 * k < left ? (&v[j].x)[k] & 0xffffu : 0u;
                    }
                }
                if (i == 0 && !bounded_wait_warp(&empty_bar[s], ((it / Cfg::kStages) & 1) ^ 1, ab, ST_TIMEOUT_SPLITTER, lane)) return;
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    const int r = r0 + (i + j) * kStep;
                    *reinterpret_cast<uint4*>(slot + (kMn ? (c >> 3) * 8192 : 0) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[j];
                }
            }
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&full_bar[s]);
        }
    }
}

template <int MODE, int VAR, class O, bool LONG>
__global__ void __launch_bounds__(GroupedCfg<MODE, VAR>::kThreads, 1)
grouped_kernel(const __grid_constant__ GroupedParams p, const __grid_constant__ GroupedMaps maps) {
    using Cfg = GroupedCfg<MODE, VAR>;
    constexpr int STAGES = Cfg::kStages, kPair = Cfg::kPair;
    // k-blocks that are added up in tensor memory before the epilogue takes them. The tensor core cuts its sums off rather than rounding them: a step of
    // 16 k takes about 4e-9 of the result where signs are mixed (8e-5 of an fp32 gradient over 65536 rows) and 1.1e-7 where all products are positive
    // (7e-3 of a gradient over 2^20 rows). For fp32 results the epilogue adds runs of 32 steps in registers, rounding to nearest (5e-7 at every length, 2.7e-6 of positive products); for
    // 16-bit ones, in the LONG form that longer contractions take, runs of 512 steps (f16) or 4096 (bf16): about 5.5e-5 and 4.4e-4 of positive products, a
    // ninth of what the rounding to that type does. In the gradient each tile goes by its own group's rows.
    constexpr bool kRuns = sizeof(O) == 4 || LONG;
    constexpr int kRun = kRuns ? grouped_run(sizeof(O) == 4 ? GR_OUT_F32 : (std::is_same<O, __half>::value ? GR_OUT_F16 : GR_OUT_BF16)) : 1 << 30;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* out_tiles = smem + STAGES * Cfg::kStageBytes;
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(out_tiles + Cfg::kOutBytes);  // leader's: all CTAs' data landed
    uint64_t* empty_bar = full_bar + STAGES;       // per CTA: the MMAs that read the stage retired
    uint64_t* tail_bar = empty_bar + STAGES;       // gradient, per CTA: its own part of a ragged block landed
    uint64_t* fixed_bar = tail_bar + STAGES;       // gradient, leader's: all CTAs have cleared the ragged block's end
    uint64_t* tfull_bar = fixed_bar + STAGES;      // per CTA: accumulator complete (2)
    uint64_t* tempty_bar = tfull_bar + 2;          // leader's: accumulator drained by all CTAs (2)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
    uint32_t* abort_slot = tmem_slot + 1;
    int* off = reinterpret_cast<int*>(tmem_slot + 4);
    int* first = off + kMaxGroups + 4;
    GroupedTile* list = reinterpret_cast<GroupedTile*>((reinterpret_cast<uintptr_t>(first + kMaxGroups + 4) + 15) & ~uintptr_t(15));

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int rank = kPair == 2 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
    const AbortCtx ab{abort_slot, p.status, p.wait_cycles > 0 ? p.wait_cycles : kWaitTimeoutCycles};
    const int worker = blockIdx.x / kPair, num_workers = gridDim.x / kPair;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(&full_bar[s], Cfg::kWarps ? 3 : 1);
            ptx::mbar_init(&empty_bar[s], 1);
            ptx::mbar_init(&tail_bar[s], 1);
            ptx::mbar_init(&fixed_bar[s], kPair);
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(&tfull_bar[a], 1);
            ptx::mbar_init(&tempty_bar[a], Cfg::kEpiWarps * kPair);
        }
        *abort_slot = 0u;
        ptx::fence_mbar_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc<kPair>(tmem_slot, Cfg::kTmemCols);
        ptx::tmem_relinquish<kPair>();
    }
    ptx::grid_dep_launch();
    ptx::grid_dep_wait();
    const bool valid = grouped_tables<MODE, VAR>(p, off, first);
    __syncthreads();
    if (valid) grouped_list<MODE, VAR>(p, off, first, list, worker, num_workers);
    ptx::tc_fence_before_sync();
    __syncthreads();
    if constexpr (kPair == 2) ptx::cluster_sync();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    if (!valid) {   // every CTA sees the same offsets, so all of them leave here or none does
        if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(p.status, ST_BAD_OFFSETS);
        if (warp == 1) ptx::tmem_dealloc<kPair>(tmem_base, Cfg::kTmemCols);
        return;
    }

    const GroupedTiles<MODE, VAR> tiles = {p, off, first, list, worker, num_workers};

    // the forms for one CTA and for a pair
    auto load2 = [&](void* dst, const void* map, uint64_t* bar, int owner, int c0, int c1) {
        if constexpr (kPair == 2) ptx::tma_load_2d_pair(dst, map, ptx::map_to_cta(bar, owner), c0, c1);
        else ptx::tma_load_2d(dst, map, bar, c0, c1);
    };
    auto load3 = [&](void* dst, const void* map, uint64_t* bar, int owner, int c0, int c1, int c2) {
        if constexpr (kPair == 2) ptx::tma_load_3d_pair(dst, map, ptx::map_to_cta(bar, owner), c0, c1, c2);
        else ptx::tma_load_3d(dst, map, bar, c0, c1, c2);
    };
    auto commit_all = [&](uint64_t* bar) {   // to this barrier of every CTA
        if constexpr (kPair == 2) {
            ptx::umma_commit_pair(ptx::map_to_cta(bar, 0));
            ptx::umma_commit_pair(ptx::map_to_cta(bar, 1));
        } else {
            ptx::umma_commit(bar);
        }
    };

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer (every CTA). The issuing lane is an elected one: the compiler
        // then knows that it is alone, and a k-block's copies take it 170 cycles instead of 520 (which bounded blocks of less than
        // 0.36 us: 27 groups of 64 rows, 5760 x 1408: 98 -> 71 us)
        if (ptx::elect_one()) {
            if (!Cfg::kWarps && p.K > 0 && p.rows > 0) {   // else a map may describe nothing
                ptx::prefetch_tensormap(&maps.p);
                ptx::prefetch_tensormap(&maps.q[0]);
            }
            int it = 0;
            bool ok = true;
            // Test hook for the bounded waits: without the copies from this k-block on the other roles give up (a bound of the loop: a test in it took 0.4 of
            // the 6.7 us of 8 groups of 2 rows, 1024 x 1024)
            const int stop = p.skip_stage > 0 ? p.skip_stage - 1 : 0x7fffffff;
            GroupedTile g;
            for (int i_tile = 0; ok && tiles.get(i_tile, g); ++i_tile) {
                const int part = g.ncols / kPair, brought = min(g.num_kb, stop - it);   // columns of this CTA, k-blocks
                const int n0 = g.n0 + rank * 128;
                const int c0 = g.c0 + rank * part;
                for (int kb = 0; kb < brought; ++kb, ++it) {
                    const int s = it % STAGES;
                    const uint32_t ph = (it / STAGES) & 1;
                    if (!bounded_wait(&empty_bar[s], ph ^ 1, ab, ST_TIMEOUT_PRODUCER)) { ok = false; break; }
                    uint8_t* sp = smem + s * Cfg::kStageBytes;
                    uint8_t* sq = sp + Cfg::kPBytes;
                    uint64_t* bar = &full_bar[s];
                    int owner = 0;
                    if constexpr (MODE == GR_GRAD) {
                        const int qboxes = part > 64 ? 2 : 1, row = g.row0 + kb * 64;
                        const bool ragged = g.tail < 64 && kb == g.num_kb - 1;
                        const int steps = ragged ? (g.tail + 15) >> 4 : 4;   // of 16 rows
                        const int bytes = steps * (2 + qboxes) * 2048;
                        if (ragged) {
                            // each CTA's part is credited to its own barrier, for its clearing warp; the stage's barrier only keeps its phase
                            ptx::mbar_expect_tx(&tail_bar[s], bytes);
                            if (rank == 0) ptx::mbar_arrive(&full_bar[s]);
                            bar = &tail_bar[s];
                            owner = rank;
                        } else if (rank == 0) {
                            ptx::mbar_expect_tx(&full_bar[s], kPair * bytes);
                        }
                        if (steps == 4) {
                            load3(sp, &maps.p, bar, owner, n0, row, 0);
                            load3(sp + 8192, &maps.p, bar, owner, n0 + 64, row, 0);
                            load2(sq, &maps.q[0], bar, owner, c0, row);
                            if (qboxes == 2) load2(sq + 8192, &maps.q[0], bar, owner, c0 + 64, row);
                        } else {   // only the steps that are multiplied (24 groups of 73 rows, 776 x 1416: 22.9 us, with whole blocks 23.8; of 1 row 21.3 and 23.5)
                            for (int j = 0; j < steps; ++j) {
                                load3(sp + j * 2048, &maps.q[1], bar, owner, n0, row + j * 16, 0);
                                load3(sp + 8192 + j * 2048, &maps.q[1], bar, owner, n0 + 64, row + j * 16, 0);
                                load2(sq + j * 2048, &maps.q[2], bar, owner, c0, row + j * 16);
                                if (qboxes == 2) load2(sq + 8192 + j * 2048, &maps.q[2], bar, owner, c0 + 64, row + j * 16);
                            }
                        }
                    } else {
                        if (rank == 0) ptx::mbar_expect_tx(&full_bar[s], kPair * ((Cfg::kWarps ? 0 : Cfg::kPBytes) + part * 128));
                        if constexpr (Cfg::kWarps) {
                        } else if constexpr (MODE == GR_FWD_MN) {
                            load3(sp, &maps.p, bar, owner, n0, kb * 64, g.e);
                            load3(sp + 8192, &maps.p, bar, owner, n0 + 64, kb * 64, g.e);
                        } else {
                            load3(sp, &maps.p, bar, owner, kb * 64, n0, g.e);
                        }
                        // boxes of 128, 64, 32 and 16 rows: at most three a block (eight boxes of 16 rows kept the thread busy for longer
                        // than the block's MMAs)
                        int j = 0;
#pragma unroll
                        for (int b = 0; b < 4; ++b)
                            if (part & (128 >> b)) {
                                load2(sq + j * 128, &maps.q[b], bar, owner, kb * 64, c0 + j);
                                j += 128 >> b;
                            }
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer (leader CTA only)
        if (rank == 0 && ptx::elect_one()) {
            int it = 0, lt = 0;
            uint32_t fixed_ph = 0;
            bool ok = true;
            GroupedTile g;
            uint32_t idesc = 0;
            constexpr uint32_t kStepMn = (16 * 128) >> 4, kStepK = 32 >> 4;
            constexpr uint32_t kStepP = Cfg::kPMn ? kStepMn : kStepK;
            constexpr uint32_t kStepQ = Cfg::kGrad ? kStepMn : kStepK;
            auto wait_block = [&](int i, int kb) -> bool {   // k-block kb of the tile, the i-th of this CTA
                const int s = i % STAGES;
                if (Cfg::kGrad && g.tail < 64 && kb == g.num_kb - 1) {
                    if (!bounded_wait(&fixed_bar[s], (fixed_ph >> s) & 1, ab, ST_TIMEOUT_MMA)) return false;
                    fixed_ph ^= 1u << s;
                } else {
                    if (!bounded_wait(&full_bar[s], (i / STAGES) & 1, ab, ST_TIMEOUT_MMA)) return false;
                }
                ptx::tc_fence_after_sync();
                return true;
            };
            auto steps_of = [&](int kb) -> int { return Cfg::kGrad && kb == g.num_kb - 1 ? (g.tail + 15) >> 4 : 4; };   // of 16 k
            auto issue = [&](uint32_t d_tmem, int kb, int i, int steps) {
                const uint32_t sp = ptx::smem_u32(smem + (i % STAGES) * Cfg::kStageBytes);
                const uint64_t dp = ptx::make_smem_desc(sp, Cfg::kPMn ? 8192 : 16, 1024);
                const uint64_t dq = ptx::make_smem_desc(sp + Cfg::kPBytes, Cfg::kGrad ? 8192 : 16, 1024);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < steps) ptx::umma<ptx::KIND_F16, kPair>(d_tmem, dp + j * kStepP, dq + j * kStepQ, idesc, (kb | j) ? 1u : 0u);
            };
            for (int i_tile = 0; ok && tiles.get(i_tile, g); ++i_tile) {
                if (g.num_kb == 0) continue;   // nothing to add up: the epilogue writes zeros
                idesc = make_instr_desc(1, p.bf16 ? 1 : 0, Cfg::kPMn, Cfg::kGrad, 128 * kPair, g.ncols);
                for (int kb0 = 0; kb0 < g.num_kb && ok; kb0 += kRun, ++lt) {
                    const int acc = lt & 1, kb1 = min(g.num_kb, kb0 + kRun);
                    ok = bounded_wait(&tempty_bar[acc], ((lt >> 1) & 1) ^ 1, ab, ST_TIMEOUT_MMA);
                    ptx::tc_fence_after_sync();
                    for (int kb = kb0; kb < kb1 && ok; ++kb) {
                        ok = wait_block(it + kb, kb);
                        if (!ok) break;
                        issue(tmem_base + acc * Cfg::kTileC, kb - kb0, it + kb, steps_of(kb));
                        commit_all(&empty_bar[(it + kb) % STAGES]);
                    }
                    if (ok) commit_all(&tfull_bar[acc]);
                }
                it += g.num_kb;
            }
        }
    } else if (Cfg::kGrad && warp == 2 + Cfg::kEpiWarps) {
        // ------------------------------------------------------------ clears the end of ragged blocks (every CTA)
        int it = 0;
        uint32_t tail_ph = 0;
        GroupedTile g;
        for (int i_tile = 0; tiles.get(i_tile, g); ++i_tile) {
            it += g.num_kb;
            if (g.num_kb == 0 || g.tail == 64) continue;
            const int s = (it - 1) % STAGES;
            if (!bounded_wait_warp(&tail_bar[s], (tail_ph >> s) & 1, ab, ST_TIMEOUT_SPLITTER, lane)) break;
            tail_ph ^= 1u << s;
            uint8_t* sp = smem + s * Cfg::kStageBytes;
            const int boxes = Cfg::kPBytes / 8192 + (g.ncols / kPair > 64 ? 2 : 1);
            const int end = ((g.tail + 15) & ~15) * 128;   // of the last step of 16 rows that is multiplied
            for (int b = 0; b < boxes; ++b)
                for (int i = g.tail * 128 + lane * 16; i < end; i += 512)
                    *reinterpret_cast<uint4*>(sp + b * 8192 + i) = make_uint4(0, 0, 0, 0);
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_cluster(&fixed_bar[s], 0);
        }
    } else if (Cfg::kWarps && warp >= 2 + Cfg::kEpiWarps) {
        // ------------------------------------------------------------ warps that bring a B which TMA cannot read in place
        if constexpr (Cfg::kWarps) grouped_load<MODE, VAR>(p, tiles, smem, full_bar, empty_bar, ab);
    } else {
        // ------------------------------------------------------------ epilogue (every CTA, its own 128 n): two warps to a quarter of the
        // lanes, each takes every other 32 columns
        const int q = warp & 3, turn = (warp - 2) >> 2;
        const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
        uint8_t* out_tile = out_tiles + (turn * 2 + (q >> 1)) * 4096;
        int lt = 0;
        bool ok = true;
        GroupedTile g;
        for (int i_tile = 0; ok && tiles.get(i_tile, g); ++i_tile) {
            constexpr bool kPuts = sizeof(O) == 2 && (!LONG || MODE == GR_GRAD);
            if (kRuns && (!kPuts || g.num_kb > kRun)) {
                if constexpr (kRuns) {
                    constexpr int kPieces = Cfg::kTileC / 64;   // of 32 columns for each warp
                    float sums[kPieces][32];
#pragma unroll
                    for (int i = 0; i < kPieces; ++i)
#pragma unroll
                        for (int j = 0; j < 32; ++j) sums[i][j] = 0.f;
                    for (int kb = 0; kb < g.num_kb && ok; kb += kRun, ++lt) {
                        const int acc = lt & 1;
                        ok = bounded_wait_warp(&tfull_bar[acc], (lt >> 1) & 1, ab, ST_TIMEOUT_EPILOGUE, lane);
                        if (!ok) break;
                        ptx::tc_fence_after_sync();
#pragma unroll
                        for (int i = 0; i < kPieces; ++i) {
                            uint32_t r[32];
                            ptx::tmem_ld_32x32(lane_base + acc * Cfg::kTileC + turn * 32 + i * 64, r);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 32; ++j) sums[i][j] += __uint_as_float(r[j]);
                        }
                        ptx::tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) {
                            if constexpr (kPair == 2) ptx::mbar_arrive_peer(&tempty_bar[acc], 0);
                            else ptx::mbar_arrive(&tempty_bar[acc]);
                        }
                    }
                    const int n = g.n0 + rank * 128 + q * 32 + lane;
                    O* dst = static_cast<O*>(p.c) + (MODE == GR_GRAD ? g.e * p.bs_c : 0) + g.c0 * p.ldc + n;
                    if (ok && n < p.N)
#pragma unroll
                        for (int i = 0; i < kPieces; ++i) {
                            const int c = turn * 32 + i * 64;
                            grouped_store(dst + c * p.ldc, p.ldc, g.cols - c, sums[i]);
                        }
                }
            } else if constexpr (kPuts) {
                const int acc = lt & 1;
                const uint32_t parity = (lt >> 1) & 1;
                const int n = g.n0 + rank * 128 + q * 32;
                O* dst = static_cast<O*>(p.c) + (MODE == GR_GRAD ? g.e * p.bs_c : 0) + g.c0 * p.ldc + n;
                if (g.num_kb) {
                    ok = bounded_wait_warp(&tfull_bar[acc], parity, ab, ST_TIMEOUT_EPILOGUE, lane);
                    ptx::tc_fence_after_sync();
                }
                const int n64 = n & ~63;   // of the two warps that write together
                if (n64 < p.N) {
#pragma unroll 1
                    for (int c = turn * 32; c < g.cols; c += 64) {
                        const uint32_t taddr = lane_base + acc * Cfg::kTileC + c;
                        ok = grouped_put<O, Cfg::kWarps ? 1 : 4>(ok, taddr, g.num_kb == 0, out_tile, dst + (n64 - n) + c * p.ldc, p.ldc, p.N - n64, g.cols - c,
                                                                 lane, q & 1, 1 + turn * 2 + (q >> 1));
                        if (!ok) break;
                    }
                }
                if (ok && g.num_kb) {
                    ptx::tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) {
                        if constexpr (kPair == 2) ptx::mbar_arrive_peer(&tempty_bar[acc], 0);
                        else ptx::mbar_arrive(&tempty_bar[acc]);
                    }
                }
                if (g.num_kb) ++lt;
            }
        }
    }

    // ---------------------------------------------------------------- teardown
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (*abort_slot) __nanosleep(200000);
    if constexpr (kPair == 2) ptx::cluster_sync();  // neither CTA may release shared memory or TMEM the pair's MMAs still use
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc<kPair>(tmem_base, Cfg::kTmemCols);
    }
}

// ---------------------------------------------------------------- few tiles: the contraction split over a cluster
// Forward products of a few rows, or with a few columns, have fewer 128 x 128 tiles than the GPU has SMs, and one SM brings weights at 60 to 80 GB/s
// only. Here a cluster of `splits` CTAs shares a tile: each adds up its run of k-blocks, hands the fp32 sums of 32 n x 32 columns to the CTA that owns
// them through distributed shared memory, and the owners add the parts in the order of the ranks and write the results. (64 rows, 16384 x 4096, 32
// tiles: four CTAs a tile, 36 us.) Tiles of 32 columns for groups of a few rows leave room for twice the blocks in flight.
template <int VAR>
struct SplitCfg {
    static constexpr int kTileC = VAR == GR_TILE_32 ? 32 : 128;
    static constexpr int kStages = VAR == GR_TILE_32 ? 8 : 4;
    static constexpr int kQBytes = kTileC * 128;
    static constexpr int kStageBytes = 128 * 128 + kQBytes;
    static constexpr int kUnitBytes = 32 * 32 * 4;           // sums of 32 n x 32 columns
    static constexpr int kPartBytes = (VAR == GR_TILE_32 ? 8 : 16) * kUnitBytes;   // an owner's units times the ranks: 4 or 16 units in a tile, 8 ranks
    static constexpr int kThreads = (2 + 8) * 32;
    static constexpr int kTmemCols = 128;
    static constexpr int kTableBytes = 2 * (kMaxGroups + 4) * 4 + 16;
    static constexpr int kSmemBytes = kStages * kStageBytes + kPartBytes + kTableBytes + 2048 + (2 * kStages + 1) * 8 + 24 + 1024;
    static_assert(kSmemBytes <= 232448, "shared memory budget exceeded");
};

template <int MODE, int VAR, class O>
__global__ void __launch_bounds__(SplitCfg<VAR>::kThreads, 1)
grouped_split_kernel(const __grid_constant__ GroupedParams p, const __grid_constant__ GroupedMaps maps, int splits) {
    using SplitC = SplitCfg<VAR>;
    constexpr int STAGES = SplitC::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* parts = reinterpret_cast<float*>(smem + STAGES * SplitC::kStageBytes);   // [unit of this owner][rank][column][n]
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * SplitC::kStageBytes + SplitC::kPartBytes);
    uint64_t* empty_bar = full_bar + STAGES;
    uint64_t* tfull_bar = empty_bar + STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfull_bar + 1);
    uint32_t* abort_slot = tmem_slot + 1;
    int* off = reinterpret_cast<int*>(tmem_slot + 4);
    int* first = off + kMaxGroups + 4;
    GroupedTile* list = reinterpret_cast<GroupedTile*>((reinterpret_cast<uintptr_t>(first + kMaxGroups + 4) + 15) & ~uintptr_t(15));

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int rank = static_cast<int>(ptx::cluster_ctarank());
    const AbortCtx ab{abort_slot, p.status, p.wait_cycles > 0 ? p.wait_cycles : kWaitTimeoutCycles};
    const int worker = blockIdx.x / splits, num_workers = gridDim.x / splits;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(&full_bar[s], 1);
            ptx::mbar_init(&empty_bar[s], 1);
        }
        ptx::mbar_init(tfull_bar, 1);
        *abort_slot = 0u;
        ptx::fence_mbar_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc<1>(tmem_slot, SplitC::kTmemCols);
        ptx::tmem_relinquish<1>();
    }
    ptx::grid_dep_launch();
    ptx::grid_dep_wait();
    const bool valid = grouped_tables<MODE, VAR>(p, off, first);
    __syncthreads();
    if (valid) grouped_list<MODE, VAR>(p, off, first, list, worker, num_workers);
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync();   // every CTA of the cluster runs before its shared memory is written
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    if (!valid) {
        if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(p.status, ST_BAD_OFFSETS);
        if (warp == 1) ptx::tmem_dealloc<1>(tmem_base, SplitC::kTmemCols);
        return;
    }

    int it = 0;
    const GroupedTiles<MODE, VAR> tiles = {p, off, first, list, worker, num_workers};
    const long long total = static_cast<long long>(first[p.E]) * ((p.N + 127) / 128);
    uint32_t phase = 0;   // of the accumulator's barrier: it completes once for every tile with k-blocks
    GroupedTile g;
    for (int i_tile = 0; tiles.get(i_tile, g); ++i_tile) {
        const int kb0 = rank * g.num_kb / splits, nkb = (rank + 1) * g.num_kb / splits - kb0;   // this CTA's run, possibly empty
        if (warp == 0) {
            // -------------------------------------------------------- TMA producer
            if (ptx::elect_one()) {
                const int brought = p.skip_stage > 0 ? min(nkb, max(0, p.skip_stage - 1 - it)) : nkb;   // test hook, as in grouped_kernel
                for (int i = 0; i < brought; ++i) {
                    const int s = (it + i) % STAGES, kb = kb0 + i;
                    if (!bounded_wait(&empty_bar[s], (((it + i) / STAGES) & 1) ^ 1, ab, ST_TIMEOUT_PRODUCER)) break;
                    uint8_t* sp = smem + s * SplitC::kStageBytes;
                    uint8_t* sq = sp + 128 * 128;
                    ptx::mbar_expect_tx(&full_bar[s], 128 * 128 + g.ncols * 128);
                    if constexpr (MODE == GR_FWD_MN) {
                        ptx::tma_load_3d(sp, &maps.p, &full_bar[s], g.n0, kb * 64, g.e);
                        ptx::tma_load_3d(sp + 8192, &maps.p, &full_bar[s], g.n0 + 64, kb * 64, g.e);
                    } else {
                        ptx::tma_load_3d(sp, &maps.p, &full_bar[s], kb * 64, g.n0, g.e);
                    }
                    int j = 0;
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        if (g.ncols & (128 >> b)) {
                            ptx::tma_load_2d(sq + j * 128, &maps.q[b], &full_bar[s], kb * 64, g.c0 + j);
                            j += 128 >> b;
                        }
                }
            }
        } else if (warp == 1) {
            // -------------------------------------------------------- MMA issuer
            if (ptx::elect_one()) {
                const uint32_t idesc = make_instr_desc(1, p.bf16 ? 1 : 0, MODE == GR_FWD_MN, false, 128, g.ncols);
                constexpr uint32_t kStepP = MODE == GR_FWD_MN ? (16 * 128) >> 4 : 32 >> 4, kStepQ = 32 >> 4;
                bool ok = true;
                for (int i = 0; i < nkb && ok; ++i) {
                    const int s = (it + i) % STAGES;
                    ok = bounded_wait(&full_bar[s], ((it + i) / STAGES) & 1, ab, ST_TIMEOUT_MMA);
                    if (!ok) break;
                    ptx::tc_fence_after_sync();
                    const uint32_t sp = ptx::smem_u32(smem + s * SplitC::kStageBytes);
                    const uint64_t dp = ptx::make_smem_desc(sp, MODE == GR_FWD_MN ? 8192 : 16, 1024);
                    const uint64_t dq = ptx::make_smem_desc(sp + 128 * 128, 16, 1024);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        ptx::umma<ptx::KIND_F16, 1>(tmem_base, dp + j * kStepP, dq + j * kStepQ, idesc, (i | j) ? 1u : 0u);
                    ptx::umma_commit(&empty_bar[s]);
                }
                if (ok && nkb) ptx::umma_commit(tfull_bar);
            }
        } else {
            // -------------------------------------------------------- hands 32 n x 32 columns at a time to their owners
            const int q = warp & 3, turn = (warp - 2) >> 2;
            bool have = nkb > 0;
            if (have) {
                have = bounded_wait_warp(tfull_bar, phase, ab, ST_TIMEOUT_EPILOGUE, lane);
                ptx::tc_fence_after_sync();
            }
            for (int c = turn * 32; c < g.cols; c += 64) {
                uint32_t r[32];
                if (have) {
                    ptx::tmem_ld_32x32(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + c, r);
                    ptx::tmem_ld_wait();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) r[j] = 0u;
                }
                const int unit = (c >> 5) * 4 + q;
                const uint32_t at = ptx::map_to_cta(parts + (unit / splits * splits + rank) * 1024 + lane, unit % splits);
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (c + j < g.cols) ptx::st_cluster(at + j * 128, r[j]);
            }
            ptx::tc_fence_before_sync();
        }
        it += nkb;
        if (nkb) phase ^= 1u;
        __syncwarp();
        ptx::cluster_sync();   // all parts have arrived
        ptx::tc_fence_after_sync();
        if (warp >= 2) {
            const int units = 4 * ((g.cols + 31) >> 5);
            for (int i = warp - 2; i < (units - rank + splits - 1) / splits * 32; i += 8) {
                const int own = i >> 5, unit = own * splits + rank, j = i & 31;
                const int col = (unit >> 2) * 32 + j, n = g.n0 + (unit & 3) * 32 + lane;
                if (unit >= units || col >= g.cols) continue;
                const float* part = parts + (own * splits * 32 + j) * 32 + lane;
                float v = part[0];
                for (int k = 1; k < splits; ++k) v += part[k * 1024];
                if (n < p.N) {
                    O* dst = static_cast<O*>(p.c) + (g.c0 + col) * p.ldc + n;
                    *dst = grouped_round<O>(v);
                }
            }
        }
        if (worker + (i_tile + 1ll) * num_workers < total) {   // the parts have been read: the next tile may overwrite them
            __syncwarp();
            ptx::cluster_sync();
        }
    }

    __syncthreads();
    if (*abort_slot) __nanosleep(200000);
    if (warp == 1) ptx::tmem_dealloc<1>(tmem_base, SplitC::kTmemCols);
}

}  // namespace t2sp
