// Grouped products on CTA pairs. The operands are exchanged against the other GEMM kernels: the 256 rows of a pair's
// MMA are columns n of the output and the MMA's columns are rows t of the group (forward) or indices k (gradient of B), so
// that a group's ragged end costs an MMA of fewer columns (any multiple of 32) instead of rows computed in vain, and a
// weight tile that meets a handful of rows is still fetched at full width.
//
//   forward   D[n][t] = sum_k B[e][k][n] A[t][k]       tiles of 256 n x up to 256 rows of one group
//   gradient  D[n][k] = sum_t D[t][n] A[t][k]          tiles of 256 n x up to 256 k of one group's matrix; the contraction
//                                                      runs over the group's rows, whose last block is ragged
//
// The group boundaries are read here, on the device: every CTA loads the offsets, checks them and builds the table of
// first tiles in its prologue. Roles per CTA as in umma_pair.cuh (warp 0 producer, 1 MMA, 2-5 epilogue); the gradient has a
// warp 6 that clears the rows behind the group's end in its last block, in both operands (they belong to other groups or to nobody and may
// hold anything), before the MMA reads it.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "grouped.h"
#include "umma_core.cuh"

namespace t2sp {

template <int MODE>
struct GroupedCfg {
    static constexpr bool kGrad = MODE == GR_GRAD;
    static constexpr bool kPMn = MODE != GR_FWD_K;           // the MMA's A operand (n) is MN-major
    static constexpr int kStages = 6;
    static constexpr int kBlockK = 64;
    static constexpr int kPBytes = 128 * 128;                 // 128 n x 64 k of one CTA
    static constexpr int kQBytes = 128 * 128;                 // up to 128 columns x 64 k of one CTA
    static constexpr int kStageBytes = kPBytes + kQBytes;
    static constexpr int kThreads = kGrad ? 7 * 32 : 6 * 32;
    static constexpr int kTmemCols = 512;                     // two 256-column accumulators
    static constexpr int kNumBars = 4 * kStages + 4;
    static constexpr int kTableBytes = 2 * (kMaxGroups + 4) * 4;  // offsets, first tile of each group
    static constexpr int kOutBytes = 4 * 2 * 2048;            // two 32 x 32 tiles of 16-bit results for each epilogue warp
    static constexpr int kSmemBytes = kStages * kStageBytes + kOutBytes + kTableBytes + kNumBars * 8 + 16 + 1024;
    static_assert(kSmemBytes <= 232448, "shared memory budget exceeded");
};

// One tile of the output and its contraction.
struct GroupedTile {
    int e, n0, c0;      // group, first n, first column (row t of the group in the forward, k in the gradient)
    int cols;           // columns that exist (up to 256)
    int ncols;          // columns the MMA computes: cols rounded up to 32 (gradient: 128, whole swizzle atoms in both CTAs)
    int num_kb;         // k-blocks, 0: the result is zero
    int row0, tail;     // gradient: first row of the group; rows in its last block (64: not ragged)
};

template <int MODE>
__device__ __forceinline__ bool grouped_tile(const GroupedParams& p, const int* off, const int* first, int t, int& e, GroupedTile& g) {
    const int nblk = (p.N + 255) >> 8;
    if constexpr (MODE == GR_GRAD) {
        const int kblk = (p.K + 255) >> 8, per = nblk * kblk;
        if (t >= per * p.E) return false;
        g.e = t / per;
        int mb, kb;
        tile_coords(t - g.e * per, nblk, kblk, 8, mb, kb);
        g.n0 = mb * 256;
        g.c0 = kb * 256;
        g.cols = min(256, p.K - g.c0);
        g.row0 = off[g.e];
        const int rows = off[g.e + 1] - g.row0;
        g.num_kb = (rows + 63) >> 6;
        g.tail = rows - (g.num_kb - 1) * 64;
    } else {
        if (t >= first[p.E]) return false;
        while (t >= first[e + 1]) ++e;   // tiles are visited in increasing order
        g.e = e;
        const int lo = off[e], rows = off[e + 1] - lo;
        const int tiles = (rows + 255) >> 8;
        int mb, tb;
        tile_coords(t - first[e], nblk, tiles, 8, mb, tb);
        const int per = ((rows + tiles - 1) / tiles + 31) & ~31;   // near-equal tiles
        g.n0 = mb * 256;
        g.c0 = lo + tb * per;
        g.cols = min(per, lo + rows - g.c0);
        g.num_kb = (p.K + 63) >> 6;
        g.row0 = 0;
        g.tail = 64;
    }
    g.ncols = MODE == GR_GRAD ? (g.cols + 127) & ~127 : (g.cols + 31) & ~31;
    return true;
}

// Offsets into shared memory, checked, and the number of the first tile of every group (forward). Returns false when the
// offsets decrease or leave the rows; every thread of the CTA gets the verdict.
template <int MODE>
__device__ __forceinline__ bool grouped_tables(const GroupedParams& p, int* off, int* first) {
    int bad = 0;
    for (int e = threadIdx.x; e <= p.E; e += blockDim.x) off[e] = p.offsets[e];
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) bad |= off[e] < 0 || off[e + 1] < off[e] || off[e + 1] > p.rows;
    if (__syncthreads_or(bad)) return false;
    if (MODE != GR_GRAD) {
        if (threadIdx.x < 32) {
            const int lane = threadIdx.x, nblk = (p.N + 255) >> 8;
            int base = 0;
            for (int e0 = 0; e0 < p.E; e0 += 32) {
                const int e = e0 + lane;
                int v = e < p.E ? ((off[e + 1] - off[e] + 255) >> 8) * nblk : 0;
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
    return true;   // the caller synchronises the CTA before the tables are used
}

template <class O> __device__ __forceinline__ uint32_t pack16(uint32_t lo, uint32_t hi);
template <> __device__ __forceinline__ uint32_t pack16<__half>(uint32_t lo, uint32_t hi) {
    const __half2 v = __floats2half2_rn(__uint_as_float(lo), __uint_as_float(hi));
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(uint32_t lo, uint32_t hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(lo), __uint_as_float(hi));
    return *reinterpret_cast<const uint32_t*>(&v);
}

// 16-bit results of 32 n x 32 columns through a transposed tile in shared memory ([column][n], 64 bytes a column, 16-byte pieces at
// piece ^ (column / 2 % 4)): four instructions write it, four write it out, 16 bytes a lane and eight columns at a time. `n_left`, `cols`: what
// exists of the 32 n (from the warp's first one on) and of the columns. (One 2-byte store a column and lane: a gradient tile of
// 256 x 256 with little to add up took 5 us to leave, a multiple of its products.)
template <class O>
__device__ __forceinline__ void grouped_put(uint32_t taddr, bool zero, uint8_t* tile, O* dst, long long ld, int n_left, int cols, int lane) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t r[16];
        if (!zero) {
            ptx::tmem_ld_16x256b_x4(taddr + (static_cast<uint32_t>(h * 16) << 16), r);
            ptx::tmem_ld_wait();
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) r[j] = 0u;
        }
        const int piece = 2 * h + ((lane >> 3) & 1);
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const int col = 8 * (i + (lane >> 4)) + (lane & 7);
            ptx::stmatrix_x4_trans(ptx::smem_u32(tile) + col * 64 + ((piece ^ ((col >> 1) & 3)) << 4), pack16<O>(r[4 * i], r[4 * i + 1]),
                                   pack16<O>(r[4 * i + 2], r[4 * i + 3]), pack16<O>(r[4 * i + 4], r[4 * i + 5]),
                                   pack16<O>(r[4 * i + 6], r[4 * i + 7]));
        }
    }
    __syncwarp();
    const int piece = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int col = 8 * i + (lane >> 2);
        const uint4 v = *reinterpret_cast<const uint4*>(tile + col * 64 + ((piece ^ ((col >> 1) & 3)) << 4));
        if (col < cols && piece * 8 < n_left) *reinterpret_cast<uint4*>(dst + col * ld + piece * 8) = v;
    }
}

// Writes 32 columns of the accumulator: lane = n, one output row (or k) for each column. Each store instruction writes 32
// consecutive n. For fp32 results, and for places that take no 16-byte stores.
template <class O>
__device__ __forceinline__ void grouped_store(O* dst, long long ld, int cols, const uint32_t (&r)[32]) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
        if (j < cols) {
            const float v = __uint_as_float(r[j]);
            if constexpr (sizeof(O) == 4) dst[j * ld] = v;
            else if constexpr (std::is_same<O, __half>::value) dst[j * ld] = __float2half_rn(v);
            else dst[j * ld] = __float2bfloat16_rn(v);
        }
}

template <int MODE, class O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GroupedCfg<MODE>::kThreads, 1)
grouped_kernel(const __grid_constant__ GroupedParams p, const __grid_constant__ GroupedMaps maps) {
    using Cfg = GroupedCfg<MODE>;
    constexpr int STAGES = Cfg::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * Cfg::kStageBytes + Cfg::kOutBytes);  // leader's: both CTAs' data landed
    uint64_t* empty_bar = full_bar + STAGES;       // per CTA: the MMAs that read the stage retired
    uint64_t* tail_bar = empty_bar + STAGES;       // gradient, per CTA: its own part of a ragged block landed
    uint64_t* fixed_bar = tail_bar + STAGES;       // gradient, leader's: both CTAs have cleared the ragged block's end
    uint64_t* tfull_bar = fixed_bar + STAGES;      // per CTA: accumulator complete (2)
    uint64_t* tempty_bar = tfull_bar + 2;          // leader's: accumulator drained by both CTAs (2)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
    uint32_t* abort_slot = tmem_slot + 1;
    uint8_t* out_tiles = smem + STAGES * Cfg::kStageBytes;
    int* off = reinterpret_cast<int*>(tmem_slot + 4);
    int* first = off + kMaxGroups + 4;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = ptx::cluster_ctarank();
    const AbortCtx ab{abort_slot, p.status, p.wait_cycles > 0 ? p.wait_cycles : kWaitTimeoutCycles};
    const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

    // every CTA sees the same offsets, so all of them leave here or none does
    if (!grouped_tables<MODE>(p, off, first)) {
        if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(p.status, ST_BAD_OFFSETS);
        return;
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(&full_bar[s], 1);
            ptx::mbar_init(&empty_bar[s], 1);
            ptx::mbar_init(&tail_bar[s], 1);
            ptx::mbar_init(&fixed_bar[s], 2);
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(&tfull_bar[a], 1);
            ptx::mbar_init(&tempty_bar[a], 8);  // 4 epilogue warps in each CTA
        }
        *abort_slot = 0u;
        ptx::fence_mbar_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc<2>(tmem_slot, Cfg::kTmemCols);
        ptx::tmem_relinquish<2>();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer (both CTAs)
        if (lane == 0) {
            if (p.K > 0 && p.rows > 0) {   // else the maps describe nothing and no tile has a k-block
                ptx::prefetch_tensormap(&maps.p);
                ptx::prefetch_tensormap(&maps.q);
            }
            int it = 0, e = 0;
            bool ok = true;
            GroupedTile g;
            for (int t = pair; ok && grouped_tile<MODE>(p, off, first, t, e, g); t += num_pairs) {
                const int half = g.ncols >> 1;
                const int n0 = g.n0 + static_cast<int>(rank) * 128;
                const int c0 = g.c0 + static_cast<int>(rank) * half;
                for (int kb = 0; kb < g.num_kb; ++kb, ++it) {
                    const int s = it % STAGES;
                    const uint32_t ph = (it / STAGES) & 1;
                    if (!bounded_wait(&empty_bar[s], ph ^ 1, ab, ST_TIMEOUT_PRODUCER)) { ok = false; break; }
                    uint8_t* sp = smem + s * Cfg::kStageBytes;
                    uint8_t* sq = sp + Cfg::kPBytes;
                    uint32_t bar;
                    if constexpr (MODE == GR_GRAD) {
                        const int qboxes = half > 64 ? 2 : 1;
                        const int bytes = Cfg::kPBytes + qboxes * 8192;
                        if (g.tail < 64 && kb == g.num_kb - 1) {
                            // ragged block: each CTA's part is credited to its own barrier, for its clearing warp; the
                            // stage's barrier only keeps its phase
                            ptx::mbar_expect_tx(&tail_bar[s], bytes);
                            if (rank == 0) ptx::mbar_arrive(&full_bar[s]);
                            bar = ptx::map_to_cta(&tail_bar[s], rank);
                        } else {
                            if (rank == 0) ptx::mbar_expect_tx(&full_bar[s], 2 * bytes);
                            bar = ptx::map_to_cta(&full_bar[s], 0);
                        }
                        const int row = g.row0 + kb * 64;
                        ptx::tma_load_3d_pair(sp, &maps.p, bar, n0, row, 0);
                        ptx::tma_load_3d_pair(sp + 8192, &maps.p, bar, n0 + 64, row, 0);
                        ptx::tma_load_2d_pair(sq, &maps.q, bar, c0, row);
                        if (qboxes == 2) ptx::tma_load_2d_pair(sq + 8192, &maps.q, bar, c0 + 64, row);
                    } else {
                        if (rank == 0) ptx::mbar_expect_tx(&full_bar[s], 2 * (Cfg::kPBytes + half * 128));
                        bar = ptx::map_to_cta(&full_bar[s], 0);
                        if constexpr (MODE == GR_FWD_MN) {
                            ptx::tma_load_3d_pair(sp, &maps.p, bar, n0, kb * 64, g.e);
                            ptx::tma_load_3d_pair(sp + 8192, &maps.p, bar, n0 + 64, kb * 64, g.e);
                        } else {
                            ptx::tma_load_3d_pair(sp, &maps.p, bar, kb * 64, n0, g.e);
                        }
                        if (half == 128) {
                            ptx::tma_load_2d_pair(sq, &maps.q, bar, kb * 64, c0);
                        } else {
                            for (int j = 0; j < half; j += 16)
                                ptx::tma_load_2d_pair(sq + j * 128, &maps.q16, bar, kb * 64, c0 + j);
                        }
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer (leader CTA only)
        if (lane == 0 && rank == 0) {
            int it = 0, lt = 0, e = 0;
            uint32_t fixed_ph = 0;
            bool ok = true;
            GroupedTile g;
            constexpr uint32_t kStepMn = (16 * 128) >> 4, kStepK = 32 >> 4;
            constexpr uint32_t kStepP = Cfg::kPMn ? kStepMn : kStepK;
            constexpr uint32_t kStepQ = Cfg::kGrad ? kStepMn : kStepK;
            for (int t = pair; ok && grouped_tile<MODE>(p, off, first, t, e, g); t += num_pairs) {
                if (g.num_kb == 0) continue;   // nothing to add up: the epilogue writes zeros
                const int acc = lt & 1;
                if (!bounded_wait(&tempty_bar[acc], ((lt >> 1) & 1) ^ 1, ab, ST_TIMEOUT_MMA)) { ok = false; break; }
                ptx::tc_fence_after_sync();
                const uint32_t d_tmem = tmem_base + acc * 256;
                const uint32_t idesc = make_instr_desc(1, p.bf16 ? 1 : 0, Cfg::kPMn, Cfg::kGrad, 256, g.ncols);
                for (int kb = 0; kb < g.num_kb; ++kb, ++it) {
                    const int s = it % STAGES;
                    if (Cfg::kGrad && g.tail < 64 && kb == g.num_kb - 1) {
                        if (!bounded_wait(&fixed_bar[s], (fixed_ph >> s) & 1, ab, ST_TIMEOUT_MMA)) { ok = false; break; }
                        fixed_ph ^= 1u << s;
                    } else {
                        if (!bounded_wait(&full_bar[s], (it / STAGES) & 1, ab, ST_TIMEOUT_MMA)) { ok = false; break; }
                    }
                    ptx::tc_fence_after_sync();
                    const uint32_t sp = ptx::smem_u32(smem + s * Cfg::kStageBytes);
                    const uint64_t dp = ptx::make_smem_desc(sp, Cfg::kPMn ? 8192 : 16, 1024);
                    const uint64_t dq = ptx::make_smem_desc(sp + Cfg::kPBytes, Cfg::kGrad ? 8192 : 16, 1024);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        ptx::umma<ptx::KIND_F16, 2>(d_tmem, dp + j * kStepP, dq + j * kStepQ, idesc, (kb | j) ? 1u : 0u);
                    ptx::umma_commit_pair(ptx::map_to_cta(&empty_bar[s], 0));
                    ptx::umma_commit_pair(ptx::map_to_cta(&empty_bar[s], 1));
                }
                if (ok) {
                    ptx::umma_commit_pair(ptx::map_to_cta(&tfull_bar[acc], 0));
                    ptx::umma_commit_pair(ptx::map_to_cta(&tfull_bar[acc], 1));
                }
                ++lt;
            }
        }
    } else if (Cfg::kGrad && warp == 6) {
        // ------------------------------------------------------------ clears the end of ragged blocks (both CTAs)
        int it = 0, e = 0;
        uint32_t tail_ph = 0;
        GroupedTile g;
        for (int t = pair; grouped_tile<MODE>(p, off, first, t, e, g); t += num_pairs) {
            it += g.num_kb;
            if (g.num_kb == 0 || g.tail == 64) continue;
            const int s = (it - 1) % STAGES;
            if (!bounded_wait_warp(&tail_bar[s], (tail_ph >> s) & 1, ab, ST_TIMEOUT_SPLITTER, lane)) break;
            tail_ph ^= 1u << s;
            uint8_t* sp = smem + s * Cfg::kStageBytes;
            const int boxes = (g.ncols >> 1) > 64 ? 4 : 3;
            for (int b = 0; b < boxes; ++b)
                for (int i = g.tail * 128 + lane * 16; i < 8192; i += 512)
                    *reinterpret_cast<uint4*>(sp + b * 8192 + i) = make_uint4(0, 0, 0, 0);
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_cluster(&fixed_bar[s], 0);
        }
    } else {
        // ------------------------------------------------------------ epilogue (both CTAs, own 128 n)
        const int q = warp & 3;
        const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
        int lt = 0, e = 0;
        GroupedTile g;
        for (int t = pair; grouped_tile<MODE>(p, off, first, t, e, g); t += num_pairs) {
            const int acc = lt & 1;
            const int n = g.n0 + static_cast<int>(rank) * 128 + q * 32;
            O* dst = static_cast<O*>(p.c) + (MODE == GR_GRAD ? g.e * p.bs_c : 0) + g.c0 * p.ldc + n;
            if (g.num_kb) {
                if (!bounded_wait_warp(&tfull_bar[acc], (lt >> 1) & 1, ab, ST_TIMEOUT_EPILOGUE, lane)) break;
                ptx::tc_fence_after_sync();
            }
#pragma unroll 1
            for (int c = 0; c < g.cols; c += 32) {
                const uint32_t taddr = lane_base + acc * 256 + c;
                if constexpr (sizeof(O) == 2) {
                    if (p.wide_out) {
                        grouped_put(taddr, g.num_kb == 0, out_tiles + (q * 2 + ((c >> 5) & 1)) * 2048, dst + c * p.ldc, p.ldc, p.N - n, g.cols - c, lane);
                        continue;
                    }
                }
                uint32_t r[32];
                if (g.num_kb) {
                    ptx::tmem_ld_32x32(taddr, r);
                    ptx::tmem_ld_wait();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) r[j] = 0u;
                }
                if (n + lane < p.N) grouped_store(dst + c * p.ldc + lane, p.ldc, g.cols - c, r);
            }
            if (g.num_kb) {
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive_peer(&tempty_bar[acc], 0);
                ++lt;
            }
        }
    }

    // ---------------------------------------------------------------- teardown
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (*abort_slot) __nanosleep(200000);
    ptx::cluster_sync();  // neither CTA may release shared memory or TMEM the pair's MMAs still use
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc<2>(tmem_base, Cfg::kTmemCols);
    }
}

}  // namespace t2sp
