// Products whose matrix depends on the row: parameter blocks and launchers (definitions in launch_grouped.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "umma_params.h"

namespace t2sp {

constexpr int kMaxGroups = 1024;  // the kernels keep the groups' tables in shared memory

enum : int { GR_FWD_MN = 0, GR_FWD_K = 1, GR_GRAD = 2 };  // B with n innermost, B with k innermost, gradient of B
// 128 x 128 by one CTA, 256 x 256 by a pair, 128 x 32 by one (of a cluster that shares the contraction), 128 x 128 with
// a B that warps bring
enum : int { GR_TILE_128 = 0, GR_TILE_256 = 1, GR_TILE_32 = 2, GR_TILE_WARPS = 3 };
enum : int { GR_OUT_F32 = 0, GR_OUT_BF16 = 1, GR_OUT_F16 = 2 };
// k-blocks of 64 whose products are added up in tensor memory at a time (see grouped_kernel)
__host__ __device__ constexpr int grouped_run(int out) { return out == GR_OUT_F32 ? 8 : (out == GR_OUT_BF16 ? 1024 : 128); }

// Forward: C[t][n] = sum_k A[t][k] * B[e][k][n] for offsets[e] <= t < offsets[e+1]; rows outside every group are not
// touched. Gradient of B: G[e][k][n] = sum_{t in e} A[t][k] * D[t][n], zero for an empty group.
// The inputs are read through tensor maps; strides in elements.
struct GroupedParams {
    void* c;               // forward: C, rows x N; gradient: G, E x K x N
    const int* offsets;    // E + 1
    long long ldc, bs_c;   // row pitch of C or G, stride between the matrices of G
    int rows, E, K, N;
    int bf16;              // element type of the inputs: 1 bf16, 0 f16
    // an operand B that TMA cannot read in place, read by warps instead (null: through the map)
    const uint16_t *b_src, *b_end;
    long long b_ld, b_bs;
    long long wait_cycles; // limit of every mbarrier wait in SM cycles, 0: kWaitTimeoutCycles
    int skip_stage;        // test hook for the bounded waits: the producers leave out the copies from this k-block on (1-based; 0 = none)
    unsigned* status;
};

struct GroupedMaps {
    CUtensorMap p;      // B (n, k, e), box 64 x 64, or (k, n, e), box 64 k x 128 n; gradient: D (n, t, 1), box 64 x 64
    CUtensorMap q[4];   // forward: A (k, t), 64 k x 128, 64, 32 and 16 rows a box; gradient: A (k, t), 64 k x 64 rows, then D and A with 16 rows a box
};

cudaError_t grouped_launch(int mode, int out, const GroupedParams& p, const GroupedMaps& maps, cudaStream_t stream);

// Whether a B that TMA cannot read in place is better read by warps (through b_src) than copied first.
bool grouped_warps_worthwhile(int mode, int out, const GroupedParams& p);

// dst[m][r][i] (row pitch ld_dst, dense matrices) = src[m * bs_src + r * ld_src + i], 16-bit elements; ld_dst is a multiple of 8. Up to
// two operands in one launch.
struct Repack {
    const uint16_t* src;
    uint16_t* dst;
    long long ld_src, bs_src, ld_dst;
    int inner, rows, matrices;
    unsigned blocks;       // set by the launcher
};
cudaError_t repack16_launch(Repack* jobs, int count, cudaStream_t stream);

}  // namespace t2sp
