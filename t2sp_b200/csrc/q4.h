// Matrices of 4-bit integers with group scales: layout, parameter blocks and launchers (launch_q4.cu).
//
// A matrix W(n, k) is held as w = (nibble - 8) * scale(n, k / group). The nibbles are laid out for the A fragments of the tensor cores'
// m16n8k32 (8-bit) and m16n8k16 (16-bit) instructions: blocks of 16 n x 64 k of 512 bytes, a lane's 16 bytes one after the other. Lane
// 4 g + t holds rows g and g + 8; its 32-bit word w holds k = 16 w + 4 t + j in byte j, row g in the low nibble and row g + 8 in the high
// one. So word & 0x0f0f0f0f is an operand register of four unsigned bytes, and word & 0x000f000f a pair of 16-bit values (j = 0, 2).
// Blocks run along k, then n, then the matrices.
// Scales: 16 for a strip of 16 n in the order g * 2 + (row >= 8), strips along the groups of k, then n, then the matrices.
// What lies beyond N or K holds nibble 8 and scale 0, so it contributes nothing.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "umma_params.h"

namespace t2sp {

__host__ __device__ __forceinline__ int q4_kblocks(int K) { return (K + 63) / 64; }
__host__ __device__ __forceinline__ int q4_strips(int N) { return (N + 15) / 16; }
__host__ __device__ __forceinline__ int q4_groups(int K, int group) { return (q4_kblocks(K) * 64 + group - 1) / group; }

struct Q4Params {
    const void* w;        // pack: the 16-bit matrices; unpack: where they go (wout)
    void* wout;
    const uint16_t* w_end; // behind the last element of w
    long long ldw, bs_w;  // elements between rows (k rows of n, or n rows of k with trans_b) and between matrices
    int trans_b;
    uint8_t* q;
    uint16_t* s;
    int E, K, N, group;
    int bf16;
    // products
    const void* x;        // T x K
    const uint16_t* x_end;
    long long ldx;
    const int* index;     // R matrix numbers or null
    void* y;              // R x N
    long long ldy;
    int R, per;           // row r reads row r / per of x
    int out_f32;
    long long wait_cycles; // limit of every mbarrier wait in SM cycles, 0: kWaitTimeoutCycles
    int skip_stage;        // test hook for the bounded waits: the copies of this slot of every group of warps are left out (1-based; 0 = none)
    unsigned* status;
};

cudaError_t q4_pack_launch(const Q4Params& p, cudaStream_t stream);
cudaError_t q4_unpack_launch(const Q4Params& p, cudaStream_t stream);
// Whether the rows' x and index fit the kernel's shared memory.
bool q4_gemv_fits(int K, int group, int R, bool indexed);
cudaError_t q4_gemv_launch(const Q4Params& p, cudaStream_t stream);

}  // namespace t2sp
