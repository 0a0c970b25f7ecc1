// Products whose matrix depends on the row: parameter blocks and launchers (definitions in launch_grouped.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "umma_params.h"

namespace t2sp {

constexpr int kMaxGroups = 1024;  // the kernels keep the groups' tables in shared memory

// Forward: C[t][n] = sum_k A[t][k] * B[e][k][n] for offsets[e] <= t < offsets[e+1]; rows outside every group are not
// touched. Gradient of B: G[e][k][n] = sum_{t in e} A[t][k] * D[t][n], zero for an empty group.
// Strides in elements; the innermost stride of every operand is 1.
struct GroupedParams {
    const void* a;         // A: rows x K
    const void* b;         // forward: B, E x K x N (trans_b: E x N x K); gradient: D, rows x N
    void* c;               // forward: C, rows x N; gradient: G, E x K x N
    const int* offsets;    // E + 1
    long long lda, ldb, ldc;
    long long bs_b, bs_c;  // strides between the matrices of B and of G
    int rows, E, K, N;
    int trans_b;
    int grad;
    int bf16;              // element type of the inputs: 1 bf16, 0 f16
    int out_f32;           // output element: 1 fp32, 0 the inputs' type
    unsigned* status;
};

cudaError_t grouped_launch(const GroupedParams& p, cudaStream_t stream);

}  // namespace t2sp
