// Grouped products: instantiations and launchers (umma_grouped.cuh), and the copy that makes operands fit for TMA.
#include "umma_grouped.cuh"
#include "launch_util.cuh"
#include "umma_launch.h"

namespace t2sp {

namespace {

template <int MODE, class O>
cudaError_t launch_typed(const GroupedParams& p, const GroupedMaps& maps, int grid, cudaStream_t stream) {
    using Cfg = GroupedCfg<MODE>;
    auto kern = grouped_kernel<MODE, O>;
    static std::atomic<bool> configured[kMaxDev];
    if (cudaError_t e = allow_smem(kern, Cfg::kSmemBytes, configured)) return e;
    kern<<<grid, Cfg::kThreads, Cfg::kSmemBytes, stream>>>(p, maps);
    return cudaGetLastError();
}

template <int MODE>
cudaError_t launch_mode(int out, const GroupedParams& p, const GroupedMaps& maps, int grid, cudaStream_t stream) {
    if (out == GR_OUT_F32) return launch_typed<MODE, float>(p, maps, grid, stream);
    if (out == GR_OUT_BF16) return launch_typed<MODE, __nv_bfloat16>(p, maps, grid, stream);
    return launch_typed<MODE, __half>(p, maps, grid, stream);
}

__global__ void repack16_kernel(const uint16_t* __restrict__ src, long long ld_src, long long bs_src, uint16_t* __restrict__ dst,
                                long long ld_dst, int inner, int rows, long long pieces) {
    const long long idx = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    if (idx >= pieces) return;
    const int per_row = static_cast<int>(ld_dst >> 3);
    const int i = static_cast<int>(idx % per_row) * 8;
    const long long row = idx / per_row;   // over all matrices
    const uint16_t* s = src + (row / rows) * bs_src + (row % rows) * ld_src + i;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t lo = i + 2 * j < inner ? s[2 * j] : 0, hi = i + 2 * j + 1 < inner ? s[2 * j + 1] : 0;
        w[j] = lo | (hi << 16);
    }
    *reinterpret_cast<uint4*>(dst + row * ld_dst + i) = make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace

cudaError_t grouped_launch(int mode, int out, const GroupedParams& p, const GroupedMaps& maps, cudaStream_t stream) {
    // at most this many tiles: a tile of each group more than the rows alone would need
    const long long nblk = (p.N + 255) / 256;
    const long long tiles = mode == GR_GRAD ? nblk * ((p.K + 255) / 256) * p.E
                                            : nblk * (p.rows / 256 + (p.rows < p.E ? p.rows : p.E));
    const long long pairs = core_sm_count() / 2;
    const int grid = 2 * static_cast<int>(tiles < pairs ? (tiles > 0 ? tiles : 1) : pairs);
    if (mode == GR_FWD_MN) return launch_mode<GR_FWD_MN>(out, p, maps, grid, stream);
    if (mode == GR_FWD_K) return launch_mode<GR_FWD_K>(out, p, maps, grid, stream);
    return launch_mode<GR_GRAD>(out, p, maps, grid, stream);
}

cudaError_t repack16_launch(const void* src, long long ld_src, long long bs_src, void* dst, long long ld_dst, int inner, int rows,
                            int matrices, cudaStream_t stream) {
    const long long pieces = (ld_dst >> 3) * rows * matrices;
    repack16_kernel<<<static_cast<unsigned>((pieces + 255) / 256), 256, 0, stream>>>(
        static_cast<const uint16_t*>(src), ld_src, bs_src, static_cast<uint16_t*>(dst), ld_dst, inner, rows, pieces);
    return cudaGetLastError();
}

}  // namespace t2sp
