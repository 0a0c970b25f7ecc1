// Grouped products: instantiations and launchers (umma_grouped.cuh), and the copy that makes operands fit for TMA.
#include "umma_grouped.cuh"
#include "launch_util.cuh"
#include "row16.cuh"
#include "umma_launch.h"

namespace t2sp {

namespace {

template <int MODE, int VAR, class O, bool LONG>
cudaError_t launch_typed(const GroupedParams& p, const GroupedMaps& maps, int workers, cudaStream_t stream) {
    using Cfg = GroupedCfg<MODE, VAR>;
    auto kern = grouped_kernel<MODE, VAR, O, LONG>;
    static std::atomic<bool> configured[kMaxDev];
    if (cudaError_t e = allow_smem(kern, Cfg::kSmemBytes, configured)) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(workers * Cfg::kPair);
    cfg.blockDim = dim3(Cfg::kThreads);
    cfg.dynamicSmemBytes = Cfg::kSmemBytes;
    cfg.stream = stream;
    // programmatic stream serialization: the launch is set up while the kernel before it ends; grouped_kernel waits for
    // that one before it touches memory
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = Cfg::kPair;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, p, maps);
}

template <int MODE, int VAR, bool LONG = false>
cudaError_t launch_var(int out, const GroupedParams& p, const GroupedMaps& maps, long long tiles, cudaStream_t stream) {
    const long long slots = core_sm_count() / GroupedCfg<MODE, VAR>::kPair;
    const int workers = static_cast<int>(tiles < slots ? (tiles > 0 ? tiles : 1) : slots);
    if constexpr (VAR != GR_TILE_WARPS)
        if (out == GR_OUT_F32) return launch_typed<MODE, VAR, float, false>(p, maps, workers, stream);
    if (out == GR_OUT_BF16) return launch_typed<MODE, VAR, __nv_bfloat16, LONG>(p, maps, workers, stream);
    return launch_typed<MODE, VAR, __half, LONG>(p, maps, workers, stream);
}

template <int MODE, int VAR, class O>
cudaError_t split_typed(const GroupedParams& p, const GroupedMaps& maps, int workers, int splits, cudaStream_t stream) {
    auto kern = grouped_split_kernel<MODE, VAR, O>;
    static std::atomic<bool> configured[kMaxDev];
    if (cudaError_t e = allow_smem(kern, SplitCfg<VAR>::kSmemBytes, configured)) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(workers * splits);
    cfg.blockDim = dim3(SplitCfg<VAR>::kThreads);
    cfg.dynamicSmemBytes = SplitCfg<VAR>::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, p, maps, splits);
}

template <int MODE, int VAR>
cudaError_t launch_split(int out, const GroupedParams& p, const GroupedMaps& maps, long long tiles, int splits, cudaStream_t stream) {
    const long long slots = core_sm_count() / splits;
    const int workers = static_cast<int>(tiles < slots ? (tiles > 0 ? tiles : 1) : slots);
    if (out == GR_OUT_F32) return split_typed<MODE, VAR, float>(p, maps, workers, splits, stream);
    if (out == GR_OUT_BF16) return split_typed<MODE, VAR, __nv_bfloat16>(p, maps, workers, splits, stream);
    return split_typed<MODE, VAR, __half>(p, maps, workers, splits, stream);
}

// Tiles of a call: how the rows fall into the groups is known on the device only. `most`: an upper bound (a tile of each group
// more than the rows alone would need); else as if the rows were spread evenly.
long long count_tiles(int mode, const GroupedParams& p, int tn, int tc, bool most) {
    const long long nblk = (p.N + tn - 1) / tn;
    if (mode == GR_GRAD) return nblk * ((p.K + tc - 1) / tc) * p.E;
    const int groups = p.rows < p.E ? p.rows : p.E;
    if (most) return nblk * (p.rows / tc + groups);
    const int mean = (p.rows + groups - 1) / groups;
    return nblk * groups * ((mean + tc - 1) / tc);
}

// Whether a 16-bit result's contraction (of the gradient: the rows of all groups together) may be longer than a run. (The LONG form of the kernel costs
// the gradient of 64 groups of 256 rows, 2048 x 1024, 6 % where no group is: 206 -> 218 us. Where it has the registers of the warps that bring B, it costs
// 27 groups of 2 rows, 9001 x 1409, f16, 220 -> 261 us.)
bool is_long(int mode, int out, const GroupedParams& p) { return out != GR_OUT_F32 && (mode == GR_GRAD ? p.rows : p.K) > 64 * grouped_run(out); }

// Which tiles. 256 x 256 by a pair brings an SM 32 KB a k-block, and its two accumulators let one tile drain under the next one's products.
// (512 x 256, 48 KB for twice the products but one accumulator, was taken out: 16384 rows in 8 groups, K = 4096, N = 8192: 776 us against 766; gradient
// with 1024 rows a group, 2048 x 2048: 143 against 120.) 128 x 128 by single CTAs where all of them run at once (1000 rows,
// 512 x 512: 6.0 us against 8.6; 256 rows, 4096 x 4096: 14.5 against 24.4; the gradient's outputs are too large for that to pay).
// Of these, clusters share a tile's contraction where that saves more than handing over the sums costs. Measured for 8 tiles, in us with k-blocks: one CTA
// 4.1 + 0.138 kb; of 2, 4 and 8 CTAs with 32 columns 5.9 + 0.069 kb, 5.5 + 0.034 kb and 5.5 + 0.018 kb, with 128 columns
// 11.2 + 0.09 kb, 9.3 + 0.046 kb and 8.3 + 0.026 kb.
template <int MODE>
cudaError_t launch_mode(int out, const GroupedParams& p, const GroupedMaps& maps, cudaStream_t stream) {
    const bool runs = is_long(MODE, out, p);
    if constexpr (MODE != GR_GRAD) {
        if (p.b_src) {
            const long long tiles = count_tiles(MODE, p, 128, 128, true);
            return runs ? launch_var<MODE, GR_TILE_WARPS, true>(out, p, maps, tiles, stream) : launch_var<MODE, GR_TILE_WARPS>(out, p, maps, tiles, stream);
        }
        const long long t128 = count_tiles(MODE, p, 128, 128, false);
        const int kb = (p.K + 63) / 64;
        const bool narrow = p.rows <= 32ll * p.E;   // about a tile of 32 columns to a group
        for (int splits = 8; splits >= 2; splits /= 2) {
            const int least = narrow ? (splits == 8 ? 12 : splits == 4 ? 16 : 28) : (splits == 8 ? 32 : splits == 4 ? 48 : 128);
            if (t128 * splits <= core_sm_count() - (splits == 8 ? 20 : 4) && kb >= least &&   // clusters do not fill every GPC
                kb <= grouped_run(out) * splits)                                               // no longer runs than in the other kernel
                return narrow ? launch_split<MODE, GR_TILE_32>(out, p, maps, count_tiles(MODE, p, 128, 32, true), splits, stream)
                              : launch_split<MODE, GR_TILE_128>(out, p, maps, count_tiles(MODE, p, 128, 128, true), splits, stream);
        }
        if (t128 <= core_sm_count()) {
            const long long tiles = count_tiles(MODE, p, 128, 128, true);
            return runs ? launch_var<MODE, GR_TILE_128, true>(out, p, maps, tiles, stream) : launch_var<MODE, GR_TILE_128>(out, p, maps, tiles, stream);
        }
    }
    const long long tiles = count_tiles(MODE, p, 256, 256, true);
    return runs ? launch_var<MODE, GR_TILE_256, true>(out, p, maps, tiles, stream) : launch_var<MODE, GR_TILE_256>(out, p, maps, tiles, stream);
}

__global__ void __launch_bounds__(256) repack16_kernel(const Repack a, const Repack b) {
    const bool second = blockIdx.x >= a.blocks;
    const Repack& j = second ? b : a;
    // a warp takes 32 pieces of a row at a time
    const int per_row = static_cast<int>(j.ld_dst >> 3), runs = (per_row + 31) / 32;
    const long long idx = ((blockIdx.x - (second ? a.blocks : 0)) * 256ll + threadIdx.x) >> 5;
    const long long row = idx / runs;   // over all matrices
    const int i = (static_cast<int>(idx - row * runs) * 32 + (threadIdx.x & 31)) * 8;
    if (row >= static_cast<long long>(j.rows) * j.matrices || i >= j.ld_dst) return;
    const uint16_t* s = j.src + (row / j.rows) * j.bs_src + (row % j.rows) * j.ld_src + i;
    const uint16_t* end = j.src + (j.matrices - 1) * j.bs_src + (j.rows - 1) * j.ld_src + j.inner;
    *reinterpret_cast<uint4*>(j.dst + row * j.ld_dst + i) = row16_load(s, j.inner - i, j.src, end);
}

}  // namespace

cudaError_t grouped_launch(int mode, int out, const GroupedParams& p, const GroupedMaps& maps, cudaStream_t stream) {
    if (mode == GR_FWD_MN) return launch_mode<GR_FWD_MN>(out, p, maps, stream);
    if (mode == GR_FWD_K) return launch_mode<GR_FWD_K>(out, p, maps, stream);
    return launch_mode<GR_GRAD>(out, p, maps, stream);
}

// Where each group has one tile of columns, B is read once and the copy costs more than the products: 18 groups of 57 rows, 3520 x 2767: 153 us
// by warps against 226 with the copy; 27 groups of 2 rows, 5759 x 1408: 173 against 285; 128 rows a group 209 against 230. With more rows
// the warps read B again for every tile (250 rows, 1001 x 2001: 54 against 44), and with few tiles they cannot keep the memory busy while the
// copy lets a cluster share a tile (2 tiles, K = 5378: 60 against 15).
bool grouped_warps_worthwhile(int mode, int out, const GroupedParams& p) {
    if (mode == GR_GRAD || out == GR_OUT_F32 || p.rows == 0 || p.E == 0) return false;
    const long long groups = p.rows < p.E ? p.rows : p.E;
    return p.rows <= 128 * groups && 3 * count_tiles(mode, p, 128, 128, false) >= 2 * core_sm_count();
}

cudaError_t repack16_launch(Repack* jobs, int count, cudaStream_t stream) {
    unsigned blocks = 0;
    for (int n = 0; n < count; ++n) {
        const long long runs = ((jobs[n].ld_dst >> 3) + 31) / 32;
        jobs[n].blocks = static_cast<unsigned>((static_cast<long long>(jobs[n].rows) * jobs[n].matrices * runs + 7) / 8);
        blocks += jobs[n].blocks;
    }
    repack16_kernel<<<blocks, 256, 0, stream>>>(jobs[0], jobs[count - 1]);
    return cudaGetLastError();
}

}  // namespace t2sp
