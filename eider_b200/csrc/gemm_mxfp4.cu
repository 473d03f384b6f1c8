// The MXFP4 GEMM kernels: the dense and gated forms of gemm_dense.cu and the grouped form over routed experts.
#include "gemm_launch.cuh"

namespace eider {
namespace gemm {

cudaError_t launch_dense_mxf4(uint32_t block_n, const CUtensorMap& map_rows, const CUtensorMap& map_cols, Params p, cudaStream_t stream) {
    return epilogue_kind(p) == kEpiBf16 ? dispatch_dense<kMxf4, false>(block_n, map_rows, map_cols, p, stream)
                                        : dispatch_dense<kMxf4, true>(block_n, map_rows, map_cols, p, stream);
}

cudaError_t launch_gated_mxf4(const CUtensorMap& map_rows, const CUtensorMap& map_cols, Params p, cudaStream_t stream) {
    return dispatch_gated<kMxf4>(map_rows, map_cols, p, stream);
}

cudaError_t launch_grouped_mxf4(const CUtensorMap& map_rows, const CUtensorMap& map_cols, Params p, uint32_t max_row_tiles, cudaStream_t stream,
                                const ShortRowMaps& short_rows) {
    p.col_tiles = (p.group_cols + 255) / 256;
    const uint32_t items = max_row_tiles * p.col_tiles;
    // (sixteen epilogue warps, one 64-column step each, as in NVFP4)
    if (p.act_packed) return launch<kMxf4, 256, false, 1, true, 16>(map_rows, map_cols, p, items, stream, short_rows);
    return launch<kMxf4, 256, false, 1, true>(map_rows, map_cols, p, items, stream, short_rows);
}

}  // namespace gemm
}  // namespace eider
