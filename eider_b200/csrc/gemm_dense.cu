// The dense GEMM kernels (row-major output), apart from the decode and grouped forms so that both compile side by side.
#include "gemm_launch.cuh"

namespace eider {
namespace gemm {

cudaError_t launch_dense(int kind, uint32_t block_n, const CUtensorMap& map_rows, const CUtensorMap& map_cols, Params p, cudaStream_t stream) {
    if (kind == kMxf4) return launch_dense_mxf4(block_n, map_rows, map_cols, p, stream);
    const bool plain = epilogue_kind(p) == kEpiBf16;
    if (kind == kNvf4)
        return plain ? dispatch_dense<kNvf4, false>(block_n, map_rows, map_cols, p, stream)
                     : dispatch_dense<kNvf4, true>(block_n, map_rows, map_cols, p, stream);
    return plain ? dispatch_dense<kFp8, false>(block_n, map_rows, map_cols, p, stream) : dispatch_dense<kFp8, true>(block_n, map_rows, map_cols, p, stream);
}

cudaError_t launch_gated(int kind, const CUtensorMap& map_rows, const CUtensorMap& map_cols, Params p, cudaStream_t stream) {
    return kind == kMxf4 ? launch_gated_mxf4(map_rows, map_cols, p, stream) : dispatch_gated<kNvf4>(map_rows, map_cols, p, stream);
}

}  // namespace gemm
}  // namespace eider
