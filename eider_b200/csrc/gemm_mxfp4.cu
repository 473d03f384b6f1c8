// The MXFP4 GEMM kernels: the dense and gated forms of gemm_dense.cu and the grouped form over routed experts.  The mainloop is the NVFP4
// one at the same MMA rate with half as many scale tiles a stage (a block is 32 elements, not 16).  Bound: the tensor cores and, at few row
// tiles, operands from L2 into shared memory.
//
// Measured (B200): 512 x 5120 -> 27648 30.9 us (4.7 PFLOP/s; NVFP4 32), 8192 x 5120 -> 27648 387 us (6.0 PFLOP/s), 2048 x 13824 -> 5120 53.4 us;
// gate/up 2048 x 5120 -> 2 x 13824 with SiLU * up -> MXFP4 in its epilogue 91 us; the experts' pair of 4096 tokens, 8 of 128 experts, 2048 /
// 768, 65 + 53 us, of 77 tokens 40 + 22 us (weights at 5 TB/s); one token's layer 8.6 + 6.8 us.  K 13824 -> N 5120 with 1 / 16 / 64 / 128 tokens 22.5 / 20.7 / 16.4 / 16.9 us:
// 80 tiles of 54 stages each, and no split K.
//
// Outputs whose N is no multiple of 16 elements, or that are not 32-byte aligned, go out one element an access (kEpiOther), which CTA pairs
// feel most: 512 x 2912 -> 5000 53.8 us, -> 5008 10.3 us; 2048 x 2912 -> 5000 148, -> 5008 20.4.  333 tokens have an odd number of row
// tiles and so tiles of one CTA: 10.3 us at N 5000.
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
