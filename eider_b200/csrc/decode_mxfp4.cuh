// The MXFP4 product for few tokens whose activations are terms of tensor-core operands (decode_mxfp4_terms.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "map_cache.h"

namespace eider {
namespace decode_mx {

// x f32 or bf16 [tokens][k], k % 128 == 0, w 32-byte aligned, n <= 65535 * 128; the scales in tiles; `status`: a device word for a wait that
// ran out (umma::Status).
size_t terms_workspace_bytes(uint32_t tokens, uint32_t k, int input_is_bf16);
cudaError_t run_terms(gemm::FifoCache<CUtensorMap>& maps, const void* x, int input_is_bf16, uint32_t tokens, const uint8_t* w, const uint8_t* scales,
                      const void* c, void* d, float beta, int out_is_bf16, uint32_t n, uint32_t k, uint8_t* workspace, uint32_t* status,
                      cudaStream_t stream);

}  // namespace decode_mx
}  // namespace eider
