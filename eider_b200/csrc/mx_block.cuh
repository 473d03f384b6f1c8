// MXFP4 blocks: 32 consecutive elements of a row as E2M1 codes with one E8M0 scale byte c that stands for 2^(c - 127), 255 for NaN.
//
//   c = clamp(floor(log2(amax)) - 2 + 127, 0, ..)      code = E2M1, nearest even, saturating at 6, of x * 2^(127 - c)
//
// (the OCP microscaling format's conversion: 2 is the exponent of E2M1's largest value).  An all-zero block has c = 0; a block with
// a NaN or an infinity has c = 255 and stands for NaN, so that a poisoned activation shows in every output instead of saturating.
// Scaling by a power of two is exact wherever the result can matter: what underflows is far below the smallest boundary 0.25.
#pragma once

#include "common.cuh"

namespace eider {
namespace mx {

constexpr uint32_t kBlock = 32;
constexpr uint32_t kNanCode = 255;

// Bytes of the tiled scale buffer: the 128-row x 4-block tiles of common.cuh with blocks of 32 elements, i.e. the layout of an
// NVFP4 matrix of half the row length.
__host__ __device__ inline size_t scale_layout_len(size_t outer, size_t inner) {
    return (outer + 127) / 128 * 128 * (((inner + kBlock - 1) / kBlock + 3) / 4 * 4);
}
__host__ __device__ inline size_t tiled_offset(uint32_t outer, uint32_t block, uint32_t blocks) {
    const uint32_t in_tile = outer % 128;
    return (static_cast<size_t>(block / 4) * 4 + static_cast<size_t>(outer / 128) * round_up_u32(blocks, 4)) * 128 + (in_tile % 32) * 16 +
           (in_tile / 32) * 4 + block % 4;
}

#ifdef __CUDACC__

// |v| as an integer: ordered like the values, infinities above them and NaNs above those.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// Scale byte of a block whose largest |x| has these bits.  (Subnormal maxima have exponent field 0 and get c = 0 too.)
__device__ __forceinline__ uint32_t scale_code(uint32_t amax_bits) {
    const uint32_t e = amax_bits >> 23;
    return e == 255 ? kNanCode : e > 2 ? e - 2 : 0;
}
// 2^(127 - c) for c <= 253; what a NaN block is multiplied by does not matter (its codes stand for NaN): any finite value.
__device__ __forceinline__ float inverse_scale(uint32_t code) { return __uint_as_float(code == kNanCode ? 0x3f800000u : (254u - code) << 23); }
// 2^(c - 127), exact in f32 (2^-127 is subnormal), NaN for 255.
__device__ __forceinline__ float scale_value(uint32_t code) {
    return __uint_as_float(code == kNanCode ? 0x7fffffffu : code == 0 ? 0x00400000u : code << 23);
}
// Eight scaled values -> their codes, the first in the low nibble.
__device__ __forceinline__ uint32_t pack8(const float* v) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) w |= static_cast<uint32_t>(e2m1x2_code(v[i], v[i + 1])) << (4 * i);
    return w;
}
// A whole block in one thread.
__device__ __forceinline__ uint32_t quantize_block(float (&v)[32], uint32_t (&words)[4]) {
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) amax = max(amax, abs_bits(v[i]));
    const uint32_t code = scale_code(amax);
    const float inv = inverse_scale(code);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= inv;
#pragma unroll
    for (int i = 0; i < 4; ++i) words[i] = pack8(v + 8 * i);
    return code;
}

// SiLU(gate) * up in front of the quantizer, the stand-alone one and the GEMM epilogues alike (so their bytes agree): hardware
// exponential and reciprocal.  The exponential's error grows with its argument, so the result is off by about (|gate| + 8) * 2^-23 of
// itself, 1e-5 at most, where a code's boundaries lie a quarter of its value apart.  Below gate -87.3, where e^-gate passes 2^126, the
// quotient is 0 instead of 2^-119 * up or less.
__device__ __forceinline__ float silu_mul(float g, float u) { return __fmul_rn(__fdividef(g, __fadd_rn(1.0f, __expf(-g))), u); }

#endif  // __CUDACC__

}  // namespace mx
}  // namespace eider
