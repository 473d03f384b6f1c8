// MXFP4 quantizers and their inverse: rows of activations or weights, SiLU * up rows, and rows of a routed layer written straight to
// their routes.  The format is in mx_block.cuh; the products are in gemm_mxfp4.cu and decode_mxfp4.cu.
//
// Every kernel gives a lane eight consecutive elements (16 bytes of bf16, one 4-byte word of codes), four lanes a block and sixteen
// lanes a UNIT of four blocks: 128 elements whose four scale bytes are one word of the tiled layout.  The block maximum takes two
// shuffles, the scale word two more; loads and stores of a warp are contiguous.
//
// Bound: HBM, elements in and 17/32 byte an element out.  Measured (B200): 16384 x 13824 bf16 135 us (4.3 TB/s, 0.65 of a copy), 4096 x 8192
// f32 26.4 us (0.88), 512 x 5120 5.4 us, one row of 5120 1.7 us; the inverse 16384 x 13824 150 us; SiLU * up 2048 x 13824 45.3 us (0.87), 128 x
// 13824 6.2.  Counters of 4096 x 13824 bf16: the quantizer issues 14.5 warp instructions per 32 elements, mostly on the ALU pipe (68 % busy,
// issue slots 65 %), with 27 of 64 warps resident (64 registers); the inverse 17.8 (ALU 76 %, issue 73 %, 35 warps), as it puts an element
// together bit by bit.  So both are bound by their instructions before memory.
#include <algorithm>

#include "common.cuh"
#include "mx_block.cuh"
#include "quant_block.cuh"
#include "eider_b200.h"

namespace eider {
namespace {

constexpr uint32_t kFullMask = 0xffffffffu;
constexpr uint32_t kUnit = 128;

// Eight elements at p, from aligned rows in 16-byte loads.  (Never with __ldg: to the compiler a read-only load has no order with
// griddepcontrol.wait.)
template <bool VEC> __device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    if (VEC) {
        const float4 a = __ldcg(reinterpret_cast<const float4*>(p)), b = __ldcg(reinterpret_cast<const float4*>(p) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __ldcg(p + i);
    }
}
template <bool VEC> __device__ __forceinline__ void load8(const uint16_t* p, float (&v)[8]) {
    if (VEC) {
        const uint4 u = __ldcg(reinterpret_cast<const uint4*>(p));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = __uint_as_float(w[j] << 16);
            v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = bf16_bits_to_float(__ldcg(p + i));
    }
}

// What a quantizer reads: rows of f32 or bf16 values, or f32 rows of gate and up halves.
template <typename T, bool VEC> struct PlainRows {
    const T* input;
    size_t stride;
    __device__ __forceinline__ void load(uint32_t row, uint32_t k, float (&v)[8]) const { load8<VEC>(input + row * stride + k, v); }
};
struct SiluRows {
    const float* input;
    size_t stride;
    uint32_t inner;
    __device__ __forceinline__ void load(uint32_t row, uint32_t k, float (&v)[8]) const {
        float up[8];
        load8<true>(input + row * stride + k, v);
        load8<true>(input + row * stride + inner + k, up);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = mx::silu_mul(v[i], up[i]);
    }
};

// A lane's eight elements -> their code word and their block's scale byte (four lanes of a block, all of them here).
__device__ __forceinline__ uint32_t quantize8(float (&v)[8], uint32_t& code) {
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, mx::abs_bits(v[i]));
    amax = max(amax, __shfl_xor_sync(kFullMask, amax, 1));
    amax = max(amax, __shfl_xor_sync(kFullMask, amax, 2));
    code = mx::scale_code(amax);
    const float inv = mx::inverse_scale(code);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= inv;
    return mx::pack8(v);
}
// The four scale bytes of a unit as a word, in all sixteen lanes.
__device__ __forceinline__ uint32_t scale_word(uint32_t code, uint32_t lane16) {
    uint32_t word = code << (8 * (lane16 >> 2));
    word |= __shfl_xor_sync(kFullMask, word, 4);
    word |= __shfl_xor_sync(kFullMask, word, 8);
    return word;
}

// rows x inner -> packed codes, and scale bytes in the tiled layout with its padding (ROW_MAJOR: [rows][inner / 32] instead).
// Bound: HBM, the input read once and 17/32 byte an element written.
// ACTIVATION: launched as a programmatic dependent that lets the next launch start early; not for weights, which the GEMMs
// request before they wait for the launch in front of them.
constexpr uint32_t kQuantThreads = 256;
constexpr uint32_t kQuantAhead = 4;  // units a half-warp has on their way
template <typename Rows, bool ROW_MAJOR, bool ACTIVATION>
__global__ void __launch_bounds__(kQuantThreads) quantize_mxfp4_kernel(const Rows source, uint8_t* __restrict__ packed, uint8_t* __restrict__ scales,
                                                                       uint32_t rows, uint32_t inner, uint32_t units, const FastDiv units_per_row) {
    if (ACTIVATION) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
    const uint32_t thread = blockIdx.x * kQuantThreads + threadIdx.x, threads = gridDim.x * kQuantThreads;
    const uint32_t lane16 = threadIdx.x & 15, step = threads / 16;
    const uint32_t padded_blocks = units_per_row.d * 4;
    // (the bound is the warp's, so that its two halves leave together)
    for (uint32_t first = thread / 32 * 2; first < units; first += step * kQuantAhead) {
        const uint32_t mine = first + ((threadIdx.x >> 4) & 1);
        float v[kQuantAhead][8];
        uint32_t row[kQuantAhead], u[kQuantAhead];
        bool live[kQuantAhead];
#pragma unroll
        for (uint32_t a = 0; a < kQuantAhead; ++a) {
            const uint32_t unit = mine + a * step;
            row[a] = units_per_row.div(unit);
            u[a] = unit - row[a] * units_per_row.d;
            live[a] = unit < units && u[a] * kUnit + lane16 * 8 < inner;
            if (live[a]) {
                source.load(row[a], u[a] * kUnit + lane16 * 8, v[a]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[a][i] = 0.0f;
            }
        }
#pragma unroll
        for (uint32_t a = 0; a < kQuantAhead; ++a) {
            uint32_t code;
            const uint32_t w = quantize8(v[a], code);
            const uint32_t k = u[a] * kUnit + lane16 * 8;
            if (live[a]) reinterpret_cast<uint32_t*>(packed + static_cast<size_t>(row[a]) * (inner / 2))[k / 8] = w;
            if (ROW_MAJOR) {
                if (live[a] && (lane16 & 3) == 0) scales[static_cast<size_t>(row[a]) * (inner / 32) + k / 32] = static_cast<uint8_t>(code);
            } else {
                const uint32_t word = scale_word(code, lane16);
                if (lane16 == 0 && mine + a * step < units)
                    *reinterpret_cast<uint32_t*>(scales + (static_cast<size_t>(row[a] / 128) * padded_blocks + u[a] * 4) * 128 + (row[a] % 32) * 16 +
                                                 (row[a] / 32 % 4) * 4) = word;
            }
        }
    }
    if (!ROW_MAJOR) zero_padding_rows(scales, rows, inner / 2, thread, threads);
}

template <bool ROW_MAJOR, bool ACTIVATION, typename Rows>
cudaError_t launch_quantize(const Rows& source, uint8_t* packed, uint8_t* scales, uint32_t rows, uint32_t inner, cudaStream_t stream) {
    const uint64_t per_row = (static_cast<uint64_t>(inner) + kUnit - 1) / kUnit, units = rows * per_row;
    // (indices of units up to a grid step beyond the last have to stay below 2^31)
    if (units > 0x40000000u) return cudaErrorInvalidValue;
    const uint32_t ctas = static_cast<uint32_t>(std::min<uint64_t>((units + kQuantThreads / 16 - 1) / (kQuantThreads / 16), 148u * 8u));
    auto kernel = quantize_mxfp4_kernel<Rows, ROW_MAJOR, ACTIVATION>;
    const FastDiv div(static_cast<uint32_t>(per_row));
    if (ACTIVATION)
        return launch_dependent(kernel, dim3(ctas), kQuantThreads, 0, stream, source, packed, scales, rows, inner, static_cast<uint32_t>(units), div);
    kernel<<<ctas, kQuantThreads, 0, stream>>>(source, packed, scales, rows, inner, static_cast<uint32_t>(units), div);
    return cudaGetLastError();
}

template <bool ROW_MAJOR, bool ACTIVATION>
cudaError_t quantize_rows(const void* input, int input_is_bf16, size_t stride, uint8_t* packed, uint8_t* scales, uint32_t rows, uint32_t inner,
                          cudaStream_t stream) {
    const uintptr_t address = reinterpret_cast<uintptr_t>(input);
    if (input_is_bf16) {
        const auto* x = static_cast<const uint16_t*>(input);
        if (address % 16 == 0 && stride % 8 == 0)
            return launch_quantize<ROW_MAJOR, ACTIVATION>(PlainRows<uint16_t, true>{x, stride}, packed, scales, rows, inner, stream);
        return launch_quantize<ROW_MAJOR, ACTIVATION>(PlainRows<uint16_t, false>{x, stride}, packed, scales, rows, inner, stream);
    }
    const auto* x = static_cast<const float*>(input);
    if (address % 16 == 0 && stride % 4 == 0)
        return launch_quantize<ROW_MAJOR, ACTIVATION>(PlainRows<float, true>{x, stride}, packed, scales, rows, inner, stream);
    return launch_quantize<ROW_MAJOR, ACTIVATION>(PlainRows<float, false>{x, stride}, packed, scales, rows, inner, stream);
}

// The inverse: a lane's eight codes times their block's scale.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) dequantize_mxfp4_kernel(const uint8_t* __restrict__ packed, const uint8_t* __restrict__ scales,
                                                                         T* __restrict__ out, uint32_t inner, uint32_t units,
                                                                         const FastDiv units_per_row) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t thread = blockIdx.x * kQuantThreads + threadIdx.x, step = gridDim.x * kQuantThreads / 16;
    const uint32_t lane16 = threadIdx.x & 15, padded_blocks = units_per_row.d * 4;
    for (uint32_t first = thread / 16; first < units; first += step * kQuantAhead) {
        uint32_t words[kQuantAhead], codes[kQuantAhead], row[kQuantAhead], k[kQuantAhead];
        bool live[kQuantAhead];
#pragma unroll
        for (uint32_t a = 0; a < kQuantAhead; ++a) {
            const uint32_t unit = first + a * step;
            row[a] = units_per_row.div(unit);
            const uint32_t u = unit - row[a] * units_per_row.d;
            k[a] = u * kUnit + lane16 * 8;
            live[a] = unit < units && k[a] < inner;
            words[a] = codes[a] = 0;
            if (live[a]) {
                words[a] = __ldcg(reinterpret_cast<const uint32_t*>(packed + static_cast<size_t>(row[a]) * (inner / 2)) + k[a] / 8);
                codes[a] = __ldcg(scales + (static_cast<size_t>(row[a] / 128) * padded_blocks + u * 4) * 128 + (row[a] % 32) * 16 + (row[a] / 32 % 4) * 4 +
                                 (lane16 >> 2));
            }
        }
#pragma unroll
        for (uint32_t a = 0; a < kQuantAhead; ++a) {
            if (!live[a]) continue;
            const float s = mx::scale_value(codes[a]);
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = e2m1_value(words[a] >> (4 * i) & 15u) * s;
            T* dst = out + static_cast<size_t>(row[a]) * inner + k[a];
            if constexpr (sizeof(T) == 2) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                    w[i] = *reinterpret_cast<const uint32_t*>(&h);
                }
                *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
                reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
                reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
        }
    }
}

// Row-major scale bytes of `groups` stacked matrices [rows][blocks] -> the tiled layout, each matrix on row tiles of its own.
__global__ void __launch_bounds__(256) mx_scales_to_tiled_kernel(const uint8_t* __restrict__ src, uint8_t* __restrict__ dst, uint32_t groups,
                                                                 uint32_t rows, uint32_t blocks) {
    const uint32_t row_tiles = (rows + 127) / 128, padded = round_up_u32(blocks, 4);
    const size_t total = static_cast<size_t>(groups) * row_tiles * 128 * padded;
    for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<size_t>(gridDim.x) * 256) {
        // i is the destination: [tile][group of four blocks][row % 32][row / 32 % 4][block % 4]
        const size_t tile = i / (128 * padded);
        const uint32_t in = static_cast<uint32_t>(i - tile * 128 * padded);
        const uint32_t block = in / 512 * 4 + in % 4;
        const uint32_t row = static_cast<uint32_t>(tile % row_tiles) * 128 + in % 512 / 16 + in % 16 / 4 * 32;
        const size_t group = tile / row_tiles;
        dst[i] = row < rows && block < blocks ? src[(group * rows + row) * blocks + block] : 0;
    }
}

// Rows of a routed layer: a token's row is quantized once and written to all of its routes, one CTA per token and group of routes.
// Bound: HBM, the rows read once and 17/32 byte an element and route written.  4096 x 2048 bf16, 8 routes each: 17.5 us for 52 MB; 9.8 million
// warp instructions, issue slots 54 %, ALU 52 %: the CTA per token with its barrier and the stores' addressing, not memory.
constexpr uint32_t kMaxSlots = 64;
constexpr uint32_t kSpreadRows = 148, kSpreadSlots = 8;  // fewer rows than SMs: a row's routes in groups of eight, a CTA each
template <typename T>
__global__ void __launch_bounds__(1024) moe_quantize_routes_mxfp4_kernel(const T* __restrict__ input, const uint32_t* __restrict__ route_to_sorted,
                                                                         const uint32_t* __restrict__ sorted_routes,
                                                                         const uint32_t* __restrict__ sorted_experts,
                                                                         const uint32_t* __restrict__ offsets, uint8_t* __restrict__ packed,
                                                                         uint8_t* __restrict__ scales, uint32_t routes, uint32_t routes_per_row,
                                                                         uint32_t slots_per_cta, uint32_t inner, uint32_t tile_bytes) {
    __shared__ size_t row_at[kMaxSlots], scale_at[kMaxSlots];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t token = blockIdx.x, lane16 = threadIdx.x & 15;
    const T* src = input + static_cast<size_t>(token) * inner;
    float v[8];
    const bool first_live = threadIdx.x * 8 < inner;
    if (first_live) load8<true>(src + threadIdx.x * 8, v);
    const uint32_t slot0 = blockIdx.y * slots_per_cta, slots = min(slots_per_cta, routes_per_row - slot0);
    if (threadIdx.x < slots) {
        const uint32_t route = token * routes_per_row + slot0 + threadIdx.x, sorted = __ldcg(route_to_sorted + route);
        size_t row = ~static_cast<size_t>(0), scale = 0;
        if (sorted < routes && __ldcg(sorted_routes + sorted) == route) {  // (a route to an expert that does not exist has no place)
            const uint32_t expert = __ldcg(sorted_experts + sorted), offset = __ldcg(offsets + expert);
            row = static_cast<size_t>(sorted) * (inner / 2);
            scale = ((static_cast<size_t>(offset) + 127) / 128 + expert) * tile_bytes + mx::tiled_offset(sorted - offset, 0, inner / mx::kBlock);
        }
        row_at[threadIdx.x] = row;
        scale_at[threadIdx.x] = scale;
    }
    __syncthreads();
    for (uint32_t base = 0; base < inner; base += blockDim.x * 8) {  // (whole warps)
        const uint32_t k = base + threadIdx.x * 8;
        if (k < inner) {
            if (base != 0) load8<true>(src + k, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        }
        uint32_t code;
        const uint32_t w = quantize8(v, code), word = scale_word(code, lane16);
        for (uint32_t s = 0; s < slots; ++s) {
            const size_t row = row_at[s];
            if (row == ~static_cast<size_t>(0)) continue;
            if (k < inner) *reinterpret_cast<uint32_t*>(packed + row + k / 2) = w;
            // the lanes of a unit take turns with the slots; a row's last unit writes the padding blocks' zeros
            if ((s & 15) == lane16 && k / kUnit * kUnit < inner) *reinterpret_cast<uint32_t*>(scales + scale_at[s] + (k / kUnit) * 512) = word;
        }
    }
}

bool rows_ok(uint32_t rows, uint32_t inner) { return rows != 0 && inner != 0 && inner % mx::kBlock == 0 && inner <= 0x40000000u; }
bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace
}  // namespace eider

using namespace eider;

extern "C" {

size_t eider_b200_mxfp4_scale_layout_len(size_t outer, size_t inner) { return mx::scale_layout_len(outer, inner); }

cudaError_t eider_b200_quantize_mxfp4_on_stream(const void* input, int input_is_bf16, size_t row_stride, uint8_t* packed, uint8_t* scales,
                                                uint32_t tokens, uint32_t in_features, cudaStream_t stream) {
    if (!input || !packed || !scales || !rows_ok(tokens, in_features) || row_stride < in_features || !aligned(input, input_is_bf16 ? 2 : 4) ||
        !aligned(packed, 4) || !aligned(scales, 16))
        return cudaErrorInvalidValue;
    return quantize_rows<false, true>(input, input_is_bf16, row_stride, packed, scales, tokens, in_features, stream);
}

cudaError_t eider_b200_quantize_mxfp4_weight_on_stream(const void* weight, int input_is_bf16, uint8_t* packed, uint8_t* scales_row_major,
                                                       uint32_t out_features, uint32_t in_features, cudaStream_t stream) {
    if (!weight || !packed || !scales_row_major || !rows_ok(out_features, in_features) || !aligned(weight, input_is_bf16 ? 2 : 4) || !aligned(packed, 4))
        return cudaErrorInvalidValue;
    return quantize_rows<true, false>(weight, input_is_bf16, in_features, packed, scales_row_major, out_features, in_features, stream);
}

cudaError_t eider_b200_silu_mul_halves_quantize_mxfp4_on_stream(const float* gate_up, uint8_t* packed, uint8_t* scales, uint32_t tokens, uint32_t inner,
                                                                cudaStream_t stream) {
    if (!gate_up || !packed || !scales || !rows_ok(tokens, inner) || !aligned(gate_up, 16) || !aligned(packed, 4) ||
        !aligned(scales, 16))
        return cudaErrorInvalidValue;
    return launch_quantize<false, true>(SiluRows{gate_up, 2 * static_cast<size_t>(inner), inner}, packed, scales, tokens, inner, stream);
}

cudaError_t eider_b200_dequantize_mxfp4_on_stream(const uint8_t* packed, const uint8_t* scales, void* output, int output_is_bf16, uint32_t rows,
                                                  uint32_t in_features, cudaStream_t stream) {
    if (!packed || !scales || !output || !rows_ok(rows, in_features) || !aligned(packed, 4) || !aligned(output, 16)) return cudaErrorInvalidValue;
    const uint64_t per_row = (static_cast<uint64_t>(in_features) + kUnit - 1) / kUnit, units = rows * per_row;
    if (units > 0x40000000u) return cudaErrorInvalidValue;
    const uint32_t ctas = static_cast<uint32_t>(std::min<uint64_t>((units + kQuantThreads / 16 - 1) / (kQuantThreads / 16), 148u * 8u));
    const FastDiv div(static_cast<uint32_t>(per_row));
    if (output_is_bf16)
        return launch_dependent(dequantize_mxfp4_kernel<uint16_t>, dim3(ctas), kQuantThreads, 0, stream, packed, scales,
                                static_cast<uint16_t*>(output), in_features, static_cast<uint32_t>(units), div);
    return launch_dependent(dequantize_mxfp4_kernel<float>, dim3(ctas), kQuantThreads, 0, stream, packed, scales, static_cast<float*>(output),
                            in_features, static_cast<uint32_t>(units), div);
}

cudaError_t eider_b200_mxfp4_scales_to_tiled_on_stream(const uint8_t* scales_row_major, uint8_t* scales_tiled, uint32_t groups, uint32_t out_features,
                                                       uint32_t in_features, cudaStream_t stream) {
    if (!scales_row_major || !scales_tiled || groups == 0 || !rows_ok(out_features, in_features)) return cudaErrorInvalidValue;
    mx_scales_to_tiled_kernel<<<148 * 8, 256, 0, stream>>>(scales_row_major, scales_tiled, groups, out_features, in_features / mx::kBlock);
    return cudaGetLastError();
}

cudaError_t eider_b200_moe_quantize_routes_mxfp4_on_stream(const void* input, int input_is_bf16, const uint32_t* route_to_sorted,
                                                           const uint32_t* sorted_routes, const uint32_t* sorted_experts,
                                                           const uint32_t* expert_offsets, uint8_t* packed, uint8_t* scales, uint32_t rows,
                                                           uint32_t routes_per_row, uint32_t in_features, uint32_t scale_tile_bytes,
                                                           cudaStream_t stream) {
    if (!input || !route_to_sorted || !sorted_routes || !sorted_experts || !expert_offsets || !packed || !scales || !rows_ok(rows, in_features) ||
        routes_per_row == 0 || routes_per_row > kMaxSlots || static_cast<uint64_t>(rows) * routes_per_row > 0xffffffffu ||
        scale_tile_bytes != (in_features / mx::kBlock + 3) / 4 * 4 * 128 || !aligned(input, 16) || !aligned(packed, 4) || !aligned(scales, 4))
        return cudaErrorInvalidValue;
    const uint32_t routes = rows * routes_per_row;
    const uint32_t slots_per_cta = rows < kSpreadRows ? std::min(routes_per_row, kSpreadSlots) : routes_per_row;
    // a thread per eight elements, in whole warps and at least one per route slot
    const uint32_t threads = std::min(1024u, std::max((in_features / 8 + 31) / 32 * 32, (slots_per_cta + 31) / 32 * 32));
    const dim3 grid(rows, (routes_per_row + slots_per_cta - 1) / slots_per_cta);
    if (input_is_bf16)
        return launch_dependent(moe_quantize_routes_mxfp4_kernel<uint16_t>, grid, threads, 0, stream, static_cast<const uint16_t*>(input),
                                route_to_sorted, sorted_routes, sorted_experts, expert_offsets, packed, scales, routes, routes_per_row,
                                slots_per_cta, in_features, scale_tile_bytes);
    return launch_dependent(moe_quantize_routes_mxfp4_kernel<float>, grid, threads, 0, stream, static_cast<const float*>(input), route_to_sorted,
                            sorted_routes, sorted_experts, expert_offsets, packed, scales, routes, routes_per_row, slots_per_cta, in_features,
                            scale_tile_bytes);
}

}  // extern "C"
