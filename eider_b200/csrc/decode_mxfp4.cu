// W4A16 product of MXFP4 weights for few tokens: y[t][n] = sum_k x[t][k] * w[n][k] (+ beta * C), the weights streamed once for 16 tokens.  This
// is the form for a handful of tokens and for every K that is a multiple of 32; takes_terms says which calls go to the other.
//
// Bound: HBM, N * K * 17/32 bytes of weights.  A CTA of eight warps has 16 or 32 rows and their whole K, so nothing leaves a CTA but its
// results: no partial sums, the same order of additions in every run.
//  * A warp has every eighth step of 128 elements of the CTA's rows, which it copies (cp.async) into a ring of its own: warps never
//    wait for each other.  Scales and the first steps are requested before the launch in front is awaited; three CTAs an SM have
//    up to 190 KB on their way.
//  * 16 rows x 32 elements (a block) at a time go through mma.m16n8k16 with the tokens as the eight columns.  E2M1 codes become f16 by
//    one conversion per pair (exact), the sum of a block (two MMAs) is taken in f32 and then added times its two block scales in f32, so
//    the weights are never multiplied out and no MMA chain is longer than a block.
//  * x is made f16 by a launch of its own (prepare_mxfp4_kernel), which runs while the weights are on their way.  Made in the loop, with a
//    maximum, two shuffles and a vote a step in front of the MMAs, the product took 13.2 us for one token and 16.6 for eight
//    (K 5120 -> N 13824), with eight warps or sixteen.
//  * The warps' sums over K meet in shared memory, in warp order.
#include <algorithm>
#include <atomic>
#include <new>

#include "gemm_launch.cuh"
#include "decode_mxfp4.cuh"
#include "mx_block.cuh"
#include "quant_block.cuh"
#include "eider_b200.h"

namespace eider {
namespace decode_mx {

constexpr uint32_t kWarps = 8;
constexpr uint32_t kStepBytes = 64, kStepBlocks = 4;  // of a row: 128 elements
constexpr uint32_t kMaxDepth = 8;                     // steps a warp has on their way
constexpr uint32_t kSmemMost = 227 * 1024;
// Three CTAs an SM (80 registers), two (128) where the activations of a step take 64 of them.
__host__ __device__ constexpr uint32_t ctas_per_sm(int operands) { return operands > 2 ? 2 : 3; }
constexpr uint32_t kFull = 0xffffffffu;

struct Params {
    const uint16_t* x;         // prepared: f16 [tokens * terms][k]
    const uint32_t* x_scales;  // [steps][x_scale_tokens]: a step's four scale bytes, of this launch's tokens
    const uint8_t* w;          // [n][k / 2]
    const uint8_t* scales;     // [n][pitch]
    void* out;
    const void* c;
    float beta;
    int out_is_bf16;
    uint32_t tokens, n, k, pitch, depth, x_scale_tokens;
};

__host__ __device__ constexpr uint32_t reduce_pitch(uint32_t tiles) { return tiles * 16 + 4; }  // (rows of a token; + 4: the fragments' stores meet no bank twice)

// 16 bytes into shared memory, zeros if not `live`.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}
// All but the newest `pending` groups of copies are there.
__device__ __forceinline__ void wait_copies(uint32_t pending) {
    switch (pending) {
        case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
        case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
        case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
        case 3: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
        case 4: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
        case 5: asm volatile("cp.async.wait_group 5;" ::: "memory"); break;
        case 6: asm volatile("cp.async.wait_group 6;" ::: "memory"); break;
        case 7: asm volatile("cp.async.wait_group 7;" ::: "memory"); break;
        default: asm volatile("cp.async.wait_group 8;" ::: "memory"); break;
    }
}
// Rows are 64 bytes: piece c of row r lies at c ^ swizzle(r), so that eight rows' equal pieces fall on different banks.
__device__ __forceinline__ uint32_t swizzle(uint32_t row) { return row >> 1 & 3; }

__device__ __forceinline__ void e2m1_f16(uint32_t w, uint32_t (&p)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(p[0]), "=r"(p[1]), "=r"(p[2]), "=r"(p[3])
        : "r"(w));
}
template <bool FIRST>
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (FIRST)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 f16x2_values(uint32_t v) {
    float2 f;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(f.x), "=f"(f.y) : "r"(v));
    return f;
}
__device__ __forceinline__ uint32_t lds32(uint32_t address) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(address));
    return v;
}

// 2^(c - 127) of byte `I` of a word.  255 gives an infinity here: a row with such a scale comes out infinite or NaN and is looked at
// again at the end.
template <int I> __device__ __forceinline__ float scale_of(uint32_t word) {
    const uint32_t field = (I < 3 ? word << (23 - 8 * I) : word >> 1) & 0x7f800000u;
    return __uint_as_float(max(field, 0x00400000u));
}

// ... of an activation's byte, which is 1 to 240
template <int I> __device__ __forceinline__ float x_scale_of(uint32_t word) {
    return __uint_as_float((I < 3 ? word << (23 - 8 * I) : word >> 1) & 0x7f800000u);
}

template <int N, typename F> __device__ __forceinline__ void static_for(F f) {
    if constexpr (N > 0) {
        static_for<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}
__device__ __forceinline__ uint32_t lds8(uint32_t address) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(address));
    return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t address) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(address));
    return v;
}
// (Activations are read with __ldca or __ldcg: to the compiler __ldg has no order with griddepcontrol.wait, and it requested what the launch in
// front had not written yet: 264 of 3200 calls came out wrong.)
// Eight consecutive elements of a token, their largest finite magnitude, and f16 terms of x * factor.
template <typename T> struct Raw8;
template <> struct Raw8<uint16_t> {
    uint4 q;
    __device__ __forceinline__ void load(const uint16_t* p, bool live) { q = live ? __ldcg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w; }
    static __device__ __forceinline__ __nv_bfloat162 pair(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(word(i) << 16);
            v[2 * i + 1] = __uint_as_float(word(i) & 0xffff0000u);
        }
    }
    __device__ __forceinline__ float finite() const {
        float v[8], m = 0.0f;
        values(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, finite_abs(v[e]));
        return m;
    }
    // (the factor is a power of two: the product is exact in bf16 but far below anything that counts)
    __device__ __forceinline__ void terms(float factor, uint32_t (&t)[1][4]) const {
        const __nv_bfloat162 f = __float2bfloat162_rn(factor);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 p = __hmul2(pair(word(i)), f);
            const uint32_t w = *reinterpret_cast<const uint32_t*>(&p);
            t[0][i] = f16x2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
        }
    }
};
template <> struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p, bool live) {
        a = live ? __ldcg(reinterpret_cast<const float4*>(p)) : make_float4(0, 0, 0, 0);
        b = live ? __ldcg(reinterpret_cast<const float4*>(p) + 1) : make_float4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    __device__ __forceinline__ float finite() const {
        float v[8], m = 0.0f;
        values(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, finite_abs(v[e]));
        return m;
    }
    __device__ __forceinline__ void terms(float factor, uint32_t (&t)[2][4]) const {
        float v[8];
        values(v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float lo = v[2 * i] * factor, hi = v[2 * i + 1] * factor;
            t[0][i] = f16x2(lo, hi);
            const float2 first = f16x2_values(t[0][i]);
            // (of an infinity or NaN the first term is all there is)
            t[1][i] = f16x2(fabsf(first.x) < INFINITY ? lo - first.x : 0.0f, fabsf(first.y) < INFINITY ? hi - first.y : 0.0f);
        }
    }
};

// x as f16: every block of 32 times the power of two that brings its largest finite element to 2^14..2^15 (bf16's eight bits fit, f32 goes
// as two terms, row 2 * token and the next), and the inverse as a scale byte.  bf16 elements keep all their bits within 2^31 of the largest
// of their block, and 2^-39 of that one else.  Sixteen lanes a step of 128 elements, whose four scale bytes are a word, 1 behind the blocks.
constexpr uint32_t kPrepareThreads = 256;
template <typename XT>
__global__ void __launch_bounds__(kPrepareThreads) prepare_mxfp4_kernel(const XT* __restrict__ x, uint16_t* __restrict__ prepared, uint32_t* __restrict__ x_scales,
                                                                        uint32_t k, uint32_t steps, uint32_t x_scale_tokens) {
    constexpr uint32_t kTerms = sizeof(XT) == 4 ? 2 : 1;
    umma::griddep_launch_dependents();
    const uint32_t token = blockIdx.y, lane16 = threadIdx.x % 16, step = blockIdx.x * (kPrepareThreads / 16) + threadIdx.x / 16;
    const uint32_t at = step * 128 + lane16 * 8;
    umma::griddep_wait();
    Raw8<XT> v;
    v.load(x + static_cast<size_t>(token) * k + at, at < k);
    uint32_t largest = __float_as_uint(v.finite());
    largest = max(largest, __shfl_xor_sync(kFull, largest, 1));
    largest = max(largest, __shfl_xor_sync(kFull, largest, 2));
    // 2^(14 - floor(log2 amax)), at most 2^126, and its inverse's byte, 1 at least; an all-zero block keeps 1
    const uint32_t field = largest == 0 ? 127u : min(253u, 268u - (largest >> 23));
    uint32_t word = (at < k ? 254u - field : 1u) << (lane16 / 4 * 8);
    word |= __shfl_xor_sync(kFull, word, 4);
    word |= __shfl_xor_sync(kFull, word, 8);
    if (lane16 == 0 && step < steps) x_scales[step * x_scale_tokens + token] = word;
    if (at < k) {
        uint32_t t[kTerms][4];
        v.terms(__uint_as_float(field << 23), t);
        uint16_t* out = prepared + static_cast<size_t>(token) * kTerms * k + at;
#pragma unroll
        for (uint32_t i = 0; i < kTerms; ++i) *reinterpret_cast<uint4*>(out + i * k) = make_uint4(t[i][0], t[i][1], t[i][2], t[i][3]);
    }
}

// A result whose sum came out infinite or NaN, added up again in 64 bits: parts of a sum, or the product of an activation's and a weight's
// scale, overflow where the result does not, and a NaN scale counts as an infinity in the loop.
__device__ __noinline__ float add_again(const Params& p, uint32_t terms, uint32_t token, uint32_t row, const uint8_t* scales) {
    double sum = 0.0;
    for (uint32_t block = 0; block < p.k / mx::kBlock; ++block) {
        if (scales[block] == mx::kNanCode) return NAN;
        float part = 0.0f;
        for (uint32_t k = block * mx::kBlock; k < (block + 1) * mx::kBlock; ++k) {
            float x = 0.0f;
            for (uint32_t term = 0; term < terms; ++term) x += f16x2_values(__ldcg(p.x + (static_cast<size_t>(token) * terms + term) * p.k + k)).x;
            const uint32_t code = p.w[static_cast<size_t>(row) * (p.k / 2) + k / 2] >> (k % 2 * 4) & 15, m = code & 7;
            const float w = m < 4 ? 0.5f * m : m == 7 ? 6.0f : m - 2.0f;
            part = fmaf(x, code & 8 ? -w : w, part);
        }
        const uint32_t x_scale = __ldcg(p.x_scales + block / kStepBlocks * p.x_scale_tokens + token) >> (block % kStepBlocks * 8) & 255;
        sum += ldexp(static_cast<double>(part), static_cast<int>(x_scale + scales[block]) - 254);
    }
    return static_cast<float>(sum);
}

// TILES: 16-row MMA tiles of a CTA.
// SPREAD: consecutive blocks that take an MMA column each.  Few tokens leave most of the eight columns empty, so block j of SPREAD goes
// through column j of its token alone: the MMAs of SPREAD blocks add up in one accumulator, whose columns then get their block
// scales in one go.  SPLIT_TERMS: the two f16 terms of f32 are columns too (up to four tokens).  Else TERMS 2: MMAs of the same weights.
// COLS: groups of eight columns.
template <int TILES, int SPREAD, int TERMS, bool SPLIT_TERMS, int COLS>
__global__ void __launch_bounds__(32 * kWarps, ctas_per_sm(TERMS * COLS)) decode_mxfp4_kernel(const __grid_constant__ Params p) {
    constexpr int kSpan = SPREAD * (SPLIT_TERMS ? 2 : 1);  // columns of a token
    constexpr int kTokens = 8 * COLS / kSpan;
    constexpr int kGroups = kStepBlocks / SPREAD;
    constexpr uint32_t kRows = TILES * 16, kStage = kRows * kStepBytes;
    static_assert(COLS == 1 || kSpan == 1, "columns are spread within one group of eight");
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* scales = smem;                                  // [rows][pitch]
    uint8_t* ring = smem + kRows * p.pitch;                  // [warps][depth][rows][64 bytes], 16-byte pieces swizzled
    float* sums = reinterpret_cast<float*>(ring);            // [warps][tokens][rows], once the ring is done with
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t row0 = blockIdx.x * kRows, rows = min(kRows, p.n - row0);
    const uint32_t blocks = p.k / mx::kBlock, row_bytes = p.k / 2, steps = (p.k + 127) / 128;
    umma::griddep_launch_dependents();

    // Scales of all steps, and the first steps of weights, before the launch in front is awaited.
    for (uint32_t q = threadIdx.x; q < kRows * p.pitch / 16; q += 32 * kWarps) {
        const uint32_t row = q / (p.pitch / 16);
        copy16(umma::smem_u32(scales) + q * 16, p.scales + static_cast<size_t>(row0) * p.pitch + (row < rows ? q * 16 : 0), row < rows);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    // this lane's 16-byte pieces of a step: piece lane % 4 of rows lane / 4, + 8, ..
    const uint8_t* w = p.w + static_cast<size_t>(row0) * row_bytes + t * 16;
    const uint32_t mine = umma::smem_u32(ring) + warp * p.depth * kStage;
    auto fetch = [&](uint32_t step, uint32_t slot) {
        if (step < steps) {
            const bool inside = step * kStepBytes + t * 16 < row_bytes;
#pragma unroll
            for (uint32_t r = 0; r < kRows; r += 8) {
                const bool live = inside && g + r < rows;
                copy16(mine + slot * kStage + (g + r) * kStepBytes + ((t ^ swizzle(g + r)) << 4), live ? w + static_cast<size_t>(g + r) * row_bytes + step * kStepBytes : p.w, live);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");  // (a group for every turn, empty ones too)
    };
    for (uint32_t i = 0; i < p.depth; ++i) fetch(warp + i * kWarps, i);

    umma::griddep_wait();
    const uint32_t sub = g % SPREAD;  // this lane's block of SPREAD
    bool live[COLS];
    const uint16_t* x[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
        const uint32_t column = c * 8 + g;
        live[c] = column / kSpan < p.tokens;
        x[c] = p.x + (live[c] ? static_cast<size_t>(TERMS == 2 ? 2 * column : column / SPREAD) * p.k : 0) + sub * mx::kBlock + t * 8;
    }
    f32x2 acc[TILES][COLS][2];
#pragma unroll
    for (int u = 0; u < TILES; ++u)
#pragma unroll
        for (int c = 0; c < COLS; ++c) acc[u][c][0] = acc[u][c][1] = pack2(0.0f, 0.0f);
    const uint32_t scale_row = umma::smem_u32(scales) + g * p.pitch;

    // x of a step's group of blocks; a group's registers are refilled for the warp's next step as soon as its MMAs are out, unless
    // they are so many that this spills (5 float32 tokens, K 4064 -> N 6150: 13.7 us with two CTAs an SM, requested at the step's begin 10.2 with three)
    constexpr bool kRefill = COLS * TERMS == 1;
    uint4 b[kGroups][COLS][TERMS];
    auto load_x = [&](uint4(&to)[COLS][TERMS], uint32_t block) {
#pragma unroll
        for (int c = 0; c < COLS; ++c)
#pragma unroll
            for (int k = 0; k < TERMS; ++k)
                to[c][k] = live[c] && block + sub < blocks ? __ldca(reinterpret_cast<const uint4*>(x[c] + block * mx::kBlock + k * p.k)) : make_uint4(0, 0, 0, 0);
    };
    // scale bytes of a step for this thread's columns 2t and 2t + 1, from the first of its blocks on
    constexpr int kScaleWords = kSpan == 1 ? 2 : 1;
    uint32_t xs[COLS][kScaleWords];
    auto load_scales = [&](uint32_t step) {
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            const uint32_t token = kSpan == 1 ? c * 8 + 2 * t : 2 * t / kSpan;
            const bool some = token < p.tokens && step < steps;
            const uint32_t* at = p.x_scales + step * p.x_scale_tokens + token;
            if constexpr (kSpan == 1) {  // (pairs of tokens are 8-byte aligned; one behind the last is nobody's)
                const uint2 pair = some ? __ldca(reinterpret_cast<const uint2*>(at)) : make_uint2(0x01010101u, 0x01010101u);
                xs[c][0] = pair.x;
                xs[c][1] = pair.y;
            } else {
                xs[c][0] = (some ? __ldca(at) : 0x01010101u) >> (2 * t % SPREAD * 8);
            }
        }
    };
    if constexpr (kRefill) {
#pragma unroll
        for (int s = 0; s < kGroups; ++s) load_x(b[s], warp * kStepBlocks + s * SPREAD);
        load_scales(warp);
    }

    wait_copies(p.depth);
    __syncthreads();  // the scales are all warps'
    uint32_t slot = 0;
    for (uint32_t step = warp; step < steps; step += kWarps) {
        const uint32_t block0 = step * kStepBlocks;
        if constexpr (!kRefill) {
#pragma unroll
            for (int s = 0; s < kGroups; ++s) load_x(b[s], block0 + s * SPREAD);
            load_scales(step);
        }
        wait_copies(p.depth - 1);
        __syncwarp();
        const uint32_t tile = mine + slot * kStage + g * kStepBytes + t * 4;
        static_for<kGroups>([&](auto which) {
            constexpr int s = decltype(which)::value;
            float d[TILES][COLS][4];
#pragma unroll
            for (int in = 0; in < SPREAD; ++in) {
                const uint32_t at = ((s * SPREAD + in) ^ swizzle(g)) << 4;  // (rows 8 apart are swizzled alike)
#pragma unroll
                for (int u = 0; u < TILES; ++u) {
                    uint32_t lo[4], hi[4];
                    e2m1_f16(lds32(tile + at + u * 16 * kStepBytes), lo);
                    e2m1_f16(lds32(tile + at + (u * 16 + 8) * kStepBytes), hi);
#pragma unroll
                    for (int c = 0; c < COLS; ++c)
#pragma unroll
                        for (int k = 0; k < TERMS; ++k) {
                            const bool take = SPREAD == 1 || sub == static_cast<uint32_t>(in);
                            const uint32_t x0 = take ? b[s][c][k].x : 0u, x1 = take ? b[s][c][k].y : 0u, x2 = take ? b[s][c][k].z : 0u, x3 = take ? b[s][c][k].w : 0u;
                            if (in == 0 && k == 0) mma_f16<true>(d[u][c], lo[0], hi[0], lo[1], hi[1], x0, x1);
                            else mma_f16<false>(d[u][c], lo[0], hi[0], lo[1], hi[1], x0, x1);
                            mma_f16<false>(d[u][c], lo[2], hi[2], lo[3], hi[3], x2, x3);
                        }
                }
            }
            if constexpr (kRefill) load_x(b[s], block0 + kWarps * kStepBlocks + s * SPREAD);
            // this thread's columns 2t and 2t + 1 are neighbouring blocks of a token (or the same block of two)
            const uint32_t scale_at = scale_row + block0 + s * SPREAD + (2 * t) % SPREAD;
#pragma unroll
            for (int u = 0; u < TILES; ++u) {
                const uint32_t lo = SPREAD == 1 ? lds8(scale_at + u * 16 * p.pitch) : lds16(scale_at + u * 16 * p.pitch);
                const uint32_t hi = SPREAD == 1 ? lds8(scale_at + (u * 16 + 8) * p.pitch) : lds16(scale_at + (u * 16 + 8) * p.pitch);
                const f32x2 low = pack2(scale_of<0>(lo), SPREAD == 1 ? scale_of<0>(lo) : scale_of<1>(lo));
                const f32x2 high = pack2(scale_of<0>(hi), SPREAD == 1 ? scale_of<0>(hi) : scale_of<1>(hi));
#pragma unroll
                for (int c = 0; c < COLS; ++c) {
                    // (scales first: their product is exact but beyond f32's range, and d is 2^24 at most)
                    constexpr int kSecond = SPREAD == 1 ? s : s * SPREAD + 1;
                    const f32x2 x = pack2(x_scale_of<s * SPREAD>(xs[c][0]), x_scale_of<kSecond>(xs[c][kScaleWords - 1]));
                    acc[u][c][0] = fma2(pack2(d[u][c][0], d[u][c][1]), mul2(low, x), acc[u][c][0]);
                    acc[u][c][1] = fma2(pack2(d[u][c][2], d[u][c][3]), mul2(high, x), acc[u][c][1]);
                }
            }
        });
        if constexpr (kRefill) load_scales(step + kWarps);
        __syncwarp();  // the slot has been read
        fetch(step + p.depth * kWarps, slot);
        slot = slot + 1 == p.depth ? 0 : slot + 1;
    }

    // ---------------------------------------------------------------------- the warps' sums meet
    wait_copies(0);
    __syncthreads();
    float* here = sums + warp * kTokens * reduce_pitch(TILES);
#pragma unroll
    for (int u = 0; u < TILES; ++u)
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            const float2 row = unpack2(acc[u][c][0]), below = unpack2(acc[u][c][1]);  // rows g and g + 8
            if constexpr (kSpan == 1) {
                float* to = here + (c * 8 + 2 * t) * reduce_pitch(TILES) + u * 16 + g;
                to[0] = row.x;
                to[reduce_pitch(TILES)] = row.y;
                to[8] = below.x;
                to[reduce_pitch(TILES) + 8] = below.y;
            } else {  // a token's columns
                float lo = row.x + row.y, hi = below.x + below.y;
#pragma unroll
                for (int o = 1; o < kSpan / 2; o *= 2) {
                    lo += __shfl_xor_sync(kFull, lo, o);
                    hi += __shfl_xor_sync(kFull, hi, o);
                }
                if ((2 * t) % kSpan == 0) {
                    here[2 * t / kSpan * reduce_pitch(TILES) + u * 16 + g] = lo;
                    here[2 * t / kSpan * reduce_pitch(TILES) + u * 16 + g + 8] = hi;
                }
            }
        }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < p.tokens * rows; i += 32 * kWarps) {
        const uint32_t token = i / rows, row = i - token * rows;
        float sum = 0.0f;
#pragma unroll
        for (uint32_t v = 0; v < kWarps; ++v) sum += sums[(v * kTokens + token) * reduce_pitch(TILES) + row];
        if (!(fabsf(sum) < INFINITY)) sum = add_again(p, TERMS == 2 || SPLIT_TERMS ? 2 : 1, token, row0 + row, scales + row * p.pitch);
        const size_t index = static_cast<size_t>(token) * p.n + row0 + row;
        if (p.beta != 0.0f)
            sum = fmaf(p.beta, p.out_is_bf16 ? bf16_bits_to_float(static_cast<const uint16_t*>(p.c)[index]) : static_cast<const float*>(p.c)[index], sum);
        if (p.out_is_bf16) static_cast<uint16_t*>(p.out)[index] = float_to_bf16_bits(sum);
        else static_cast<float*>(p.out)[index] = sum;
    }
}

struct Plan {
    uint32_t max_tokens, n, k;
    uint32_t* status;
    gemm::FifoCache<CUtensorMap> maps;
};

// The weights go to the tensor cores as they are (decode_mxfp4_terms.cu) where their layout allows, but for a few tokens and weights that are
// neither long nor many.  us a layer here / there, weights beyond L2 in replayed graphs, bf16 with one, four, five and eight tokens: K 5120 ->
// N 13824 12.3 / 12.6, 13.4 / 13.0, 14.7 / 13.1, 15.2 / 13.6; K 1024 -> N 2048 2.8 / 4.6, 3.1 / 4.9, 3.3 / 4.9, 3.5 / 5.1; K 2048 -> N 1536 3.4 /
// 5.2, 3.7 / 5.4, 4.0 / 5.4, 4.2 / 5.5; K 5120 -> N 5120 8.1 / 7.5, 8.7 / 7.7, 9.1 / 7.8, 9.4 / 7.9.  f32 with one, two, three: K 5120 ->
// N 13824 12.4 / 13.3, 13.5 / 13.2, 14.5 / 13.3; K 1024 -> N 2048 3.0 / 5.2, 3.2 / 5.2, 3.3 / 5.3.  At the other bounds, one and four tokens:
// K 8064 -> N 5120 11.4 / 9.3, 12.8 / 9.4, K 8192 11.4 / 9.4, 13.0 / 9.6; K 5120 -> N 26112 22.0 / 17.8, 24.1 / 18.5, N 27648 22.2 / 18.0, 24.4 /
// 18.7.  So the bound on tokens is where the larger layers turn and the small ones have not; layers of 25 million weights and more would
// turn at one token.  More tokens: K 5120 -> N 13824 sixteen 19.8 / 13.8, 48 in three launches 50.6 / 21.7; K 13824 -> N 5120 48 73 / 19.4.
constexpr uint32_t kFewTokens = 4, kLongK = 8192;
constexpr uint64_t kManyWeights = 1ull << 27;
bool takes_terms(uint32_t tokens, uint32_t n, uint32_t k, int input_is_bf16) {
    const bool few = tokens <= (input_is_bf16 ? kFewTokens : kFewTokens / 2) && k < kLongK && static_cast<uint64_t>(n) * k < kManyWeights;
    return !few && k % 128 == 0 && n <= 65535u * 128;
}

template <int TILES, int SPREAD, int TERMS, bool SPLIT_TERMS, int COLS> cudaError_t launch(Params p, cudaStream_t stream) {
    auto kernel = decode_mxfp4_kernel<TILES, SPREAD, TERMS, SPLIT_TERMS, COLS>;
    constexpr uint32_t kRows = TILES * 16, kStage = kRows * kStepBytes * kWarps;
    constexpr uint32_t kSums = kWarps * (8 * COLS / (SPREAD * (SPLIT_TERMS ? 2 : 1))) * reduce_pitch(TILES) * 4;
    const uint32_t steps = (p.k + 127) / 128, turns = (steps + kWarps - 1) / kWarps, fixed = kRows * p.pitch;
    // as many CTAs an SM as the registers allow while the scales leave room for two stages, else fewer
    uint32_t limit = kSmemMost / ctas_per_sm(TERMS * COLS) - 1024;
    while (fixed + std::max(2 * kStage, kSums) > limit && limit < kSmemMost) limit = std::min(limit * 2, kSmemMost);
    if (fixed + std::max(kStage, kSums) > limit) return cudaErrorInvalidValue;
    p.depth = std::max(1u, std::min(std::min(turns, kMaxDepth), (limit - fixed) / kStage));
    static std::atomic<uint8_t> configured[gemm::kMaxDevices];
    if (cudaError_t st = gemm::opt_in_smem(configured, kernel, kSmemMost); st != cudaSuccess) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((p.n + kRows - 1) / kRows);
    cfg.blockDim = dim3(32 * kWarps);
    cfg.dynamicSmemBytes = fixed + std::max(p.depth * kStage, kSums);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}
template <int SPREAD, int TERMS, bool SPLIT_TERMS, int COLS> cudaError_t run(const Params& p, cudaStream_t stream) {
    // 32 rows a CTA share an activation's registers; with fewer than two and a half such CTAs an SM, 16
    return p.n >= 80u * static_cast<uint32_t>(gemm::sm_count()) ? launch<2, SPREAD, TERMS, SPLIT_TERMS, COLS>(p, stream)
                                                               : launch<1, SPREAD, TERMS, SPLIT_TERMS, COLS>(p, stream);
}
cudaError_t run_tokens(const Params& p, bool bf16, cudaStream_t stream) {
    const uint32_t tokens = p.tokens;
    if (bf16)
        return tokens <= 2   ? run<4, 1, false, 1>(p, stream)
               : tokens <= 4 ? run<2, 1, false, 1>(p, stream)
               : tokens <= 8 ? run<1, 1, false, 1>(p, stream)
                             : run<1, 1, false, 2>(p, stream);
    return tokens == 1   ? run<4, 1, true, 1>(p, stream)
           : tokens == 2 ? run<2, 1, true, 1>(p, stream)
           : tokens <= 4 ? run<1, 1, true, 1>(p, stream)
           : tokens <= 8 ? run<1, 2, false, 1>(p, stream)
                         : run<1, 2, false, 2>(p, stream);
}
uint32_t steps_of(uint32_t k) { return (k + 127) / 128; }
uint32_t x_scale_tokens(uint32_t tokens) { return (tokens + 1) / 2 * 2; }
size_t x_scale_bytes(uint32_t tokens, uint32_t k) { return (static_cast<size_t>(x_scale_tokens(tokens)) * steps_of(k) * sizeof(uint32_t) + 127) / 128 * 128; }
template <typename XT>
cudaError_t prepare(const void* x, uint16_t* prepared, uint32_t* x_scales, uint32_t tokens, uint32_t k, cudaStream_t stream) {
    const uint32_t steps = steps_of(k);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((steps + kPrepareThreads / 16 - 1) / (kPrepareThreads / 16), tokens);
    cfg.blockDim = dim3(kPrepareThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, prepare_mxfp4_kernel<XT>, static_cast<const XT*>(x), prepared, x_scales, k, steps, x_scale_tokens(tokens));
}

}  // namespace decode_mx
}  // namespace eider

using namespace eider;

extern "C" {

void* eider_b200_mxfp4_decode_create(uint32_t max_tokens, uint32_t out_features, uint32_t in_features) {
    if (max_tokens == 0 || max_tokens > 64 || out_features == 0 || in_features == 0 || in_features % mx::kBlock != 0 || in_features > 65536) return nullptr;
    auto* plan = new (std::nothrow) decode_mx::Plan{max_tokens, out_features, in_features, nullptr, {}};
    if (!plan) return nullptr;
    if (cudaMalloc(reinterpret_cast<void**>(&plan->status), sizeof(uint32_t)) != cudaSuccess) {
        delete plan;
        return nullptr;
    }
    if (cudaMemset(plan->status, 0, sizeof(uint32_t)) != cudaSuccess) {
        eider_b200_mxfp4_decode_destroy(plan);
        return nullptr;
    }
    return plan;
}

void eider_b200_mxfp4_decode_destroy(void* raw) {
    auto* plan = static_cast<decode_mx::Plan*>(raw);
    if (!plan) return;
    cudaFree(plan->status);
    delete plan;
}

cudaError_t eider_b200_mxfp4_decode_status(void* raw, uint32_t* host_status) {
    auto* plan = static_cast<decode_mx::Plan*>(raw);
    if (!plan || !host_status) return cudaErrorInvalidValue;
    return cudaMemcpy(host_status, plan->status, sizeof(uint32_t), cudaMemcpyDeviceToHost);
}

size_t eider_b200_mxfp4_w4a16_workspace_bytes(uint32_t tokens, uint32_t in_features, int input_is_bf16) {
    const size_t few = decode_mx::x_scale_bytes(tokens, in_features) + static_cast<size_t>(tokens) * in_features * (input_is_bf16 ? 2 : 4);
    return in_features % 128 == 0 ? std::max(few, decode_mx::terms_workspace_bytes(tokens, in_features, input_is_bf16)) : few;  // (whichever form it takes)
}

cudaError_t eider_b200_mxfp4_w4a16_gemv_on_stream(void* raw, const void* input, int input_is_bf16, uint32_t tokens, const uint8_t* w_values,
                                                  const uint8_t* w_scales_rows, uint32_t scale_pitch, const uint8_t* w_scales_tiled, const void* c,
                                                  void* d, float beta, int out_is_bf16, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    using namespace decode_mx;
    auto* plan = static_cast<Plan*>(raw);
    if (!plan || !input || !w_values || !w_scales_rows || !w_scales_tiled || !d || tokens == 0 || tokens > plan->max_tokens || (beta != 0.0f && !c)) return cudaErrorInvalidValue;
    if (((reinterpret_cast<uintptr_t>(input) | reinterpret_cast<uintptr_t>(w_values) | reinterpret_cast<uintptr_t>(w_scales_rows) |
          reinterpret_cast<uintptr_t>(w_scales_tiled)) & 15) != 0 ||
        !workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
        workspace_bytes < eider_b200_mxfp4_w4a16_workspace_bytes(tokens, plan->k, input_is_bf16) || scale_pitch % 16 != 0 || scale_pitch < (plan->k / mx::kBlock + 7) / 8 * 8)
        return cudaErrorInvalidValue;
    if (takes_terms(tokens, plan->n, plan->k, input_is_bf16) && (reinterpret_cast<uintptr_t>(w_values) & 31) == 0)
        return run_terms(plan->maps, input, input_is_bf16, tokens, w_values, w_scales_tiled, c, d, beta, out_is_bf16, plan->n, plan->k,
                         static_cast<uint8_t*>(workspace), plan->status, stream);
    uint32_t* x_scales = static_cast<uint32_t*>(workspace);
    uint16_t* prepared = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(workspace) + x_scale_bytes(tokens, plan->k));
    cudaError_t st = input_is_bf16 ? prepare<uint16_t>(input, prepared, x_scales, tokens, plan->k, stream)
                                   : prepare<float>(input, prepared, x_scales, tokens, plan->k, stream);
    if (st != cudaSuccess) return st;
    // (an even number: the scales of a launch's tokens come in aligned pairs)
    const uint32_t groups = (tokens + 15) / 16, each = groups == 1 ? tokens : ((tokens + groups - 1) / groups + 1) / 2 * 2;
    for (uint32_t first = 0; first < tokens; first += each) {
        const size_t out_bytes = out_is_bf16 ? 2 : 4;
        Params p{};
        p.tokens = std::min(each, tokens - first);
        p.x = prepared + static_cast<size_t>(first) * (input_is_bf16 ? 1 : 2) * plan->k;
        p.x_scales = x_scales + first;
        p.x_scale_tokens = x_scale_tokens(tokens);
        p.w = w_values;
        p.scales = w_scales_rows;
        p.out = static_cast<uint8_t*>(d) + first * out_bytes * plan->n;
        p.c = c ? static_cast<const uint8_t*>(c) + first * out_bytes * plan->n : nullptr;
        p.beta = beta;
        p.out_is_bf16 = out_is_bf16;
        p.n = plan->n;
        p.k = plan->k;
        p.pitch = scale_pitch;
        st = run_tokens(p, input_is_bf16, stream);
        if (st != cudaSuccess) return st;
    }
    return cudaSuccess;
}

}  // extern "C"
