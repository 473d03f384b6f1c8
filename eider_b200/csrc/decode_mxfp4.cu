// W4A16 product of MXFP4 weights for few tokens: y[t][n] = sum_k x[t][k] * w[n][k] (+ beta * C), the weights streamed once.
//
// Bound: HBM, N * K * 17/32 bytes of weights.  Every SM has one CTA with N / 148 rows of its own for the whole K (as many passes as rows do
// not fit), so that all of them stream the same number of bytes whatever N is: one launch, no workspace, the same order of
// additions in every run.  A CTA takes half of an SM, so that the next launch's is resident beside it, with its barriers set up and its
// first hundred kilobytes of weights on their way, when this one ends.
//  * A producer warp streams the rows in chunks of 256 elements (TMA boxes of 128 bytes x rows, 128-byte swizzle) through a ring of
//    shared memory; weights and scales are requested before the launch in front is awaited.
//  * A chunk is one warp's, for all of the CTA's rows: 16 rows x 32 elements (a block) at a time through mma.m16n8k16 with the tokens
//    as the eight columns.  E2M1 codes become f16 by one conversion per pair (exact), the sum of a block (two MMAs) is taken in f32 and
//    then added times its block scale in f32, so the weights are never multiplied out and no MMA chain is longer than a block.
//  * x becomes f16 by a power of two per token and warp that brings its largest element so far to 2^8..2^9 (it grows to 2^15 before the
//    sums are rescaled): bf16's eight bits fit, f32 goes as two f16 terms.  What is lost lies 2^-33 below the largest element.
//  * The warps' sums over K meet in shared memory, in warp order.
#include <algorithm>
#include <atomic>
#include <new>

#include "gemm_launch.cuh"
#include "tensor_maps.cuh"
#include "mx_block.cuh"
#include "eider_b200.h"

namespace eider {
namespace decode_mx {

constexpr uint32_t kChunkBytes = 128;               // 256 elements of a row
constexpr uint32_t kChunkBlocks = 8;
constexpr uint32_t kMaxWarps = 7;                   // consumer warps; the producer is the eighth
constexpr uint32_t kMaxTiles = 3;                   // 16-row MMA tiles of a CTA in a pass
// Half of an SM: one CTA of this launch and one of the next.
constexpr uint32_t kSmemLimit = 113 * 1024;
constexpr uint32_t kMaxSlots = 32;
constexpr uint32_t kFull = 0xffffffffu;

struct Params {
    const void* x;
    const uint8_t* scales;  // [n][pitch]
    void* out;
    const void* c;
    uint32_t* status;
    float beta;
    int out_is_bf16;
    uint32_t tokens, n, k, pitch;
    uint32_t rows;    // of a CTA in a pass
    uint32_t passes, chunks, warps;
    uint32_t depth;   // ring slots of a warp
};

__host__ __device__ constexpr uint32_t reduce_pitch(uint32_t tiles) { return tiles * 16 + 4; }  // (rows of a token; + 4: the fragments' stores meet no bank twice)
__host__ __device__ constexpr uint32_t slot_bytes(uint32_t tiles) { return tiles * 16 * kChunkBytes; }
inline uint32_t fixed_bytes(uint32_t tiles, uint32_t warps, uint32_t tokens, uint32_t pitch, uint32_t passes) {
    return 1024 /*alignment*/ + (passes > 1 ? 2 : 1) * tiles * 16 * pitch + warps * tokens * reduce_pitch(tiles) * 4 + (2 * kMaxSlots + 4) * 8 + 16;
}

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

__device__ __forceinline__ uint32_t lds16(uint32_t address) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(address));
    return v;
}
template <int N, typename F> __device__ __forceinline__ void static_for(F f) {
    if constexpr (N > 0) {
        static_for<N - 1>(f);
        f(std::integral_constant<int, N - 1>{});
    }
}

// Eight consecutive elements of a token, and what becomes of them: the largest finite magnitude, and f16 terms of x * factor.
template <typename T> struct Raw8;
template <> struct Raw8<uint16_t> {
    uint4 q;
    __device__ __forceinline__ void load(const uint16_t* p, bool live) { q = live ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w; }
    static __device__ __forceinline__ __nv_bfloat162 pair(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
    __device__ __forceinline__ float amax() const {
        const __nv_bfloat162 m = __hmax2(__hmax2(__habs2(pair(q.x)), __habs2(pair(q.y))), __hmax2(__habs2(pair(q.z)), __habs2(pair(q.w))));
        return fmaxf(__low2float(m), __high2float(m));
    }
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
        a = live ? __ldg(reinterpret_cast<const float4*>(p)) : make_float4(0, 0, 0, 0);
        b = live ? __ldg(reinterpret_cast<const float4*>(p) + 1) : make_float4(0, 0, 0, 0);
    }
    __device__ __forceinline__ float amax() const {
        return fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))), fmaxf(fmaxf(fabsf(b.x), fabsf(b.y)), fmaxf(fabsf(b.z), fabsf(b.w))));
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

// TILES: 16-row MMA tiles of a CTA's rows.  COLS: groups of eight MMA columns.
// SPREAD: consecutive blocks that take an MMA column each (with COLS 1).  Few tokens leave most of the eight columns empty, so block j
// of SPREAD goes through column j of its token alone: the MMAs of SPREAD blocks add up in one accumulator, whose columns then get
// their block scales in one go, and every lane converts the activations of one block instead of all of them.  About 18
// instructions for 16 x 32 weights at SPREAD 8 against 34 at 1.  SPLIT_TERMS: the two f16 terms of f32 are columns too (up to four
// tokens) instead of MMAs of their own.
template <int TILES, int COLS, int SPREAD, bool SPLIT_TERMS, typename XT>
__global__ void __launch_bounds__(32 * (kMaxWarps + 1), 2) decode_mxfp4_kernel(const __grid_constant__ CUtensorMap map_w, const Params p) {
    constexpr int kTerms = sizeof(XT) == 4 && !SPLIT_TERMS ? 2 : 1;      // MMAs of the same weights
    constexpr int kSpan = SPREAD * (SPLIT_TERMS ? 2 : 1);                // columns of a token
    constexpr uint32_t kStepBlocks = SPREAD == 8 ? 8 : 4;                // blocks of a warp's step
    constexpr uint32_t kSteps = kChunkBlocks / kStepBlocks;              // steps of a chunk
    constexpr int kStep = COLS * kTerms >= 4 ? 1 : 4 / (COLS * kTerms);  // blocks of x that a warp holds (and has on their way) at a time, COLS > 1
    constexpr int kGroups = kStepBlocks / SPREAD;                        // the same for COLS 1: a block of each of these groups
    constexpr int kAhead = SPREAD == 8 || (SPREAD == 4 && sizeof(XT) == 2) ? 4 : SPREAD > 1 ? 2 : 1;  // steps whose x is on its way, COLS 1
    constexpr uint32_t kTokens = 8 / kSpan;                              // of a group of eight columns
    static_assert(COLS == 1 || (SPREAD == 1 && !SPLIT_TERMS), "columns are spread within one group of eight");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const uint32_t scale_bytes = TILES * 16 * p.pitch, slots = p.warps * p.depth;
    uint8_t* scales = ring + slots * slot_bytes(TILES);
    float* sums = reinterpret_cast<float*>(scales + (p.passes > 1 ? 2 : 1) * scale_bytes);  // [warps][kTokens][rows]
    uint64_t* full = reinterpret_cast<uint64_t*>(sums + p.warps * kTokens * reduce_pitch(TILES));  // [slots]
    uint64_t* empty = full + kMaxSlots;                                                           // [slots]
    uint64_t* scales_full = empty + kMaxSlots;                                                    // [2]
    uint64_t* scales_empty = scales_full + 2;                                                     // [2]
    volatile uint32_t* abort_flag = reinterpret_cast<uint32_t*>(scales_empty + 2);

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < slots; ++i) {
            umma::mbar_init(&full[i], 1);
            umma::mbar_init(&empty[i], 1);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            umma::mbar_init(&scales_full[i], 1);
            umma::mbar_init(&scales_empty[i], p.warps);
        }
        *abort_flag = 0;
        umma::fence_barrier_init();
        umma::prefetch_tensormap(&map_w);
    }
    __syncthreads();
    umma::griddep_launch_dependents();

    // Chunk i (counted through the passes) is warp i % warps' alone, in one of that warp's own slots.  So a warp sees every filling of a
    // slot that it waits on, and a parity can only mean the filling before or the one it waits for.  (In a ring that all warps share a
    // warp could come to a slot a lap ahead of a copy that lands late, and take the parity of the lap before for its own.)
    auto slot_of = [&](uint32_t i) { return i % p.warps * p.depth + i / p.warps % p.depth; };
    auto phase_of = [&](uint32_t i) { return i / slots & 1; };

    if (warp == p.warps) {
        // ------------------------------------------------------------------ producer
        if (lane == 0) {
            uint32_t i = 0, pass = 0;
            bool ok = true;
            for (; ok && pass < p.passes; ++pass) {
                const uint32_t row0 = (pass * gridDim.x + blockIdx.x) * p.rows;
                if (row0 >= p.n) break;
                const uint32_t buffer = pass & 1;
                if (!umma::mbar_wait(&scales_empty[buffer], ((pass >> 1) & 1) ^ 1, abort_flag, p.status, umma::kTimeoutEmpty)) break;  // (pass: those begun)
                const uint32_t bytes = min(p.rows, p.n - row0) * p.pitch;
                umma::mbar_arrive_expect_tx(&scales_full[buffer], bytes);
                umma::bulk_load_1d(scales + buffer * scale_bytes, p.scales + static_cast<size_t>(row0) * p.pitch, bytes, &scales_full[buffer]);
                for (uint32_t c = 0; c < p.chunks; ++c, ++i) {
                    const uint32_t slot = slot_of(i);
                    if (!umma::mbar_wait(&empty[slot], phase_of(i) ^ 1, abort_flag, p.status, umma::kTimeoutEmpty)) { ok = false; break; }
                    umma::mbar_arrive_expect_tx(&full[slot], p.rows * kChunkBytes);
                    umma::tma_load_2d(ring + slot * slot_bytes(TILES), &map_w, &full[slot], static_cast<int32_t>(c * kChunkBytes), static_cast<int32_t>(row0));
                }
            }
            // The block does not leave before its copies have landed, not even after a wait ran out: bounded too.
            const long long start = clock64();
            auto landed = [&](uint64_t* bar, uint32_t parity) {
                while (!umma::mbar_try_wait(bar, parity) && clock64() - start < umma::kWaitLimitCycles) {}
            };
            for (uint32_t j = i > slots ? i - slots : 0; j < i; ++j) landed(&full[slot_of(j)], phase_of(j));
            for (uint32_t j = pass > 2 ? pass - 2 : 0; j < pass; ++j) landed(&scales_full[j & 1], (j >> 1) & 1);
        }
        return;
    }

    // ---------------------------------------------------------------------- consumers
    const uint32_t g = lane >> 2, t = lane & 3;
    const uint32_t blocks = p.k / mx::kBlock;
    const uint32_t ring_addr = umma::smem_u32(ring), scales_addr = umma::smem_u32(scales);
    umma::griddep_wait();
    const XT* x = static_cast<const XT*>(p.x) + t * 8;
    const uint32_t sub = g % SPREAD;  // this lane's block of SPREAD
    bool live[COLS];
    const XT* x_of[COLS];
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
        const uint32_t token = (n * 8 + g) / kSpan;
        live[n] = token < p.tokens;
        x_of[n] = x + (live[n] ? static_cast<size_t>(token) * p.k : 0) + sub * mx::kBlock;
    }
    bool ok = true;
    for (uint32_t pass = 0; pass < p.passes; ++pass) {
        const uint32_t row0 = (pass * gridDim.x + blockIdx.x) * p.rows;
        if (row0 >= p.n) break;
        float acc[TILES][COLS][4];
#pragma unroll
        for (int u = 0; u < TILES; ++u)
#pragma unroll
            for (int n = 0; n < COLS; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[u][n][i] = 0.0f;
        float factor[COLS];  // what token g of each group is multiplied by, a power of two; 0: nothing but zeros yet
#pragma unroll
        for (int n = 0; n < COLS; ++n) factor[n] = 0.0f;

        // Largest finite magnitude in hand -> whether the column's factor has to change, and what the sums so far change by.
        auto rescale = [&](int n, float amax, auto finite_amax) {
            amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 2));
            if (__any_sync(kFull, factor[n] == 0.0f ? amax != 0.0f : amax * factor[n] >= 32768.0f)) {
                if (__any_sync(kFull, amax == INFINITY)) {  // an infinity goes through as it is; the finite ones set the scale
                    amax = finite_amax();
                    amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 1));
                    amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 2));
                }
                float change = 1.0f;
                if (factor[n] == 0.0f ? amax != 0.0f : amax * factor[n] >= 32768.0f) {
                    const float wanted = __uint_as_float(min(254u, 262u - (__float_as_uint(amax) >> 23)) << 23);  // the largest element to 2^8..2^9
                    // (the sums so far are zero, or change by a power of two; a change too small for f32 leaves nothing of them either way)
                    if (factor[n] != 0.0f) change = __fdiv_rn(wanted, factor[n]);
                    factor[n] = wanted;
                }
                const float c0 = __shfl_sync(kFull, change, t * 8), c1 = __shfl_sync(kFull, change, t * 8 + 4);
#pragma unroll
                for (int u = 0; u < TILES; ++u) {
                    acc[u][n][0] *= c0;
                    acc[u][n][1] *= c1;
                    acc[u][n][2] *= c0;
                    acc[u][n][3] *= c1;
                }
            }
            return factor[n] == 0.0f ? 1.0f : factor[n];
        };
        constexpr int kHeld = COLS == 1 ? kGroups : kStep;
        Raw8<XT> raw[COLS][kHeld], later[kAhead - 1 + (kAhead == 1)][kHeld];  // (`later`: of the steps behind the next, COLS 1)
        auto load_x = [&](uint32_t block) {
#pragma unroll
            for (int n = 0; n < COLS; ++n)
#pragma unroll
                for (int s = 0; s < kHeld; ++s) raw[n][s].load(x_of[n] + (block + s * SPREAD) * mx::kBlock, live[n] && block + s * SPREAD + sub < blocks);
        };
        // this warp's chunks of the pass are first, first + warps, ..; its step q lies at block_at(q) of K (behind the last at or past `blocks`)
        const uint32_t chunk0 = pass * p.chunks, first = (warp + p.warps - chunk0 % p.warps) % p.warps;
        auto block_at = [&](uint32_t q) { return (first + q / kSteps * p.warps) * kChunkBlocks + q % kSteps * kStepBlocks; };
        auto load_later = [&](Raw8<XT>(&to)[kHeld], uint32_t q) {
            const uint32_t block = block_at(q);
#pragma unroll
            for (int s = 0; s < kHeld; ++s) to[s].load(x_of[0] + (block + s * SPREAD) * mx::kBlock, live[0] && block + s * SPREAD + sub < blocks);
        };
        load_x(block_at(0));
        if constexpr (COLS == 1) {
#pragma unroll
            for (int a = 0; a + 1 < kAhead; ++a) load_later(later[a], a + 1);
        }
        if (ok && !umma::mbar_wait(&scales_full[pass & 1], (pass >> 1) & 1, abort_flag, p.status, umma::kTimeoutFull)) ok = false;
        const uint32_t pass_scales = scales_addr + (pass & 1) * scale_bytes + g * p.pitch;
        for (uint32_t q = 0; ok && first + q / kSteps * p.warps < p.chunks; ++q) {
            const uint32_t i = chunk0 + first + q / kSteps * p.warps, slot = slot_of(i);
            const uint32_t block0 = block_at(q);
            const uint32_t tile = ring_addr + slot * slot_bytes(TILES) + g * kChunkBytes + t * 4, half = q % kSteps * kStepBlocks;
            auto arrive = [&] {
                ok = __all_sync(kFull, umma::mbar_wait(&full[slot], phase_of(i), abort_flag, p.status, umma::kTimeoutFull));
                return ok;
            };
            // block `in` of the step: rows of tile u as f16
            auto weights = [&](uint32_t in, int u, uint32_t (&lo)[4], uint32_t (&hi)[4]) {
                const uint32_t at = tile + (((half + in) ^ g) << 4);
                e2m1_f16(lds32(at + u * 16 * kChunkBytes), lo);
                e2m1_f16(lds32(at + (u * 16 + 8) * kChunkBytes), hi);
            };
            if constexpr (COLS == 1) {
                float amax = 0.0f;
#pragma unroll
                for (int s = 0; s < kHeld; ++s) amax = fmaxf(amax, raw[0][s].amax());
                const float f = rescale(0, amax, [&] {
                    float m = 0.0f;
#pragma unroll
                    for (int s = 0; s < kHeld; ++s) m = fmaxf(m, raw[0][s].finite());
                    return m;
                });
                uint32_t b[kHeld][kTerms][4];
#pragma unroll
                for (int s = 0; s < kHeld; ++s) {
                    if constexpr (SPLIT_TERMS) {
                        uint32_t both[2][4];
                        raw[0][s].terms(f, both);
#pragma unroll
                        for (int e = 0; e < 4; ++e) b[s][0][e] = (g / SPREAD) & 1 ? both[1][e] : both[0][e];
                    } else {
                        raw[0][s].terms(f, b[s]);
                    }
                }
                if constexpr (kAhead == 1) {
                    load_later(raw[0], q + 1);
                } else {
#pragma unroll
                    for (int s = 0; s < kHeld; ++s) raw[0][s] = later[0][s];
#pragma unroll
                    for (int a = 0; a + 2 < kAhead; ++a)
#pragma unroll
                        for (int s = 0; s < kHeld; ++s) later[a][s] = later[a + 1][s];
                    load_later(later[kAhead - 2], q + kAhead);
                }
                if (!arrive()) break;
                [[maybe_unused]] uint32_t lo4[TILES], hi4[TILES];
                if constexpr (SPREAD == 1) {
#pragma unroll
                    for (int u = 0; u < TILES; ++u) {
                        lo4[u] = lds32(pass_scales + block0 + u * 16 * p.pitch);
                        hi4[u] = lds32(pass_scales + block0 + (u * 16 + 8) * p.pitch);
                    }
                }
                static_for<kGroups>([&](auto which) {
                    constexpr int s = decltype(which)::value;
                    float d[TILES][4];
#pragma unroll
                    for (int in = 0; in < SPREAD; ++in) {
                        uint32_t m[kTerms][4];
#pragma unroll
                        for (int q = 0; q < kTerms; ++q)
#pragma unroll
                            for (int e = 0; e < 4; ++e) m[q][e] = SPREAD == 1 || sub == static_cast<uint32_t>(in) ? b[s][q][e] : 0u;
#pragma unroll
                        for (int u = 0; u < TILES; ++u) {
                            uint32_t lo[4], hi[4];
                            weights(s * SPREAD + in, u, lo, hi);
                            if (in == 0) mma_f16<true>(d[u], lo[0], hi[0], lo[1], hi[1], m[0][0], m[0][1]);
                            else mma_f16<false>(d[u], lo[0], hi[0], lo[1], hi[1], m[0][0], m[0][1]);
                            mma_f16<false>(d[u], lo[2], hi[2], lo[3], hi[3], m[0][2], m[0][3]);
                            if constexpr (kTerms == 2) {
                                mma_f16<false>(d[u], lo[0], hi[0], lo[1], hi[1], m[kTerms - 1][0], m[kTerms - 1][1]);
                                mma_f16<false>(d[u], lo[2], hi[2], lo[3], hi[3], m[kTerms - 1][2], m[kTerms - 1][3]);
                            }
                        }
                    }
                    // this thread's columns 2t and 2t + 1 are neighbouring blocks of a token (or the same block of two)
#pragma unroll
                    for (int u = 0; u < TILES; ++u) {
                        float lo0, lo1, hi0, hi1;
                        if constexpr (SPREAD == 1) {
                            lo0 = lo1 = scale_of<s>(lo4[u]);
                            hi0 = hi1 = scale_of<s>(hi4[u]);
                        } else {
                            const uint32_t at = pass_scales + block0 + s * SPREAD + (2 * t) % SPREAD;
                            const uint32_t lo2 = lds16(at + u * 16 * p.pitch), hi2 = lds16(at + (u * 16 + 8) * p.pitch);
                            lo0 = scale_of<0>(lo2);
                            lo1 = scale_of<1>(lo2);
                            hi0 = scale_of<0>(hi2);
                            hi1 = scale_of<1>(hi2);
                        }
                        acc[u][0][0] = fmaf(d[u][0], lo0, acc[u][0][0]);
                        acc[u][0][1] = fmaf(d[u][1], lo1, acc[u][0][1]);
                        acc[u][0][2] = fmaf(d[u][2], hi0, acc[u][0][2]);
                        acc[u][0][3] = fmaf(d[u][3], hi1, acc[u][0][3]);
                    }
                });
            } else {
                uint32_t lo4[TILES], hi4[TILES];
                static_for<kStepBlocks / kStep>([&](auto which) {
                    constexpr int step = decltype(which)::value * kStep;
                    if (!ok) return;
                    // this step's x as f16, then the next step's is requested
                    uint32_t b[kStep][COLS][kTerms][4];
#pragma unroll
                    for (int n = 0; n < COLS; ++n) {
                        float amax = 0.0f;
#pragma unroll
                        for (int s = 0; s < kStep; ++s) amax = fmaxf(amax, raw[n][s].amax());
                        const float f = rescale(n, amax, [&] {
                            float m = 0.0f;
#pragma unroll
                            for (int s = 0; s < kStep; ++s) m = fmaxf(m, raw[n][s].finite());
                            return m;
                        });
#pragma unroll
                        for (int s = 0; s < kStep; ++s) raw[n][s].terms(f, b[s][n]);
                    }
                    load_x(step + kStep < static_cast<int>(kStepBlocks) ? block0 + step + kStep : block_at(q + 1));
                    if (step == 0) {
                        if (!arrive()) return;
#pragma unroll
                        for (int u = 0; u < TILES; ++u) {
                            lo4[u] = lds32(pass_scales + block0 + u * 16 * p.pitch);
                            hi4[u] = lds32(pass_scales + block0 + (u * 16 + 8) * p.pitch);
                        }
                    }
                    static_for<kStep>([&](auto in_step) {
                        constexpr int s = decltype(in_step)::value;
#pragma unroll
                        for (int u = 0; u < TILES; ++u) {
                            uint32_t lo[4], hi[4];
                            weights(step + s, u, lo, hi);
                            const float s_lo = scale_of<step + s>(lo4[u]), s_hi = scale_of<step + s>(hi4[u]);
#pragma unroll
                            for (int n = 0; n < COLS; ++n) {
                                float d[4];
                                mma_f16<true>(d, lo[0], hi[0], lo[1], hi[1], b[s][n][0][0], b[s][n][0][1]);
                                mma_f16<false>(d, lo[2], hi[2], lo[3], hi[3], b[s][n][0][2], b[s][n][0][3]);
                                if constexpr (kTerms == 2) {
                                    mma_f16<false>(d, lo[0], hi[0], lo[1], hi[1], b[s][n][kTerms - 1][0], b[s][n][kTerms - 1][1]);
                                    mma_f16<false>(d, lo[2], hi[2], lo[3], hi[3], b[s][n][kTerms - 1][2], b[s][n][kTerms - 1][3]);
                                }
                                acc[u][n][0] = fmaf(d[0], s_lo, acc[u][n][0]);
                                acc[u][n][1] = fmaf(d[1], s_lo, acc[u][n][1]);
                                acc[u][n][2] = fmaf(d[2], s_hi, acc[u][n][2]);
                                acc[u][n][3] = fmaf(d[3], s_hi, acc[u][n][3]);
                            }
                        }
                    });
                });
                if (!ok) break;
            }
            __syncwarp();
            if (ok && lane == 0 && q % kSteps == kSteps - 1) umma::mbar_arrive(&empty[slot]);
        }
        if (lane == 0) umma::mbar_arrive(&scales_empty[pass & 1]);

        // ------------------------------------------------------------------ the warps' sums meet, eight tokens at a time
#pragma unroll
        for (int n = 0; n < COLS; ++n) {
            if (n * 8 >= p.tokens * kSpan) break;
            // (1 / factor, exact: 2^-127 is subnormal)
            const uint32_t field = __float_as_uint(factor[n]) >> 23;
            const float back = factor[n] == 0.0f ? 1.0f : __uint_as_float(field == 254 ? 0x00400000u : (254u - field) << 23);
            const float b0 = __shfl_sync(kFull, back, t * 8), b1 = __shfl_sync(kFull, back, t * 8 + 4);
            float* mine = sums + warp * kTokens * reduce_pitch(TILES);
#pragma unroll
            for (int u = 0; u < TILES; ++u) {
                if constexpr (kSpan == 1) {
                    mine[(2 * t) * reduce_pitch(TILES) + u * 16 + g] = acc[u][n][0] * b0;
                    mine[(2 * t + 1) * reduce_pitch(TILES) + u * 16 + g] = acc[u][n][1] * b1;
                    mine[(2 * t) * reduce_pitch(TILES) + u * 16 + g + 8] = acc[u][n][2] * b0;
                    mine[(2 * t + 1) * reduce_pitch(TILES) + u * 16 + g + 8] = acc[u][n][3] * b1;
                } else {  // a token's columns
                    float lo = acc[u][n][0] * b0 + acc[u][n][1] * b1, hi = acc[u][n][2] * b0 + acc[u][n][3] * b1;
#pragma unroll
                    for (int o = 1; o < kSpan / 2; o *= 2) {
                        lo += __shfl_xor_sync(kFull, lo, o);
                        hi += __shfl_xor_sync(kFull, hi, o);
                    }
                    if ((2 * t) % kSpan == 0) {
                        mine[2 * t / kSpan * reduce_pitch(TILES) + u * 16 + g] = lo;
                        mine[2 * t / kSpan * reduce_pitch(TILES) + u * 16 + g + 8] = hi;
                    }
                }
            }
            asm volatile("bar.sync 1, %0;" ::"r"(p.warps * 32) : "memory");
            const uint32_t tokens = min(kTokens, p.tokens - n * 8), rows = min(p.rows, p.n - row0);
            auto warps_sum = [&](uint32_t token, uint32_t row) {
                float sum = 0.0f;
                for (uint32_t w = 0; w < p.warps; ++w) sum += sums[(w * kTokens + token) * reduce_pitch(TILES) + row];
                return sum;
            };
            for (uint32_t i = threadIdx.x; i < tokens * rows; i += p.warps * 32) {
                const uint32_t token = i / rows, row = i - token * rows;
                float sum = warps_sum(token, row);
                if (!(fabsf(sum) < INFINITY)) {  // a NaN scale among the row's?
                    const uint8_t* s = p.scales + static_cast<size_t>(row0 + row) * p.pitch;
                    for (uint32_t q = 0; q < blocks; ++q)
                        if (s[q] == mx::kNanCode) sum = NAN;
                }
                const size_t index = static_cast<size_t>(n * 8 + token) * p.n + row0 + row;
                if (p.beta != 0.0f)
                    sum = fmaf(p.beta, p.out_is_bf16 ? bf16_bits_to_float(static_cast<const uint16_t*>(p.c)[index]) : static_cast<const float*>(p.c)[index], sum);
                if (p.out_is_bf16) static_cast<uint16_t*>(p.out)[index] = float_to_bf16_bits(sum);
                else static_cast<float*>(p.out)[index] = sum;
            }
            asm volatile("bar.sync 1, %0;" ::"r"(p.warps * 32) : "memory");
        }
    }
}

struct Plan {
    uint32_t max_tokens, n, k;
    uint32_t* status;
    gemm::MapCache maps_w;
};

// How a call is cut: rows of a CTA and pass, MMA tiles they take, consumer warps, ring slots of a warp.
struct Cut {
    uint32_t rows, passes, tiles, warps, depth, smem;
};
inline Cut cut(uint32_t n, uint32_t k, uint32_t pitch, uint32_t tokens, uint32_t sms) {
    const uint32_t chunks = (k + 2 * kChunkBytes - 1) / (2 * kChunkBytes);
    Cut r{};
    for (uint32_t most = kMaxTiles; most > 0; --most) {
        r.passes = (n + sms * most * 16 - 1) / (sms * most * 16);
        r.rows = (n + sms * r.passes - 1) / (sms * r.passes);
        r.tiles = (r.rows + 15) / 16;
        // as few warps as leave the one with most chunks no more of them
        const uint32_t all = chunks * r.passes, rounds = (all + kMaxWarps - 1) / kMaxWarps;
        r.warps = (all + rounds - 1) / rounds;
        const uint32_t fixed = fixed_bytes(r.tiles, r.warps, tokens, pitch, r.passes), slot = slot_bytes(r.tiles) * r.warps;
        if (fixed + slot > kSmemLimit) continue;  // (long rows of scales: fewer of them at a time)
        r.depth = std::min(std::min(kMaxSlots / r.warps, rounds), (kSmemLimit - fixed) / slot);
        r.smem = fixed + r.depth * slot;
        return r;
    }
    r.depth = 0;
    return r;
}

template <int TILES, int COLS, int SPREAD, bool SPLIT_TERMS, typename XT>
cudaError_t launch(const CUtensorMap& map, const Params& p, uint32_t ctas, uint32_t smem, cudaStream_t stream) {
    auto kernel = decode_mxfp4_kernel<TILES, COLS, SPREAD, SPLIT_TERMS, XT>;
    static std::atomic<uint8_t> configured[gemm::kMaxDevices];
    if (cudaError_t st = gemm::opt_in_smem(configured, kernel, kSmemLimit); st != cudaSuccess) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(32 * (p.warps + 1));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, map, p);
}
struct Call {
    Plan& plan;
    Params p;
    const uint8_t* w_values;
    cudaStream_t stream;
};
template <int COLS, int SPREAD, bool SPLIT_TERMS, typename XT> cudaError_t run(Call& call) {
    Params& p = call.p;
    const Cut how = cut(p.n, p.k, p.pitch, 8 / (SPREAD * (SPLIT_TERMS ? 2 : 1)), static_cast<uint32_t>(gemm::sm_count()));
    if (how.depth == 0) return cudaErrorInvalidValue;
    const CUtensorMap* map;
    cudaError_t st = call.plan.maps_w.get(&map, call.w_values, p.n, p.k / 2, p.k / 2, how.rows);
    if (st != cudaSuccess) return st;
    p.rows = how.rows;
    p.passes = how.passes;
    p.chunks = (p.k + 2 * kChunkBytes - 1) / (2 * kChunkBytes);
    p.depth = how.depth;
    p.warps = how.warps;
    const uint32_t ctas = (p.n + how.rows * how.passes - 1) / (how.rows * how.passes);
    switch (how.tiles) {
        case 1: return launch<1, COLS, SPREAD, SPLIT_TERMS, XT>(*map, p, ctas, how.smem, call.stream);
        case 2: return launch<2, COLS, SPREAD, SPLIT_TERMS, XT>(*map, p, ctas, how.smem, call.stream);
        default: return launch<3, COLS, SPREAD, SPLIT_TERMS, XT>(*map, p, ctas, how.smem, call.stream);
    }
}
cudaError_t run_tokens(Call& call, bool bf16) {
    const uint32_t tokens = call.p.tokens;
    if (bf16) {
        if (tokens == 1) return run<1, 8, false, uint16_t>(call);
        if (tokens == 2) return run<1, 4, false, uint16_t>(call);
        if (tokens <= 4) return run<1, 2, false, uint16_t>(call);
        if (tokens <= 8) return run<1, 1, false, uint16_t>(call);
        return tokens <= 16 ? run<2, 1, false, uint16_t>(call) : run<4, 1, false, uint16_t>(call);
    }
    if (tokens == 1) return run<1, 4, true, float>(call);
    if (tokens == 2) return run<1, 2, true, float>(call);
    if (tokens <= 4) return run<1, 1, true, float>(call);
    if (tokens <= 8) return run<1, 1, false, float>(call);
    return tokens <= 16 ? run<2, 1, false, float>(call) : run<4, 1, false, float>(call);
}

}  // namespace decode_mx
}  // namespace eider

using namespace eider;

extern "C" {

void* eider_b200_mxfp4_decode_create(uint32_t max_tokens, uint32_t out_features, uint32_t in_features) {
    if (max_tokens == 0 || max_tokens > 64 || out_features == 0 || in_features == 0 || in_features % mx::kBlock != 0 || in_features > 65536) return nullptr;
    auto* plan = new (std::nothrow) decode_mx::Plan{max_tokens, out_features, in_features, nullptr, {}};
    if (!plan) return nullptr;
    if (cudaMalloc(reinterpret_cast<void**>(&plan->status), sizeof(uint32_t)) != cudaSuccess || cudaMemset(plan->status, 0, sizeof(uint32_t)) != cudaSuccess) {
        cudaFree(plan->status);
        delete plan;
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

cudaError_t eider_b200_mxfp4_w4a16_gemv_on_stream(void* raw, const void* input, int input_is_bf16, uint32_t tokens, const uint8_t* w_values,
                                                  const uint8_t* w_scales_rows, uint32_t scale_pitch, const void* c, void* d, float beta,
                                                  int out_is_bf16, cudaStream_t stream) {
    using namespace decode_mx;
    auto* plan = static_cast<Plan*>(raw);
    if (!plan || !input || !w_values || !w_scales_rows || !d || tokens == 0 || tokens > plan->max_tokens || (beta != 0.0f && !c)) return cudaErrorInvalidValue;
    if (((reinterpret_cast<uintptr_t>(input) | reinterpret_cast<uintptr_t>(w_values) | reinterpret_cast<uintptr_t>(w_scales_rows)) & 15) != 0 ||
        scale_pitch % 16 != 0 || scale_pitch < (plan->k / mx::kBlock + 7) / 8 * 8)
        return cudaErrorInvalidValue;
    const uint32_t groups = (tokens + 31) / 32, each = (tokens + groups - 1) / groups;
    for (uint32_t first = 0; first < tokens; first += each) {
        Call call{*plan, {}, w_values, stream};
        Params& p = call.p;
        p.tokens = std::min(each, tokens - first);
        const size_t x_bytes = input_is_bf16 ? 2 : 4, out_bytes = out_is_bf16 ? 2 : 4;
        p.x = static_cast<const uint8_t*>(input) + first * x_bytes * plan->k;
        p.scales = w_scales_rows;
        p.out = static_cast<uint8_t*>(d) + first * out_bytes * plan->n;
        p.c = c ? static_cast<const uint8_t*>(c) + first * out_bytes * plan->n : nullptr;
        p.status = plan->status;
        p.beta = beta;
        p.out_is_bf16 = out_is_bf16;
        p.n = plan->n;
        p.k = plan->k;
        p.pitch = scale_pitch;
        const cudaError_t st = run_tokens(call, input_is_bf16);
        if (st != cudaSuccess) return st;
    }
    return cudaSuccess;
}

}  // extern "C"
