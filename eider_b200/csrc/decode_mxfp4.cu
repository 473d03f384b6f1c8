// W4A16 product of MXFP4 weights for few tokens: y[t][n] = sum_k x[t][k] * w[n][k] (+ beta * C), the weights streamed once.
//
// Bound: HBM, N * K * 17/32 bytes of weights.  Every CTA has N / 148 rows of its own for the whole K (as many passes as rows do not fit), so
// that all SMs stream the same number of bytes whatever N is and no partial sum leaves a CTA: one launch, no workspace, the same
// order of additions in every run.
//  * A producer warp streams the rows in chunks of 256 elements (TMA boxes of 128 bytes x rows, 128-byte swizzle) through a ring of
//    shared memory; weights and scales are requested before the launch in front is awaited.
//  * Each chunk is one warp's, for all of the CTA's rows: 16 rows x 32 elements (a block) at a time through mma.m16n8k16 with the tokens
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
constexpr uint32_t kMaxWarps = 11;                  // consumer warps; with the producer three a scheduler, 168 registers each
constexpr uint32_t kMaxRows = 96;                   // rows of a CTA in a pass: six MMA tiles
constexpr uint32_t kSmemLimit = 227 * 1024;
constexpr uint32_t kMaxSlots = 64;
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
    uint32_t passes, chunks, slots, warps;
};

__host__ __device__ constexpr uint32_t reduce_pitch(uint32_t tiles) { return tiles * 16 + 4; }  // (rows of a token; + 4: the fragments' stores meet no bank twice)
__host__ __device__ constexpr uint32_t slot_bytes(uint32_t tiles) { return tiles * 16 * kChunkBytes; }
inline uint32_t fixed_bytes(uint32_t tiles, uint32_t warps, uint32_t pitch, uint32_t passes) {
    return 1024 /*alignment*/ + (passes > 1 ? 2 : 1) * tiles * 16 * pitch + warps * 8 * reduce_pitch(tiles) * 4 + (2 * kMaxSlots + 4) * 8 + 16;
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
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
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

// Eight consecutive elements of a token.
template <typename T> struct Raw8;
template <> struct Raw8<uint16_t> {
    uint4 q;
    __device__ __forceinline__ void load(const uint16_t* p, bool live) { q = live ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};
template <> struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p, bool live) {
        a = live ? __ldg(reinterpret_cast<const float4*>(p)) : make_float4(0, 0, 0, 0);
        b = live ? __ldg(reinterpret_cast<const float4*>(p) + 1) : make_float4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};

// TILES: 16-row MMA tiles of a CTA's rows.  COLS: groups of eight tokens.
template <int TILES, int COLS, typename XT>
__global__ void __launch_bounds__(32 * (kMaxWarps + 1), 1) decode_mxfp4_kernel(const __grid_constant__ CUtensorMap map_w, const Params p) {
    constexpr bool kF32 = sizeof(XT) == 4;
    constexpr int kTerms = kF32 ? 2 : 1;
    constexpr int kStep = COLS * kTerms >= 4 ? 1 : 4 / (COLS * kTerms);  // blocks of x that a warp holds (and has on their way) at a time
    extern __shared__ uint8_t smem_raw[];
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const uint32_t scale_bytes = TILES * 16 * p.pitch;
    uint8_t* scales = ring + p.slots * slot_bytes(TILES);
    float* sums = reinterpret_cast<float*>(scales + (p.passes > 1 ? 2 : 1) * scale_bytes);
    uint64_t* full = reinterpret_cast<uint64_t*>(sums + p.warps * 8 * reduce_pitch(TILES));  // [slots]
    uint64_t* empty = full + kMaxSlots;                                                     // [slots]
    uint64_t* scales_full = empty + kMaxSlots;                                              // [2]
    uint64_t* scales_empty = scales_full + 2;                                               // [2]
    volatile uint32_t* abort_flag = reinterpret_cast<uint32_t*>(scales_empty + 2);

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < p.slots; ++i) {
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
                    const uint32_t slot = i % p.slots, phase = (i / p.slots) & 1;
                    if (!umma::mbar_wait(&empty[slot], phase ^ 1, abort_flag, p.status, umma::kTimeoutEmpty)) { ok = false; break; }
                    umma::mbar_arrive_expect_tx(&full[slot], p.rows * kChunkBytes);
                    umma::tma_load_2d(ring + slot * slot_bytes(TILES), &map_w, &full[slot], static_cast<int32_t>(c * kChunkBytes), static_cast<int32_t>(row0));
                }
            }
            // The block does not leave before its copies have landed, not even after a wait ran out: bounded too.
            const long long start = clock64();
            auto landed = [&](uint64_t* bar, uint32_t parity) {
                while (!umma::mbar_try_wait(bar, parity) && clock64() - start < umma::kWaitLimitCycles) {}
            };
            for (uint32_t j = i > p.slots ? i - p.slots : 0; j < i; ++j) landed(&full[j % p.slots], (j / p.slots) & 1);
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
    bool live[COLS];
    size_t x_at[COLS];
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
        live[n] = n * 8 + g < p.tokens;
        x_at[n] = live[n] ? static_cast<size_t>(n * 8 + g) * p.k : 0;
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

        Raw8<XT> raw[COLS][kStep];
        auto load_x = [&](uint32_t block) {
#pragma unroll
            for (int n = 0; n < COLS; ++n)
#pragma unroll
                for (int s = 0; s < kStep; ++s) raw[n][s].load(x + x_at[n] + static_cast<size_t>(block + s) * mx::kBlock, live[n] && block + s < blocks);
        };
        if (warp < p.chunks) load_x(warp * kChunkBlocks);
        if (ok && !umma::mbar_wait(&scales_full[pass & 1], (pass >> 1) & 1, abort_flag, p.status, umma::kTimeoutFull)) ok = false;
        const uint32_t pass_scales = scales_addr + (pass & 1) * scale_bytes;
        for (uint32_t c = warp; ok && c < p.chunks; c += p.warps) {
            const uint32_t i = pass * p.chunks + c, slot = i % p.slots, phase = (i / p.slots) & 1;
            const uint32_t tile = ring_addr + slot * slot_bytes(TILES) + g * kChunkBytes + t * 4;
            bool arrived = false;
#pragma unroll 1
            for (uint32_t step = 0; step < kChunkBlocks; step += kStep) {
                // this step's x as f16, then the next step's is requested
                uint32_t b[kStep][COLS][kTerms][4];
#pragma unroll
                for (int n = 0; n < COLS; ++n) {
                    float v[kStep][8];
                    uint32_t amax = 0;
#pragma unroll
                    for (int s = 0; s < kStep; ++s) {
                        raw[n][s].values(v[s]);
#pragma unroll
                        for (int e = 0; e < 8; ++e) amax = max(amax, mx::abs_bits(v[s][e]));
                    }
                    if (amax >= 0x7f800000u) {  // an infinity or NaN goes through as it is; the finite ones set the scale
                        amax = 0;
#pragma unroll
                        for (int s = 0; s < kStep; ++s)
#pragma unroll
                            for (int e = 0; e < 8; ++e) amax = max(amax, mx::abs_bits(v[s][e]) < 0x7f800000u ? mx::abs_bits(v[s][e]) : 0u);
                    }
                    amax = max(amax, __shfl_xor_sync(kFull, amax, 1));
                    amax = max(amax, __shfl_xor_sync(kFull, amax, 2));
                    const bool rescale = factor[n] == 0.0f ? amax != 0 : __uint_as_float(amax) * factor[n] >= 32768.0f;
                    if (__any_sync(kFull, rescale)) {
                        float change = 1.0f;
                        if (rescale) {
                            const uint32_t e = amax >> 23;
                            const float wanted = __uint_as_float(min(254u, 262u - e) << 23);  // the largest element to 2^8..2^9
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
                    const float f = factor[n] == 0.0f ? 1.0f : factor[n];
#pragma unroll
                    for (int s = 0; s < kStep; ++s)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float lo = v[s][2 * e] * f, hi = v[s][2 * e + 1] * f;
                            b[s][n][0][e] = f16x2(lo, hi);
                            if constexpr (kF32) {
                                const float2 first = f16x2_values(b[s][n][0][e]);
                                // (of an infinity or NaN the first term is all there is)
                                b[s][n][kTerms - 1][e] = f16x2(fabsf(first.x) < INFINITY ? lo - first.x : 0.0f, fabsf(first.y) < INFINITY ? hi - first.y : 0.0f);
                            }
                        }
                }
                const uint32_t next = step + kStep;
                if (next < kChunkBlocks) load_x(c * kChunkBlocks + next);
                else if (c + p.warps < p.chunks) load_x((c + p.warps) * kChunkBlocks);
                if (!arrived) {
                    if (!__all_sync(kFull, umma::mbar_wait(&full[slot], phase, abort_flag, p.status, umma::kTimeoutFull))) { ok = false; break; }
                    arrived = true;
                }
                // scale bytes of these blocks
                const uint32_t scale_at = pass_scales + g * p.pitch + c * kChunkBlocks + (step & ~3u);
#pragma unroll
                for (int u = 0; u < TILES; ++u) {
                    const uint32_t lo4 = lds32(scale_at + u * 16 * p.pitch), hi4 = lds32(scale_at + (u * 16 + 8) * p.pitch);
#pragma unroll
                    for (int s = 0; s < kStep; ++s) {
                        const uint32_t block = step + s, shift = 8 * (block & 3);
                        const uint32_t at = tile + u * 16 * kChunkBytes + ((block ^ g) << 4);
                        uint32_t lo[4], hi[4];
                        e2m1_f16(lds32(at), lo);
                        e2m1_f16(lds32(at + 8 * kChunkBytes), hi);
                        const float s_lo = mx::scale_value(lo4 >> shift & 255u), s_hi = mx::scale_value(hi4 >> shift & 255u);
#pragma unroll
                        for (int n = 0; n < COLS; ++n) {
                            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                            for (int term = 0; term < kTerms; ++term) {
                                mma_f16(d, lo[0], hi[0], lo[1], hi[1], b[s][n][term][0], b[s][n][term][1]);
                                mma_f16(d, lo[2], hi[2], lo[3], hi[3], b[s][n][term][2], b[s][n][term][3]);
                            }
                            acc[u][n][0] = fmaf(d[0], s_lo, acc[u][n][0]);
                            acc[u][n][1] = fmaf(d[1], s_lo, acc[u][n][1]);
                            acc[u][n][2] = fmaf(d[2], s_hi, acc[u][n][2]);
                            acc[u][n][3] = fmaf(d[3], s_hi, acc[u][n][3]);
                        }
                    }
                }
            }
            __syncwarp();
            if (ok && lane == 0) umma::mbar_arrive(&empty[slot]);
        }
        if (lane == 0) umma::mbar_arrive(&scales_empty[pass & 1]);

        // ------------------------------------------------------------------ the warps' sums meet, eight tokens at a time
#pragma unroll
        for (int n = 0; n < COLS; ++n) {
            if (n * 8 >= p.tokens) break;
            // (1 / factor, exact: 2^-127 is subnormal)
            const uint32_t field = __float_as_uint(factor[n]) >> 23;
            const float back = factor[n] == 0.0f ? 1.0f : __uint_as_float(field == 254 ? 0x00400000u : (254u - field) << 23);
            const float b0 = __shfl_sync(kFull, back, t * 8), b1 = __shfl_sync(kFull, back, t * 8 + 4);
            float* mine = sums + warp * 8 * reduce_pitch(TILES);
#pragma unroll
            for (int u = 0; u < TILES; ++u) {
                mine[(2 * t) * reduce_pitch(TILES) + u * 16 + g] = acc[u][n][0] * b0;
                mine[(2 * t + 1) * reduce_pitch(TILES) + u * 16 + g] = acc[u][n][1] * b1;
                mine[(2 * t) * reduce_pitch(TILES) + u * 16 + g + 8] = acc[u][n][2] * b0;
                mine[(2 * t + 1) * reduce_pitch(TILES) + u * 16 + g + 8] = acc[u][n][3] * b1;
            }
            asm volatile("bar.sync 1, %0;" ::"r"(p.warps * 32) : "memory");
            const uint32_t tokens = min(8u, p.tokens - n * 8), rows = min(p.rows, p.n - row0);
            for (uint32_t i = threadIdx.x; i < tokens * rows; i += p.warps * 32) {
                const uint32_t token = i / rows, row = i - token * rows;
                float sum = 0.0f;
                for (uint32_t w = 0; w < p.warps; ++w) sum += sums[(w * 8 + token) * reduce_pitch(TILES) + row];
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

// How a call is cut: rows of a CTA and pass, MMA tiles they take, consumer warps, ring slots.
struct Cut {
    uint32_t rows, passes, tiles, warps, slots, smem;
};
inline Cut cut(uint32_t n, uint32_t k, uint32_t pitch, uint32_t sms) {
    Cut r{};
    const uint32_t chunks = (k + 2 * kChunkBytes - 1) / (2 * kChunkBytes);
    const uint32_t rounds = (chunks + kMaxWarps - 1) / kMaxWarps;  // chunks of the warp that has most
    r.warps = (chunks + rounds - 1) / rounds;
    for (uint32_t most = kMaxRows; most >= 16; most -= 16) {
        r.passes = (n + sms * most - 1) / (sms * most);
        r.rows = (n + sms * r.passes - 1) / (sms * r.passes);
        r.tiles = (r.rows + 15) / 16;
        if (r.tiles == 5) r.tiles = 6;
        const uint32_t fixed = fixed_bytes(r.tiles, r.warps, pitch, r.passes);
        if (fixed + 2 * slot_bytes(r.tiles) > kSmemLimit) continue;
        r.slots = std::min(std::min(kMaxSlots, chunks * r.passes), (kSmemLimit - fixed) / slot_bytes(r.tiles));
        // (half of the shared memory in flight at least, while fewer rows would allow it)
        if (r.slots < std::min(4u, chunks) && most > 16) continue;
        r.smem = fixed + r.slots * slot_bytes(r.tiles);
        return r;
    }
    r.slots = 0;
    return r;
}

template <int TILES, int COLS, typename XT>
cudaError_t launch(const CUtensorMap& map, const Params& p, uint32_t ctas, uint32_t smem, cudaStream_t stream) {
    auto kernel = decode_mxfp4_kernel<TILES, COLS, XT>;
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
template <int COLS, typename XT>
cudaError_t launch_tiles(uint32_t tiles, const CUtensorMap& map, const Params& p, uint32_t ctas, uint32_t smem, cudaStream_t stream) {
    switch (tiles) {
        case 1: return launch<1, COLS, XT>(map, p, ctas, smem, stream);
        case 2: return launch<2, COLS, XT>(map, p, ctas, smem, stream);
        case 3: return launch<3, COLS, XT>(map, p, ctas, smem, stream);
        case 4: return launch<4, COLS, XT>(map, p, ctas, smem, stream);
        default: return launch<6, COLS, XT>(map, p, ctas, smem, stream);
    }
}
template <typename XT>
cudaError_t launch_cols(uint32_t cols, uint32_t tiles, const CUtensorMap& map, const Params& p, uint32_t ctas, uint32_t smem, cudaStream_t stream) {
    if (cols == 1) return launch_tiles<1, XT>(tiles, map, p, ctas, smem, stream);
    if (cols == 2) return launch_tiles<2, XT>(tiles, map, p, ctas, smem, stream);
    return launch_tiles<4, XT>(tiles, map, p, ctas, smem, stream);
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
        Params p{};
        p.tokens = std::min(each, tokens - first);
        const uint32_t cols = p.tokens <= 8 ? 1 : p.tokens <= 16 ? 2 : 4;
        const Cut how = cut(plan->n, plan->k, scale_pitch, static_cast<uint32_t>(gemm::sm_count()));
        if (how.slots == 0) return cudaErrorInvalidValue;
        const CUtensorMap* map;
        cudaError_t st = plan->maps_w.get(&map, w_values, plan->n, plan->k / 2, plan->k / 2, how.rows);
        if (st != cudaSuccess) return st;
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
        p.rows = how.rows;
        p.passes = how.passes;
        p.chunks = (plan->k + 2 * kChunkBytes - 1) / (2 * kChunkBytes);
        p.slots = how.slots;
        p.warps = how.warps;
        const uint32_t ctas = (plan->n + how.rows * how.passes - 1) / (how.rows * how.passes);
        st = input_is_bf16 ? launch_cols<uint16_t>(cols, how.tiles, *map, p, ctas, how.smem, stream)
                           : launch_cols<float>(cols, how.tiles, *map, p, ctas, how.smem, stream);
        if (st != cudaSuccess) return st;
    }
    return cudaSuccess;
}

}  // extern "C"
