// W4A16 product of MXFP4 weights for up to 64 tokens (decode_mxfp4.cu says which calls stay there): y[t][n] = sum_k x[t][k] * w[n][k] (+ beta * C),
// the weights streamed once.
//
// Bound: HBM, N * K * 17/32 bytes of weights.  The tensor cores take the weights as they are: E2M1 codes and E8M0 block scales are operands
// of tcgen05.mma kind::mxf8f6f4, and x goes in as a sum of E4M3 terms with block scales of their own, each the rounding of what the terms
// before it left.  A code has four significant bits and a sign, so two terms are all of bf16's eight bits, for elements within 2^14 of their
// block's largest, and five all of f32's twenty-four near it; what lies below loses bits (prepare_terms_kernel).  The products of terms are
// exact.
//  * A CTA has 128 rows (the MMA's M) and a part of K; all terms of all tokens are its columns, up to 128, so an MMA reads the weights from
//    shared memory once.  A term's MMAs of their own took as long as the copies: 24.8 us for one token (K 5120 -> N 13824), now 11.6.
//  * The CTAs of a cluster share their rows and split K; their sums meet through distributed shared memory in rank order: no atomics, the
//    same order of additions in every run.  As many CTAs a cluster as all clusters would run at once with three CTAs an SM (beyond 96
//    columns, tensor memory lets two, and the third waits for theirs): of 2 / 3 / 4 / 6 / 8 the product above took
//    16.1 / 13.0 / 19.2 / 17.5 / 22.5 us (nine tokens), K 13824 -> N 5120 with 4 / 6 / 8 18.1 / 14.5 / 12.9.
//  * The TMA brings 128 rows x 128 elements a step and spreads them: an operand byte holds one code whatever its width, 16 codes in the
//    lower half of 16 bytes.  This needs K % 128 == 0.  Four warps that copied them there (8 bytes a cp.async) kept it at 15.5 us without
//    a single MMA.
//  * x is prepared by a launch of its own in the operand's layout, a step one contiguous piece that a bulk copy brings, while the first
//    steps of weights are on their way.  Every CTA reads its part of it from L2: 12 KB a step of 8.5 KB of weights for 48 tokens, which is what
//    they cost beyond one (K 5120 -> N 13824: 1 token 11.6 us, 16 13.8, 48 21.7; K 13824 -> N 5120: 12.0, 13.3, 19.4; 64 tokens, whose
//    tensor memory leaves room for two CTAs an SM, 33.2 and 30.3).
#include <algorithm>
#include <atomic>

#include "gemm_launch.cuh"
#include "mx_block.cuh"
#include "decode_mxfp4.cuh"
#include "tensor_maps.cuh"

namespace eider {
namespace decode_mx {
namespace {

constexpr uint32_t kRows = 128;
constexpr uint32_t kTileBytes = kRows * 128, kScaleTile = 512;
constexpr uint32_t kMaxColumns = 128;  // terms of all tokens: one scale tile
constexpr uint32_t kThreads = 128;
constexpr uint32_t kCtasAnSm = 3;
constexpr uint32_t kMaxStages = 4;    // whose scale columns are 32
constexpr uint32_t kMaxSplits = 8;  // CTAs of a cluster
constexpr uint32_t kRing = 227 * 1024 / kCtasAnSm / 1024 * 1024 - 3072;  // two stages of 64 tokens, three of 16
constexpr uint32_t kSumPitch = kRows + 4;  // floats of a token's partial sums
constexpr uint32_t kScaleColumns = 32;
constexpr uint32_t kFull = 0xffffffffu;

// A step of prepared x: [term][tokens up to a multiple of 8][128 bytes, 16-byte pieces swizzled], then the rows' scale tile.
__host__ __device__ constexpr uint32_t terms_of(bool bf16) { return bf16 ? 2 : 5; }
__host__ __device__ constexpr uint32_t most_tokens(bool bf16) { return bf16 ? 64 : 24; }  // of a launch
__host__ __device__ constexpr uint32_t padded_of(uint32_t tokens) { return (tokens + 7) / 8 * 8; }
__host__ __device__ constexpr uint32_t columns_of(uint32_t tokens, bool bf16) { return terms_of(bf16) * padded_of(tokens); }
__host__ __device__ constexpr uint32_t step_bytes(uint32_t columns) { return columns * 128 + kScaleTile; }
__host__ __device__ constexpr uint32_t stage_bytes(uint32_t columns) { return kTileBytes + columns * 128 + 1024; }

struct Params {
    const uint8_t* x;       // prepared
    const void* raw;        // x itself
    const uint8_t* w;       // [n][k / 2]
    const uint8_t* scales;  // tiles of 128 rows x 4 blocks
    void* out;
    const void* c;
    float beta;
    int out_is_bf16, x_is_bf16;
    uint32_t tokens, padded, terms, columns, n, k, stages, tmem_columns;
    uint32_t* status;  // of a wait that ran out
};

__device__ __forceinline__ float lds_cluster(uint32_t address) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(address) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 e4m3x2_values(uint32_t codes) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(codes)));
    float2 f;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(f.x), "=f"(f.y) : "r"(h));
    return f;
}
// 2^(c - 127), c in 0 .. 254
__device__ __forceinline__ float exp2_code(uint32_t c) { return __uint_as_float(c == 0 ? 0x00400000u : c << 23); }
// Eight elements of a token from `p` on; zeros if not `live`.  (__ldcg: to the compiler __ldg has no order with griddepcontrol.wait, and it
// requested what the launch in front had not written yet: 264 of 3200 calls came out wrong.)
__device__ __forceinline__ void load8(const uint16_t* p, bool live, float (&v)[8]) {
    const uint4 q = live ? __ldcg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void load8(const float* p, bool live, float (&v)[8]) {
    const float4 a = live ? __ldcg(reinterpret_cast<const float4*>(p)) : make_float4(0, 0, 0, 0);
    const float4 b = live ? __ldcg(reinterpret_cast<const float4*>(p) + 1) : make_float4(0, 0, 0, 0);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// x as E4M3 terms: one CTA a step of 128 elements and 16 tokens, 16 threads a token of it, four a block.  A block's first scale brings its largest
// finite element to 2^7 .. 2^8; what a term leaves is at most 2^3 in its scale, so the next term's is 2^-5 of it.  bf16 elements keep all
// their bits as long as they lie within 2^14 of their block's largest, and 2^-22 of that one else; f32 elements leave at most 2^-24 of
// themselves, or 2^-37 of the largest.  An infinity or NaN goes in as NaN: resolve tells them apart.
constexpr uint32_t kPrepareThreads = 256;
template <typename XT>
__global__ void __launch_bounds__(kPrepareThreads) prepare_terms_kernel(const XT* __restrict__ x, uint8_t* __restrict__ prepared, uint32_t tokens, uint32_t padded, uint32_t k) {
    constexpr uint32_t kTerms = terms_of(sizeof(XT) == 2);
    umma::griddep_launch_dependents();
    const uint32_t columns = kTerms * padded;
    uint8_t* out = prepared + static_cast<size_t>(blockIdx.x) * step_bytes(columns);
    uint8_t* scales = out + columns * 128;
    const uint32_t part = threadIdx.x % 16, at = blockIdx.x * 128 + part * 8;
    umma::griddep_wait();
    const uint32_t token = blockIdx.y * (kPrepareThreads / 16) + threadIdx.x / 16;
    if (token < padded) {  // (whole warps: padded is a multiple of 8)
        float v[8], amax = 0.0f;
        load8(x + static_cast<size_t>(token) * k + at, token < tokens, v);
        bool odd[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            odd[i] = !(fabsf(v[i]) < INFINITY);
            if (odd[i]) v[i] = 0.0f;
            amax = fmaxf(amax, fabsf(v[i]));
        }
        amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 2));
        // floor(log2 amax) - 7, from the exponent field (a subnormal amax has 0 there and ends up at scale 0 all the same)
        uint32_t code = max(__float_as_uint(amax) >> 23, 7u) - 7u;
#pragma unroll
        for (uint32_t term = 0; term < kTerms; ++term) {
            // (2^-c in two factors: c reaches 247)
            const float down = exp2_code(254 - max(code, 127u)), up = exp2_code(254 - min(code, 127u)), scale = exp2_code(code);
            uint32_t packed[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const uint32_t codes = e4m3x2(v[i] * down * up, v[i + 1] * down * up);
                const float2 back = e4m3x2_values(codes);
                v[i] -= back.x * scale;
                v[i + 1] -= back.y * scale;
                packed[i / 4] |= codes << (i % 4 * 8);
            }
            if (term == 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (odd[i]) packed[i / 4] |= 0x7fu << (i % 4 * 8);
            }
            const uint32_t row = term * padded + token;
            *reinterpret_cast<uint2*>(out + row * 128 + (((part / 2) ^ (row & 7)) << 4) + part % 2 * 8) = make_uint2(packed[0], packed[1]);
            if (part % 4 == 0) scales[row % 32 * 16 + row / 32 * 4 + part / 4] = static_cast<uint8_t>(code);
            code = max(code, 5u) - 5u;
        }
    }
}

__device__ __forceinline__ float value_at(const void* x, int is_bf16, size_t i) {
    return is_bf16 ? bf16_bits_to_float(__ldcg(static_cast<const uint16_t*>(x) + i)) : __ldcg(static_cast<const float*>(x) + i);
}
// What a row's sum is when it came out infinite or NaN: x's infinities went in as NaNs, and parts of a sum, or the term that an element near
// f32's end is rounded up to, overflow where the result does not.  Added up in 64 bits, in order.
__device__ __noinline__ float resolve(const Params& p, uint32_t token, uint32_t row) {
    const uint8_t* scales = p.scales + static_cast<size_t>(row / 128) * (p.k / 128) * kScaleTile + row % 32 * 16 + row % 128 / 32 * 4;
    double total = 0.0;
    for (uint32_t k = 0; k < p.k; ++k) {
        const uint32_t scale = scales[static_cast<size_t>(k / 128) * kScaleTile + k / 32 % 4];
        if (scale == mx::kNanCode) return NAN;
        const float x = value_at(p.raw, p.x_is_bf16, static_cast<size_t>(token) * p.k + k);
        const uint32_t code = p.w[static_cast<size_t>(row) * (p.k / 2) + k / 2] >> (k % 2 * 4) & 15;
        total += static_cast<double>(x) * e2m1_value(code) * mx::scale_value(scale);
        if (isnan(total)) return NAN;
    }
    return static_cast<float>(total);
}

__global__ void __launch_bounds__(kThreads) decode_terms_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ Params p) {
    extern __shared__ uint8_t raw_smem[];
    uint8_t* smem = raw_smem + (1024 - (umma::smem_u32(raw_smem) & 1023)) % 1024;  // (the same offset in every CTA)
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], done;
    __shared__ uint32_t tmem_base;
    __shared__ volatile uint32_t abort_flag;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t split = blockIdx.x, splits = gridDim.x;  // the cluster is a row of the grid
    const uint32_t row0 = blockIdx.y * kRows, rows = min(kRows, p.n - row0);
    const uint32_t all_steps = p.k / 128;
    const uint32_t step0 = split * all_steps / splits, steps = (split + 1) * all_steps / splits - step0;
    const uint32_t x_bytes = step_bytes(p.columns), stage = stage_bytes(p.columns);
    const uint32_t scales_at = kTileBytes + p.columns * 128;  // in a stage: x's scale tile, then the weights'

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < p.stages; ++s) {
            umma::mbar_init(full + s, 2);
            umma::mbar_init(empty + s, 1);
        }
        umma::mbar_init(&done, 1);
        abort_flag = 0;
        umma::fence_barrier_init();
    }
    if (warp == 2) {
        umma::tmem_alloc(&tmem_base, p.tmem_columns);  // (in one piece: no CTA waits for tensor memory while it holds some)
        umma::tmem_relinquish();
    }
    umma::tc_fence_before();
    __syncthreads();
    umma::tc_fence_after();
    umma::griddep_launch_dependents();  // (not before this CTA has its tensor memory: a dependent's could be in its place)
    const uint32_t tmem = tmem_base, scale_columns = tmem + p.tmem_columns - kScaleColumns;

    if (warp == 0 || warp == 3) {
        // ------------------------------------------------------------------------------------------ copies: weights, and x behind the launch in front
        if (lane == 0) {
            const bool weights = warp == 0;
            if (!weights) umma::griddep_wait();
            const uint8_t* x = p.x + static_cast<size_t>(step0) * x_bytes;
            const uint8_t* scales = p.scales + (static_cast<size_t>(blockIdx.y) * all_steps + step0) * kScaleTile;
            const uint64_t once = umma::policy_evict_first();
            uint32_t slot = 0, phase = 1;
            for (uint32_t i = 0; i < steps; ++i) {
                if (!umma::mbar_wait(empty + slot, phase, &abort_flag, p.status, umma::kTimeoutEmpty)) break;
                uint8_t* to = smem + slot * stage;
                if (weights) {
                    umma::mbar_arrive_expect_tx(full + slot, kTileBytes / 2 + kScaleTile);  // (the barrier counts the bytes read, not those spread)
                    umma::tma_load_2d_hint(to, &map_w, full + slot, static_cast<int32_t>((step0 + i) * 128), static_cast<int32_t>(row0), once);
                    umma::bulk_load_1d(to + scales_at + kScaleTile, scales + static_cast<size_t>(i) * kScaleTile, kScaleTile, full + slot);
                } else {
                    umma::mbar_arrive_expect_tx(full + slot, x_bytes);
                    umma::bulk_load_1d(to + kTileBytes, x + static_cast<size_t>(i) * x_bytes, x_bytes, full + slot);
                }
                if (++slot == p.stages) {
                    slot = 0;
                    phase ^= 1;
                }
            }
            if (abort_flag) {  // nobody may have waited for the copies in flight
                const long long start = clock64();
                while (clock64() - start < umma::kWaitLimitCycles / 64) {}
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------------------------------------ products
        if (lane == 0) {
            const uint32_t wide = (p.columns + 15) / 16 * 16;  // (what lies behind x goes to columns that nobody reads)
            uint32_t slot = 0, phase = 0;
            for (uint32_t i = 0; i < steps; ++i) {
                if (!umma::mbar_wait(full + slot, phase, &abort_flag, p.status, umma::kTimeoutFull)) break;
                umma::tc_fence_after();
                const uint32_t at = umma::smem_u32(smem) + slot * stage;
                // scale columns are a slot's own: its MMAs are done before it is filled again
                const uint32_t sfb = scale_columns + slot * 8, sfa = sfb + 4;
                umma::tc_copy_scales(sfb, umma::smem_desc_scales(at + scales_at));
                umma::tc_copy_scales(sfa, umma::smem_desc_scales(at + scales_at + kScaleTile));
                const uint64_t a = umma::smem_desc_sw128(at), b = umma::smem_desc_sw128(at + kTileBytes);
#pragma unroll
                for (uint32_t block = 0; block < 4; ++block)
                    umma::mma_mxf8f6f4(tmem, a + block * 2, b + block * 2, umma::idesc_mxf4f8(wide, block), sfa, sfb, i + block != 0);
                umma::tc_commit(empty + slot);
                if (++slot == p.stages) {
                    slot = 0;
                    phase ^= 1;
                }
            }
            umma::tc_commit(&done);
        }
        __syncwarp();
    }

    // ------------------------------------------------------------------------------------------ the cluster's sums meet
    float* sums = reinterpret_cast<float*>(smem);  // [tokens][kSumPitch]: the ring is done with
    bool good = umma::mbar_wait(&done, 0, &abort_flag, p.status, umma::kTimeoutTmemFull);
    good = __all_sync(kFull, good && abort_flag == 0);
    umma::tc_fence_after();
    for (uint32_t c = 0; c < p.padded; c += 8) {
        float v[8] = {};
        for (uint32_t term = p.terms; term-- > 0;) {  // (the small ones first)
            uint32_t part[8];
            umma::tmem_load_32x8(tmem + (warp * 32 << 16) + term * p.padded + c, part);
            umma::tmem_load_wait();
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) v[i] += __uint_as_float(part[i]);
        }
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            if (c + i < p.tokens) sums[(c + i) * kSumPitch + warp * 32 + lane] = good ? v[i] : NAN;  // (a wait ran out: no sum, and the plan's status says so)
    }
    umma::tc_fence_before();
    __syncthreads();
    if (warp == 2) {  // before the cluster meets: no CTA holds tensor memory while it waits for another
        umma::tc_fence_after();
        umma::tmem_dealloc(tmem, p.tmem_columns);
    }
    if (splits > 1) umma::cluster_sync_all();
    umma::griddep_wait();
    const uint32_t all = p.tokens * rows, begin = static_cast<uint32_t>(static_cast<uint64_t>(all) * split / splits), end = static_cast<uint32_t>(static_cast<uint64_t>(all) * (split + 1) / splits);
    uint32_t from[kMaxSplits];
#pragma unroll
    for (uint32_t s = 0; s < kMaxSplits; ++s) from[s] = s < splits ? umma::map_to_cta(umma::smem_u32(sums), s) : 0;
    for (uint32_t i = begin + threadIdx.x; i < end; i += kThreads) {
        const uint32_t token = i / rows, row = i - token * rows;
        float v[kMaxSplits], sum = 0.0f;
#pragma unroll
        for (uint32_t s = 0; s < kMaxSplits; ++s) v[s] = s < splits ? lds_cluster(from[s] + (token * kSumPitch + row) * 4) : 0.0f;
#pragma unroll
        for (uint32_t s = 0; s < kMaxSplits; ++s)
            if (s < splits) sum += v[s];
        if (!(fabsf(sum) < INFINITY)) sum = resolve(p, token, row0 + row);
        const size_t index = static_cast<size_t>(token) * p.n + row0 + row;
        if (p.beta != 0.0f)
            sum = fmaf(p.beta, p.out_is_bf16 ? bf16_bits_to_float(static_cast<const uint16_t*>(p.c)[index]) : static_cast<const float*>(p.c)[index], sum);
        if (p.out_is_bf16) static_cast<uint16_t*>(p.out)[index] = float_to_bf16_bits(sum);
        else static_cast<float*>(p.out)[index] = sum;
    }
    if (splits > 1) umma::cluster_sync_all();  // (the others may still read this CTA's sums)
}

static_assert(kRing >= 2 * stage_bytes(kMaxColumns) && kRing >= 64 * kSumPitch * 4 && columns_of(64, true) <= kMaxColumns && columns_of(24, false) <= kMaxColumns, "ring of the most tokens");

// Clusters of `splits` CTAs that the device runs at a time with three CTAs an SM: those it would run with one CTA an SM (asked for once, with shared memory for
// no more), times the CTAs an SM.
constexpr uint32_t kSmemMost = 226 * 1024;
uint32_t clusters_at_once(uint32_t splits) {
    static std::atomic<uint32_t> known[gemm::kMaxDevices][kMaxSplits + 1];
    std::atomic<uint32_t>& entry = known[gemm::current_device()][splits];
    uint32_t count = entry.load(std::memory_order_relaxed);
    if (count == 0) {
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {splits, 1, 1};
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(splits);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = kSmemMost;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, decode_terms_kernel, &cfg) != cudaSuccess || clusters < 1) clusters = 1;
        count = static_cast<uint32_t>(clusters) * kCtasAnSm;
        entry.store(count, std::memory_order_relaxed);
    }
    return count;
}

}  // namespace

// Tokens of a launch: as many as it takes, in groups of about one size.
uint32_t group_of(uint32_t tokens, bool bf16) {
    const uint32_t groups = (tokens + most_tokens(bf16) - 1) / most_tokens(bf16);
    return (tokens + groups - 1) / groups;
}

size_t terms_workspace_bytes(uint32_t tokens, uint32_t k, int input_is_bf16) {
    return static_cast<size_t>(k / 128) * step_bytes(columns_of(group_of(tokens, input_is_bf16), input_is_bf16));
}

cudaError_t run_terms(gemm::FifoCache<CUtensorMap>& maps, const void* x, int input_is_bf16, uint32_t tokens, const uint8_t* w, const uint8_t* scales,
                      const void* c, void* d, float beta, int out_is_bf16, uint32_t n, uint32_t k, uint8_t* workspace, uint32_t* status,
                      cudaStream_t stream) {
    const CUtensorMap* map = nullptr;
    cudaError_t st = maps.get(&map, gemm::MapKey{w, n, k, k / 2, kRows}, [&](CUtensorMap* to) { return gemm::make_spread_fp4_map(to, w, n, k, kRows); });
    if (st != cudaSuccess) return st;
    static std::atomic<uint8_t> configured[gemm::kMaxDevices];
    if (st = gemm::opt_in_smem(configured, decode_terms_kernel, kSmemMost); st != cudaSuccess) return st;
    const uint32_t each = group_of(tokens, input_is_bf16), steps = k / 128, tiles = (n + kRows - 1) / kRows;
    // as many CTAs a cluster as K has steps and as all clusters run at once (by three CTAs an SM, whatever the columns)
    uint32_t splits = std::min(kMaxSplits, steps);
    while (splits > 1 && tiles > clusters_at_once(splits)) --splits;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {splits, 1, 1};
    cudaLaunchConfig_t cfg = {};
    cfg.stream = stream;
    cfg.attrs = attr;
    const size_t out_row = static_cast<size_t>(n) * (out_is_bf16 ? 2 : 4), x_row = static_cast<size_t>(k) * (input_is_bf16 ? 2 : 4);
    for (uint32_t first = 0; first < tokens; first += each) {  // (the workspace is reused: every launch waits for the one in front)
        Params p{};
        p.x = workspace;
        p.raw = static_cast<const uint8_t*>(x) + first * x_row;
        p.w = w;
        p.scales = scales;
        p.out = static_cast<uint8_t*>(d) + first * out_row;
        p.c = c ? static_cast<const uint8_t*>(c) + first * out_row : nullptr;
        p.beta = beta;
        p.out_is_bf16 = out_is_bf16;
        p.x_is_bf16 = input_is_bf16;
        p.status = status;
        p.tokens = std::min(each, tokens - first);
        p.padded = padded_of(p.tokens);
        p.terms = terms_of(input_is_bf16);
        p.columns = p.terms * p.padded;
        // (beyond 96 columns two CTAs an SM have their tensor memory at a time, not three.  Sums and scales in pieces of their own
        // would let three run, 24.4 us instead of 33.2 for 64 tokens, but hold one piece while they wait for the other)
        p.tmem_columns = p.columns + kScaleColumns <= 64 ? 64 : p.columns + kScaleColumns <= 128 ? 128 : 256;
        p.n = n;
        p.k = k;
        p.stages = std::min(std::min(kMaxStages, (steps + splits - 1) / splits), kRing / stage_bytes(p.columns));
        cfg.numAttrs = 1;
        cfg.gridDim = dim3(steps, (p.padded + kPrepareThreads / 16 - 1) / (kPrepareThreads / 16));
        cfg.blockDim = dim3(kPrepareThreads);
        cfg.dynamicSmemBytes = 0;
        st = input_is_bf16 ? cudaLaunchKernelEx(&cfg, prepare_terms_kernel<uint16_t>, static_cast<const uint16_t*>(p.raw), workspace, p.tokens, p.padded, k)
                           : cudaLaunchKernelEx(&cfg, prepare_terms_kernel<float>, static_cast<const float*>(p.raw), workspace, p.tokens, p.padded, k);
        if (st != cudaSuccess) return st;
        cfg.numAttrs = 2;
        cfg.gridDim = dim3(splits, tiles);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = kRing + 1024;
        if (st = cudaLaunchKernelEx(&cfg, decode_terms_kernel, *map, p); st != cudaSuccess) return st;
    }
    return cudaSuccess;
}

}  // namespace decode_mx
}  // namespace eider
