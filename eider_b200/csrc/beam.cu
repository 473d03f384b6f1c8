// The step behind the lm-head when several hypotheses of a sequence are kept: the k best continuations over beams and vocabulary, and
// the states of the beams they come from.
//
//   score(r, v) = beam_score[r] + logits[r][v] - log sum_u exp(logits[r][u]),   the k largest of a sequence's beams x vocab scores,
//   equal scores in the order of beam * vocab + v.
//
// The scores are compared in 64 bits: log-sum-exps differ from row to row, and f32 would tie what is not equal.  A row's sum of
// exponentials itself is of f32: hardware exponentials and partial sums, together within 2^-21 of it on normal logits up to 151936 of
// them.  So the order within a row is exact, and candidates of different rows whose scores differ by less than that may change places.
// Rows that are equal have equal sums wherever they lie: the parts of a sum are counted from the row's first element, whatever its
// address.
//
// Two launches.  beam_scan_kernel reads the logits once (bound: HBM): running maximum and sum of exponentials per thread, and the
// maximum of every 64 consecutive logits (a segment).  beam_merge_kernel, one CTA per sequence, finds the k best segments by their
// maxima (the k best elements cannot lie in any others: each of k better segments holds a better element) and then the k best of
// their elements.  Nothing of the order of vocab is written or sorted; no atomics decide an order.
//
// Measured (B200): 64 x 8 x 151936 bf16 55.4 us, the scan 37 (4.2 TB/s; its share of the floor is 23.8) and the merge 18 (four
// dependent passes over 19 thousand maxima a sequence, 64 CTAs of 148 SMs); 1 x 4 x 32000 f32 16.5 us, dependent passes of one CTA;
// reordering 64 x 8 states of 64 KB, twice, 15.8 us.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <new>

#include "common.cuh"
#include "quant_block.cuh"
#include "eider_b200.h"

namespace eider {
namespace {

constexpr uint32_t kFullMask = 0xffffffffu;
constexpr uint32_t kSegment = 64;       // logits that share a maximum
constexpr uint32_t kScanThreads = 256;
constexpr uint32_t kAhead = 4;          // 16-byte vectors a thread has on their way
constexpr uint32_t kMergeThreads = 1024;
constexpr uint32_t kCandidates = 2048;  // of a selection; more are taken one by one
constexpr uint32_t kMaxBeams = 64, kMaxK = 128;
constexpr float kLog2e = 1.4426950408889634f;

struct BeamArgs {
    const void* logits;
    size_t stride;              // elements from row to row
    const float* beam_scores;   // [batch * beams]
    const uint8_t* finished;    // [batch * beams] or null
    float* segment_max;         // [batch * beams][segments]
    float2* partial;            // [batch * beams][splits]: maximum and sum of exponentials below it
    float* out_scores;          // [batch][k]
    int32_t* out_parents;
    int32_t* out_tokens;
    uint32_t beams, vocab, k, pad_token, segments, splits, vectors_per_split;
};

// (What earlier launches wrote is not read with __ldg: to the compiler a read-only load has no order with griddepcontrol.wait.)
__device__ __forceinline__ bool row_counts(const BeamArgs& a, uint32_t row) {
    return isfinite(__ldcg(a.beam_scores + row)) && !(a.finished && __ldcg(a.finished + row));
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T> struct Vec {
    static constexpr uint32_t kElems = 16 / sizeof(T);
};
template <typename T> __device__ __forceinline__ T minus_infinity();
template <> __device__ __forceinline__ float minus_infinity<float>() { return -INFINITY; }
template <> __device__ __forceinline__ uint16_t minus_infinity<uint16_t>() { return 0xff80; }
__device__ __forceinline__ float logit_value(float v) { return v; }
__device__ __forceinline__ float logit_value(uint16_t v) { return bf16_bits_to_float(v); }
__device__ __forceinline__ void vector_values(const uint4& q, float (&v)[4]) {
    v[0] = __uint_as_float(q.x); v[1] = __uint_as_float(q.y); v[2] = __uint_as_float(q.z); v[3] = __uint_as_float(q.w);
}
__device__ __forceinline__ void vector_values(const uint4& q, float (&v)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
// Rows need not start on 16 bytes.  The 16 bytes from byte BYTES of piece v of memory on, in lane v: up to 8 it holds piece v and lacks the begin of the next lane's, beyond
// it holds piece v + 1 and lacks the end of the lane's in front, two words at most.  `edge`: those two words for the lane at the end of
// the warp, held by the lane at its other end, whose own words nobody takes.
template <uint32_t BYTES> __device__ __forceinline__ uint4 shifted_piece(const uint4& piece, const uint2& edge, uint32_t lane) {
    constexpr bool kForward = BYTES <= 8;
    constexpr uint32_t kStart = kForward ? BYTES : BYTES - 8, kFirst = kStart / 4;
    auto taken = [&](uint32_t own, uint32_t at_edge) { return __shfl_sync(kFullMask, lane == (kForward ? 0 : 31) ? at_edge : own, kForward ? lane + 1 : lane - 1); };
    uint32_t w[6];
    if constexpr (kForward) {
        w[0] = piece.x; w[1] = piece.y; w[2] = piece.z; w[3] = piece.w;
        w[4] = taken(piece.x, edge.x);
        w[5] = kStart > 4 ? taken(piece.y, edge.y) : 0;
    } else {
        w[0] = kStart < 4 ? taken(piece.z, edge.x) : 0;
        w[1] = taken(piece.w, edge.y);
        w[2] = piece.x; w[3] = piece.y; w[4] = piece.z; w[5] = piece.w;
    }
    if constexpr (kStart % 4 == 0) return make_uint4(w[kFirst], w[kFirst + 1], w[kFirst + 2], w[kFirst + 3]);
    else return make_uint4(__funnelshift_r(w[kFirst], w[kFirst + 1], 16), __funnelshift_r(w[kFirst + 1], w[kFirst + 2], 16),
                           __funnelshift_r(w[kFirst + 2], w[kFirst + 3], 16), __funnelshift_r(w[kFirst + 3], w[kFirst + 4], 16));
}

// The running maximum and sum of a CTA's part of a row, and its segments' maxima.  The row begins BYTES behind a 16-byte boundary: if that
// is not 0, a vector is the end of one piece of memory and the begin of the next.
template <typename T, uint32_t BYTES> __device__ __forceinline__ void scan_row(const BeamArgs& a, const T* logits, float* segment_max, float& top, float& sum) {
    constexpr uint32_t E = Vec<T>::kElems, kSegLanes = kSegment / E, kLead = BYTES / sizeof(T);
    constexpr uint32_t kBehind = BYTES > 8 ? 1 : 0;  // (lanes hold the pieces that their vectors end in)
    constexpr uint32_t kTurn = kScanThreads * kAhead;
    const uint32_t lane = threadIdx.x % 32;
    const uint32_t v1 = min((blockIdx.x + 1) * a.vectors_per_split, (a.vocab + E - 1) / E);
    const uint4* pieces = reinterpret_cast<const uint4*>(logits - kLead);
    // Whether the vectors from `first` on, `count` of them, come in pieces that lie in the row
    auto in_pieces = [&](uint32_t first, uint32_t count) {
        return kLead == 0 ? (first + count) * E <= a.vocab : first > 0 && (first + count + 1) * E - kLead <= a.vocab;
    };
    // A turn's vectors, requested while the turn before is worked on.  (Whole warps run the same number of turns: a split is a
    // multiple of the block.)
    uint4 next[kAhead];
    uint2 next_edge[kAhead] = {};
    auto fetch_pieces = [&](uint32_t vec, uint32_t j) {
        next[j] = __ldcg(pieces + vec + kBehind);
        if (kLead != 0 && lane == (kBehind ? 31 : 0)) next_edge[j] = __ldcg(reinterpret_cast<const uint2*>(pieces + vec - lane + (kBehind ? 0 : 32)) + kBehind);
    };
    auto fetch = [&](uint32_t base) {
        if (base + kTurn <= v1 && in_pieces(base, kTurn)) {
#pragma unroll
            for (uint32_t j = 0; j < kAhead; ++j) fetch_pieces(base + j * kScanThreads + threadIdx.x, j);
            return;
        }
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            const uint32_t vec = base + j * kScanThreads + threadIdx.x, at = vec * E;
            if (vec < v1 && (kLead == 0 ? in_pieces(vec, 1) : in_pieces(vec - lane, 32))) {
                fetch_pieces(vec, j);
            } else {  // the row's last vectors (its first ones too, if they are in no whole pieces), and none
                T v[E];
#pragma unroll
                for (uint32_t e = 0; e < E; ++e) v[e] = vec < v1 && at + e < a.vocab ? __ldcg(logits + (at + e)) : minus_infinity<T>();
                memcpy(&next[j], v, 16);
            }
        }
    };
    uint32_t base = blockIdx.x * a.vectors_per_split;
    constexpr bool kPrefetch = kLead == 0;  // (vectors in two pieces take the registers of a turn ahead)
    if (kPrefetch && base < v1) fetch(base);
    for (; base < v1; base += kTurn) {
        if (!kPrefetch) fetch(base);
        uint4 now[kAhead];
        float m[kAhead];
        const bool whole = base + kTurn <= v1 && in_pieces(base, kTurn);
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            now[j] = next[j];
            if constexpr (kLead != 0) {
                const uint32_t first = base + j * kScanThreads + threadIdx.x - lane;  // (the warp's)
                if (whole || (first < v1 && in_pieces(first, 32))) now[j] = shifted_piece<BYTES>(next[j], next_edge[j], lane);
            }
        }
        if (kPrefetch && base + kTurn < v1) fetch(base + kTurn);
        float new_top = top;
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            float x[E];
            vector_values(now[j], x);
            m[j] = x[0];
#pragma unroll
            for (uint32_t e = 1; e < E; ++e) m[j] = fmaxf(m[j], x[e]);
            new_top = fmaxf(new_top, m[j]);
        }
        // (with nothing but -infinity so far, differences to 0 keep the sum 0, or NaN for a NaN, which passes the maximum by)
        const float to = new_top > -INFINITY ? new_top : 0.0f;
        sum *= exp2_fast((top - to) * kLog2e);
        top = new_top;
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            float x[E];
            vector_values(now[j], x);
            float part = 0.0f;
#pragma unroll
            for (uint32_t e = 0; e < E; ++e) part += exp2_fast((x[e] - to) * kLog2e);
            sum += part;
        }
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
#pragma unroll
            for (uint32_t o = 1; o < kSegLanes; o *= 2) m[j] = fmaxf(m[j], __shfl_xor_sync(kFullMask, m[j], o));
            const uint32_t vec = base + j * kScanThreads + threadIdx.x;
            if (threadIdx.x % kSegLanes == 0 && vec < v1) segment_max[vec / kSegLanes] = m[j];
        }
    }
}

template <typename T, bool SHIFTED> __device__ __forceinline__ void scan(const BeamArgs& a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t row = blockIdx.y;
    if (!row_counts(a, row)) return;
    const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
    float* segment_max = a.segment_max + static_cast<size_t>(row) * a.segments;
    float top = -INFINITY, sum = 0.0f;
    const uint32_t bytes = SHIFTED ? static_cast<uint32_t>(reinterpret_cast<uintptr_t>(logits) & 15) : 0;
    if (bytes == 0) scan_row<T, 0>(a, logits, segment_max, top, sum);
    if constexpr (SHIFTED) {
        if (bytes == 4) scan_row<T, 4>(a, logits, segment_max, top, sum);
        if (bytes == 8) scan_row<T, 8>(a, logits, segment_max, top, sum);
        if (bytes == 12) scan_row<T, 12>(a, logits, segment_max, top, sum);
        if constexpr (sizeof(T) == 2) {
            if (bytes == 2) scan_row<T, 2>(a, logits, segment_max, top, sum);
            if (bytes == 6) scan_row<T, 6>(a, logits, segment_max, top, sum);
            if (bytes == 10) scan_row<T, 10>(a, logits, segment_max, top, sum);
            if (bytes == 14) scan_row<T, 14>(a, logits, segment_max, top, sum);
        }
    }
    __shared__ float tops[kScanThreads / 32], sums[kScanThreads / 32];
    auto join = [](float& t, float& s, float t2, float s2) {
        const float n = fmaxf(t, t2);
        if (n > -INFINITY) {
            s = s * exp2_fast((t - n) * kLog2e) + s2 * exp2_fast((t2 - n) * kLog2e);
        } else {
            s += s2;
        }
        t = n;
    };
#pragma unroll
    for (uint32_t o = 16; o > 0; o /= 2) {
        const float t2 = __shfl_down_sync(kFullMask, top, o), s2 = __shfl_down_sync(kFullMask, sum, o);
        join(top, sum, t2, s2);
    }
    if (threadIdx.x % 32 == 0) {
        tops[threadIdx.x / 32] = top;
        sums[threadIdx.x / 32] = sum;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < kScanThreads / 32; ++w) join(top, sum, tops[w], sums[w]);
        a.partial[static_cast<size_t>(row) * a.splits + blockIdx.x] = make_float2(top, sum);
    }
}

template <typename T> __global__ void __launch_bounds__(kScanThreads) beam_scan_kernel(const BeamArgs a) { scan<T, false>(a); }
// ... with rows that start between 16-byte boundaries, 64 registers for four CTAs an SM: 512 rows of 151935 bf16 logits cost 21 us more than
// of 151936 (with three CTAs and requests a turn ahead 23), 128 rows of f32 5 more.
template <typename T> __global__ void __launch_bounds__(kScanThreads, 4) beam_scan_shifted_kernel(const BeamArgs a) { scan<T, true>(a); }

struct Candidate {
    double score;
    uint32_t index;
};
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) { return a.score > b.score || (a.score == b.score && a.index < b.index); }
// The upper half of a score as an integer of the same order (20 bits of mantissa; -0 below 0 only splits what is then compared whole).
__device__ __forceinline__ int score_key(double score) {
    const int h = __double2hiint(score + 0.0);
    return h ^ ((h >> 31) & 0x7fffffff);
}
constexpr int kNoKey = static_cast<int>(0x80000000);

struct MergeShared {
    Candidate candidates[kCandidates];
    Candidate segments[kMaxK], elements[kMaxK];
    Candidate best[kMergeThreads / 32];
    double base[kMaxBeams], top[kMaxBeams];  // a row's scores are (logit - top) + base: base = beam score - log of the sum below top
    uint8_t counts[kMaxBeams], ended[kMaxBeams];
    int low, high;
    uint32_t found;
};

// The best `k` (fewer, if fewer have a finite score) of the entries that each(use) hands to use(candidate), spread over the threads and
// the same ones in every pass, in order, into `out`; returns how many.  The k-th largest of the threads' best keys, found by
// bisection with one counting barrier a step, bounds the k-th best entry from below; what is not under it (a few more than k
// entries) is ranked by counting, in 64 bits.
template <typename Each>
__device__ __forceinline__ uint32_t select(MergeShared& sh, uint32_t k, Candidate* out, Each each) {
    int key = kNoKey;
    each([&](const Candidate& c) {
        if (c.score > -INFINITY) key = max(key, score_key(c.score));
    });
    if (threadIdx.x == 0) {
        sh.low = 0x7fffffff;
        sh.high = kNoKey;
        sh.found = 0;
    }
    const uint32_t threads = __syncthreads_count(key != kNoKey);
    int threshold = kNoKey + 1;  // every finite score
    if (threads >= k) {
        const int highest = __reduce_max_sync(kFullMask, key), lowest = __reduce_min_sync(kFullMask, key == kNoKey ? 0x7fffffff : key);
        if (threadIdx.x % 32 == 0) {
            atomicMax(&sh.high, highest);
            atomicMin(&sh.low, lowest);
        }
        __syncthreads();
        // at least k threads have `low` or more, fewer than k have more than `high`; a few steps short of the end it is near enough
        int low = sh.low, high = sh.high;
        for (int step = 0; step < 20 && low < high; ++step) {
            const int mid = static_cast<int>((static_cast<long long>(low) + high + 1) >> 1);
            if (static_cast<uint32_t>(__syncthreads_count(key >= mid)) >= k) low = mid;
            else high = mid - 1;
        }
        threshold = low;
    }
    each([&](const Candidate& c) {
        if (c.score > -INFINITY && score_key(c.score) >= threshold) {
            const uint32_t at = atomicAdd(&sh.found, 1u);
            if (at < kCandidates) sh.candidates[at] = c;
        }
    });
    __syncthreads();
    const uint32_t found = sh.found;
    if (found <= kCandidates) {
        for (uint32_t c = threadIdx.x; c < found; c += kMergeThreads) {
            const Candidate x = sh.candidates[c];
            uint32_t rank = 0;
            for (uint32_t t = 0; t < found; ++t) rank += before(sh.candidates[t], x);
            if (rank < k) out[rank] = x;
        }
        __syncthreads();
        return min(found, k);
    }
    // Too many to rank (long runs of equal scores): the next one in order, k times.
    Candidate last{INFINITY, 0};
    for (uint32_t r = 0; r < k; ++r) {
        Candidate next{-INFINITY, 0xffffffffu};
        each([&](const Candidate& c) {
            if (c.score > -INFINITY && before(last, c) && before(c, next)) next = c;
        });
        auto join = [&](uint32_t o) {
            const Candidate other{__shfl_xor_sync(kFullMask, next.score, o), __shfl_xor_sync(kFullMask, next.index, o)};
            if (before(other, next)) next = other;
        };
#pragma unroll
        for (uint32_t o = 16; o > 0; o /= 2) join(o);
        if (threadIdx.x % 32 == 0) sh.best[threadIdx.x / 32] = next;
        __syncthreads();
        next = sh.best[threadIdx.x % (kMergeThreads / 32)];
#pragma unroll
        for (uint32_t o = 16; o > 0; o /= 2) join(o);
        last = next;
        if (threadIdx.x == 0) out[r] = last;
        __syncthreads();
    }
    return k;  // (more than kCandidates >= k were found)
}

template <typename T>
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamArgs a) {
    extern __shared__ __align__(16) uint8_t raw[];
    MergeShared& sh = *reinterpret_cast<MergeShared*>(raw);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t batch = blockIdx.x, row0 = batch * a.beams;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    // the sum of exponentials of every row from its splits, in 64 bits
    for (uint32_t w = warp; w < a.beams; w += kMergeThreads / 32) {
        const uint32_t row = row0 + w;
        const bool ended = a.finished && __ldcg(a.finished + row) && isfinite(__ldcg(a.beam_scores + row));
        bool counts = row_counts(a, row);
        double base = __ldcg(a.beam_scores + row);
        float top = 0.0f;
        if (counts) {
            const float2* partial = a.partial + static_cast<size_t>(row) * a.splits;
            top = -INFINITY;
            for (uint32_t s = lane; s < a.splits; s += 32) top = fmaxf(top, __ldcg(partial + s).x);
#pragma unroll
            for (uint32_t o = 16; o > 0; o /= 2) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
            double sum = 0.0;
            for (uint32_t s = lane; s < a.splits; s += 32) {
                const float2 p = __ldcg(partial + s);
                if (p.y != 0.0f) sum += p.y * exp(static_cast<double>(p.x) - top);
            }
#pragma unroll
            for (uint32_t o = 16; o > 0; o /= 2) sum += __shfl_xor_sync(kFullMask, sum, o);
            // (the top stays apart: among logits of 3e38 a sum with it would lose the rest)
            const double below = log(sum);
            counts = isfinite(below) && isfinite(top);
            base -= below;
        }
        if (lane == 0) {
            sh.base[w] = base;
            sh.top[w] = top;
            sh.counts[w] = counts;
            sh.ended[w] = ended;
        }
    }
    __syncthreads();
    // The best segments: a row's maxima are read by a warp or several, eight a lane on their way; a finished beam is one entry, in the
    // place of its first segment.
    const float* maxima = a.segment_max + static_cast<size_t>(row0) * a.segments;
    constexpr uint32_t kWarps = kMergeThreads / 32, kFetch = 8;
    const uint32_t parts = (kWarps + a.beams - 1) / a.beams, per_part = (a.segments + parts - 1) / parts;
    const uint32_t segments = select(sh, a.k, sh.segments, [&](auto use) {
        for (uint32_t item = warp; item < a.beams * parts; item += kWarps) {
            const uint32_t w = item / parts, part = item - w * parts;
            if (!sh.counts[w]) {
                if (sh.ended[w] && part == 0 && lane == 0) use(Candidate{sh.base[w], w * a.segments});
                continue;
            }
            const double top = sh.top[w], base = sh.base[w];
            const uint32_t last = min((part + 1) * per_part, a.segments);
            for (uint32_t s = part * per_part + lane; s < last; s += 32 * kFetch) {
                float x[kFetch];
#pragma unroll
                for (uint32_t i = 0; i < kFetch; ++i) x[i] = s + 32 * i < last ? __ldcg(maxima + static_cast<size_t>(w) * a.segments + s + 32 * i) : -INFINITY;
#pragma unroll
                for (uint32_t i = 0; i < kFetch; ++i) use(Candidate{(x[i] - top) + base, w * a.segments + s + 32 * i});
            }
        }
    });
    // the best of their elements
    const uint32_t elements = select(sh, a.k, sh.elements, [&](auto use) {
        for (uint32_t j = threadIdx.x; j < segments * kSegment; j += kMergeThreads) {
            const uint32_t at = sh.segments[j / kSegment].index, w = at / a.segments, s = at - w * a.segments;
            if (sh.ended[w]) {
                if (j % kSegment == 0) use(Candidate{sh.base[w], w * a.vocab + a.pad_token});
                continue;
            }
            const T* logits = static_cast<const T*>(a.logits) + (row0 + w) * a.stride;
            const uint32_t token = s * kSegment + j % kSegment;
            if (token < a.vocab) use(Candidate{(logit_value(__ldcg(logits + token)) - sh.top[w]) + sh.base[w], w * a.vocab + token});
        }
    });
    for (uint32_t r = threadIdx.x; r < a.k; r += kMergeThreads) {
        uint32_t index = 0;
        float score = -INFINITY;
        if (r < elements) {
            index = sh.elements[r].index;
            score = static_cast<float>(sh.elements[r].score);
        } else {
            // candidates without a finite score, in order: the (r - elements)-th index that is not among the ones above
            index = r - elements;
            bool moved = true;
            while (moved) {  // (every taken index at or below it moves it on by one; it settles after `elements` steps at most)
                uint32_t taken = 0;
                for (uint32_t e = 0; e < elements; ++e) taken += sh.elements[e].index <= index;
                const uint32_t next = r - elements + taken;
                moved = next != index;
                index = next;
            }
        }
        const size_t at = static_cast<size_t>(batch) * a.k + r;
        a.out_scores[at] = score;
        a.out_parents[at] = static_cast<int32_t>(index / a.vocab);
        a.out_tokens[at] = static_cast<int32_t>(index % a.vocab);
    }
}

// ---- states ------------------------------------------------------------------------------------------------
// dst[batch][beam] = src[batch][parents[batch][beam]], several states in one launch.  Bound: HBM, every row read and written once (a
// row with several children comes out of L2 again).  A CTA copies a stretch of one row, four 16-byte pieces a thread on their way.
constexpr uint32_t kStates = 24;  // of a launch
constexpr uint32_t kCopyThreads = 256;
constexpr uint32_t kStretch = kCopyThreads * 4 * 16;
struct ReorderArgs {
    const uint8_t* src[kStates];
    uint8_t* dst[kStates];
    size_t row_bytes[kStates];
    const int32_t* parents;
    size_t parent_stride;
    uint32_t beams;
};
__global__ void __launch_bounds__(kCopyThreads) beam_reorder_kernel(const ReorderArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t row = blockIdx.x, batch = row / a.beams, beam = row - batch * a.beams;
    const size_t bytes = a.row_bytes[blockIdx.z];
    const int32_t parent = __ldcg(a.parents + batch * a.parent_stride + beam);
    if (parent < 0 || static_cast<uint32_t>(parent) >= a.beams) return;  // (no such beam: the row stays as it is)
    const uint8_t* src = a.src[blockIdx.z] + (static_cast<size_t>(batch) * a.beams + parent) * bytes;
    uint8_t* dst = a.dst[blockIdx.z] + static_cast<size_t>(row) * bytes;
    const bool wide = ((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) & 15) == 0;
    for (size_t at = static_cast<size_t>(blockIdx.y) * kStretch; at < bytes; at += static_cast<size_t>(gridDim.y) * kStretch) {
        const size_t left = bytes - at;
        size_t done = 0;
        if (wide) {
            uint4 q[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const size_t o = (j * kCopyThreads + threadIdx.x) * 16;
                if (o + 16 <= left) q[j] = __ldcg(reinterpret_cast<const uint4*>(src + at + o));
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const size_t o = (j * kCopyThreads + threadIdx.x) * 16;
                if (o + 16 <= left) *reinterpret_cast<uint4*>(dst + at + o) = q[j];
            }
            done = left / 16 * 16;
        }
        for (size_t o = done + threadIdx.x; o < left && o < kStretch; o += kCopyThreads) dst[at + o] = __ldcg(src + at + o);
    }
}

uint32_t segments_of(uint32_t vocab) { return (vocab + kSegment - 1) / kSegment; }
uint32_t vectors_of(uint32_t vocab, bool bf16) { return (vocab + (bf16 ? 7 : 3)) / (bf16 ? 8 : 4); }
// Splits of a row: a dozen CTAs an SM, so that the last ones do not leave most SMs idle, while a split keeps a few thousand logits.
uint32_t vectors_per_split(uint32_t rows, uint32_t vocab, bool bf16) {
    const uint32_t wanted = std::max(1u, (148u * 12u + rows - 1) / rows);
    const uint32_t per = (vectors_of(vocab, bf16) + wanted - 1) / wanted;
    return (per + kScanThreads - 1) / kScanThreads * kScanThreads;
}
uint32_t splits_of(uint32_t rows, uint32_t vocab, bool bf16) {
    const uint32_t per = vectors_per_split(rows, vocab, bf16);
    return (vectors_of(vocab, bf16) + per - 1) / per;
}
// Whether an output lies over a state, any state, or over another output: all are copied at once, and a row would be read or written
// after another copy had written there.  (States may share memory.)  In the order of addresses each output has to begin behind all
// that came before it, and each state behind the outputs.
bool outputs_overlap(const void* const* src, void* const* dst, const size_t* row_bytes, uint32_t count, size_t rows) {
    struct Span {
        uintptr_t begin, end;
        bool written;
    };
    std::unique_ptr<Span[]> spans(new (std::nothrow) Span[2 * static_cast<size_t>(count)]);
    if (!spans) return true;
    for (uint32_t i = 0; i < count; ++i) {
        const auto s = reinterpret_cast<uintptr_t>(src[i]), d = reinterpret_cast<uintptr_t>(dst[i]);
        spans[2 * i] = {s, s + row_bytes[i] * rows, false};
        spans[2 * i + 1] = {d, d + row_bytes[i] * rows, true};
    }
    std::sort(spans.get(), spans.get() + 2 * static_cast<size_t>(count), [](const Span& a, const Span& b) { return a.begin < b.begin; });
    uintptr_t written = 0, read = 0;
    for (size_t i = 0; i < 2 * static_cast<size_t>(count); ++i) {
        const Span& s = spans[i];
        if (s.begin < written || (s.written && s.begin < read)) return true;
        (s.written ? written : read) = std::max(s.written ? written : read, s.end);
    }
    return false;
}
bool beam_shape_ok(uint32_t batch, uint32_t beams, uint32_t vocab) {
    return batch != 0 && beams != 0 && beams <= kMaxBeams && vocab != 0 && batch <= 0xffffu / beams && vocab <= 0x7fffffffu / beams - 64;
}

}  // namespace
}  // namespace eider

using namespace eider;

extern "C" {

size_t eider_b200_beam_select_workspace_bytes(uint32_t batch, uint32_t beams, uint32_t vocab, int logits_are_bf16) {
    if (!beam_shape_ok(batch, beams, vocab)) return 0;
    const size_t rows = static_cast<size_t>(batch) * beams;
    return rows * (splits_of(batch * beams, vocab, logits_are_bf16) * sizeof(float2) + segments_of(vocab) * sizeof(float));
}

cudaError_t eider_b200_beam_select_on_stream(const void* logits, int logits_are_bf16, size_t row_stride, const float* beam_scores,
                                             const uint8_t* finished, uint32_t pad_token, float* out_scores, int32_t* out_parents,
                                             int32_t* out_tokens, uint32_t batch, uint32_t beams, uint32_t vocab, uint32_t k, void* workspace,
                                             size_t workspace_bytes, cudaStream_t stream) {
    if (!logits || !beam_scores || !out_scores || !out_parents || !out_tokens || !workspace || !beam_shape_ok(batch, beams, vocab) ||
        row_stride < vocab || k == 0 || k > kMaxK || k > static_cast<uint64_t>(beams) * vocab || (finished && pad_token >= vocab) ||
        (reinterpret_cast<uintptr_t>(logits) & (logits_are_bf16 ? 1 : 3)) != 0 || (reinterpret_cast<uintptr_t>(workspace) & 7) != 0 ||
        workspace_bytes < eider_b200_beam_select_workspace_bytes(batch, beams, vocab, logits_are_bf16))
        return cudaErrorInvalidValue;
    BeamArgs a{};
    const uint32_t rows = batch * beams;
    a.logits = logits;
    a.stride = row_stride;
    a.beam_scores = beam_scores;
    a.finished = finished;
    a.out_scores = out_scores;
    a.out_parents = out_parents;
    a.out_tokens = out_tokens;
    a.beams = beams;
    a.vocab = vocab;
    a.k = k;
    a.pad_token = pad_token;
    a.segments = segments_of(vocab);
    a.vectors_per_split = vectors_per_split(rows, vocab, logits_are_bf16);
    a.splits = splits_of(rows, vocab, logits_are_bf16);
    a.partial = static_cast<float2*>(workspace);
    a.segment_max = reinterpret_cast<float*>(a.partial + static_cast<size_t>(rows) * a.splits);
    const dim3 scan(a.splits, rows);
    const bool shifted = ((reinterpret_cast<uintptr_t>(logits) | row_stride * (logits_are_bf16 ? 2 : 4)) & 15) != 0;
    const auto scan_kernel = logits_are_bf16 ? (shifted ? beam_scan_shifted_kernel<uint16_t> : beam_scan_kernel<uint16_t>)
                                             : (shifted ? beam_scan_shifted_kernel<float> : beam_scan_kernel<float>);
    const cudaError_t st = launch_dependent(scan_kernel, scan, kScanThreads, 0, stream, a);
    if (st != cudaSuccess) return st;
    return logits_are_bf16 ? launch_dependent(beam_merge_kernel<uint16_t>, dim3(batch), kMergeThreads, sizeof(MergeShared), stream, a)
                           : launch_dependent(beam_merge_kernel<float>, dim3(batch), kMergeThreads, sizeof(MergeShared), stream, a);
}

cudaError_t eider_b200_beam_reorder_on_stream(const void* const* src, void* const* dst, const size_t* row_bytes, uint32_t count,
                                              const int32_t* parents, size_t parent_stride, uint32_t batch, uint32_t beams, cudaStream_t stream) {
    if (!src || !dst || !row_bytes || count == 0 || !parents || batch == 0 || beams == 0 || parent_stride < beams ||
        static_cast<uint64_t>(batch) * beams > 0x7fffffffu)
        return cudaErrorInvalidValue;
    for (uint32_t i = 0; i < count; ++i)
        if (!src[i] || !dst[i] || row_bytes[i] == 0) return cudaErrorInvalidValue;
    if (outputs_overlap(src, dst, row_bytes, count, static_cast<size_t>(batch) * beams)) return cudaErrorInvalidValue;
    for (uint32_t first = 0; first < count; first += kStates) {
        ReorderArgs a{};
        const uint32_t states = std::min(kStates, count - first);
        size_t longest = 0;
        for (uint32_t i = 0; i < states; ++i) {
            a.src[i] = static_cast<const uint8_t*>(src[first + i]);
            a.dst[i] = static_cast<uint8_t*>(dst[first + i]);
            a.row_bytes[i] = row_bytes[first + i];
            longest = std::max(longest, a.row_bytes[i]);
        }
        a.parents = parents;
        a.parent_stride = parent_stride;
        a.beams = beams;
        const uint32_t stretches = static_cast<uint32_t>(std::min<size_t>((longest + kStretch - 1) / kStretch, 1024));
        const cudaError_t st = launch_dependent(beam_reorder_kernel, dim3(batch * beams, stretches, states), kCopyThreads, 0, stream, a);
        if (st != cudaSuccess) return st;
    }
    return cudaSuccess;
}

}  // extern "C"
