// One token a row from given random numbers: ls_hip_sample_enqueue.
//
// e_i = exp((l_i - top) / T), w_i = e_i in whole steps of 2^-32. Ranked by (logit descending, id ascending) the
// kept tokens are a prefix of the ranking: everything above a cut logit, and of the tokens equal to it the
// first few by id. Weights of a set are summed as whole numbers, so no order of atomics changes a result; only the weight
// of a whole row (no filter, or top-p without top-k) is a sum of floats, chunk by chunk in a fixed order.
//
// One pass over the logits, in two launches. A workgroup of the first takes a chunk of a row and leaves its best token,
// the sum of its exponentials and, in order of id, its candidates: as many of its largest logits as the record holds.
// A workgroup of the second takes a row: it finds the cuts of top-k and of top-p among the candidates by radix
// selection (parts of the range of their 32-bit order, with the count and the weight of each). Whatever lies above the
// largest logit that is no candidate (`outside`) is known completely. Where a cut falls below:
//  - top-p alone: the chunks also left histograms of count and weight over bins of T / 16. They name the bin of
//    the cut, whose tokens are picked from the row (one pass of comparisons) and selected among; the chunks'
//    weights above the cut point to the chunk that holds the token, and only that is read again;
//  - otherwise (top-k beyond the candidates, a bin of more tokens than there is room for) the workgroup selects
//    over the whole row.
// Without filters the chunks' sums point to the chunk that holds the token.
//
// Bound by the waits between the steps of a workgroup: 256 rows of 50257 fp32 logits with top-k take 20 + 11 us for
// 51 MB (a greedy pick, which needs none of the steps, 13), one row of 32768 7 + 9. A row whose nucleus is wide costs
// most: 64 rows of 131072, each with settings of its own, 13 + 37 us. One launch, in which a row's last chunk went on
// with the row, gave the chunks half the waves (its registers): 73 us for 64 rows with top-k, where the first form in
// two took 28 (now 22). For a few rows, whose chunks do not fill the card with either, it was not measured.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cerrno>
#include "kernel_launch.h"
#include "leanstream_hip.h"
#include "wave_ops.h"

// Arrays that a closure reaches stay in registers only where it is inlined.
#define LS_INLINE __attribute__((always_inline))

namespace lsamd {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kMaxVocab = 1u << 20;   // sums stay below 2^52
constexpr uint32_t kMaxChunks = 128;       // of a row
constexpr uint32_t kCandidates = 4096;     // of a row, 8 a thread
constexpr uint32_t kChunkCandidates = 256; // of a chunk, at most
constexpr uint32_t kRowBlock = 256;        // rows of a launch
constexpr int kBins = 512;                 // steps of T / 16 down from a chunk's best logit: weights to e^-32
constexpr int kCountShift = 46;            // a bin: count << 46 | weight (at most 2^13 tokens of up to 2^32)
constexpr uint64_t kWeight = (1ull << kCountShift) - 1;
constexpr uint32_t kAll = 0xffffffffu;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_float(__bf16 x) { return (float)x; }

// Order of the logits as unsigned numbers; -0 and +0 are equal, NaN is -inf.
__device__ __forceinline__ uint32_t order_of(float l) {
    if (!(l == l)) l = -INFINITY;
    const uint32_t u = __float_as_uint(l + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t order) {
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}

// floor (or ceil) of total * fraction, the fraction in steps of 2^-24 (total < 2^52)
__device__ __forceinline__ uint64_t share(uint64_t total, float fraction, bool up) {
    const uint64_t m = fraction > 0.0f ? (uint64_t)((double)fminf(fraction, 1.0f) * 16777216.0) : 0;
    return m * (total >> 24) + ((m * (total & 0xffffff) + (up ? 0xffffff : 0)) >> 24);
}

// Exponentials of a row. log2(e) / T is held in two floats, and its product with the distance is split into
// whole and fraction before it is rounded: the error of e stays near one unit in its last place.
struct Scale {
    float hi, lo, bins;
    __device__ __forceinline__ explicit Scale(float temperature) {
        const double c = 1.4426950408889634 / (double)temperature;
        hi = (float)c;
        lo = hi < INFINITY ? (float)(c - (double)hi) : 0.0f;
        bins = fmaxf(fminf(16.0f / temperature, 3e38f), 0x1p-126f);   // never 0: inf * 0 has no place among the bins
    }
    // bin on the scale of all logits of a row, rising with the logit
    __device__ __forceinline__ float steps(float l) const { return fminf(fmaxf(floorf(l * bins), -1e9f), 1e9f); }
    __device__ __forceinline__ int bin(float l) const { return (int)steps(l); }
    // the smallest logit of bin b or above: a few units in the last place around b / bins
    __device__ __forceinline__ float first_of(int b) const {
        if (b <= -1000000000) return -INFINITY;
        if (b > 1000000000) return INFINITY;
        float v = (float)b / bins;
        for (int i = 0; i < 4 && steps(v) >= (float)b; ++i) v = nextafterf(v, -INFINITY);
        for (int i = 0; i < 8 && !(steps(v) >= (float)b); ++i) v = nextafterf(v, INFINITY);
        return v;
    }
    // exp((l - top) / T) 2^up for l <= top; 0 for -inf
    __device__ __forceinline__ float e(float l, float top, int up = 0) const {
        const float t = l - top;
        const float whole = fmaxf(rintf(t * hi), -200.0f);
        const float part = fmaf(t, hi, -whole) + t * lo;
        const float x = fmaxf(ldexpf(__builtin_amdgcn_exp2f(part), (int)whole + up), 0.0f);
        // equal also where both are infinite; NaN (-inf at an infinite temperature, an infinite scale) became 0
        return l == top ? ldexpf(1.0f, up) : x;
    }
    // weight in steps of 2^-32 from e 2^32; the best token's 2^32 is held as 2^32 - 1
    static __device__ __forceinline__ uint32_t weight_of(float e, bool best) {
        return (uint32_t)fminf(rintf(e), 4294967040.0f) | (best ? 255u : 0u);
    }
    __device__ __forceinline__ uint32_t weight(float l, float top) const { return weight_of(e(l, top, 32), l == top); }
};

// A prefix of the ranking: every order above `order`, and the first `ties` ids of those equal to it.
struct Cut {
    uint32_t order, ties;
};

struct Shared {
    uint64_t weights[256];
    uint32_t counts[256];
    uint64_t wave64[kWaves];
    double wave_sum[kWaves];
    uint32_t wave32[kWaves];
    float wave_float[kWaves];
    uint64_t before_weight;
    uint32_t before_count, digit, turn, token;
    // of the row's chunks
    double sums[kMaxChunks];
    uint64_t list[kMaxChunks];
    double unit[kMaxChunks];
    int shift[kMaxChunks];
    float tops[kMaxChunks];
    uint32_t held[kMaxChunks];
    uint64_t few[64];
};
struct ChunkShared {
    uint64_t bins[kBins];
    double wave_sum[kWaves];
    float wave_float[kWaves], wave_mean[kWaves];
    uint32_t wave32[kWaves], digit;
};

// Exclusive sum over the threads, and the total. The scratch array is free again after the next barrier.
template <class V>
__device__ __forceinline__ V block_before(V x, V* scratch, V* total) {
    const V upto = wave_upto(x);
    if ((threadIdx.x & 63) == 63) scratch[threadIdx.x >> 6] = upto;
    __syncthreads();
    V before = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        if (i == (int)(threadIdx.x >> 6)) before = sum;
        sum += scratch[i];
    }
    *total = sum;
    return before + upto - x;
}

// The shortest prefix within `limit` whose count reaches need_count or whose weight reaches need_weight, of the
// tokens with an order in [base, high] that each(f) hands to f(order, weight); all of `limit` if none does.
// kept: the weight of that prefix. Few: of at most 2^13 tokens, whose count and weight go into one word. A limit with
// fewer ties than there are must weigh need_weight. Every pass counts the 256 equal parts of the range and goes on with
// the one in which a sum is reached, until it is one logit or holds so few tokens that one wave ranks them.
template <bool Few, class Each>
__device__ __forceinline__ Cut select(const Each& each, uint32_t base, uint32_t high, Cut limit, uint32_t need_count,
                                      uint64_t need_weight, Shared& sh, uint64_t* kept) {
    uint64_t before_weight = 0;
    base = max(base, limit.order);
    for (;;) {
        const int shift = max(0, 24 - __clz((int)((high - base) | 1)));
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += kThreads) sh.weights[i] = 0, sh.counts[i] = 0;
        if (threadIdx.x == 0) sh.turn = 0;
        __syncthreads();
        each([&](uint32_t order, uint32_t weight) LS_INLINE {
            if (!weight || order < base || order > high) return;
            const uint32_t part = (order - base) >> shift;
            if constexpr (!Few) atomicAdd(&sh.counts[part], 1u);
            atomicAdd((unsigned long long*)&sh.weights[part], (Few ? 1ull << kCountShift : 0) + weight);
        });
        __syncthreads();
        // The first part from above at which one of the sums is reached: a lane takes four. Where a part is one
        // logit, only its ties count of the limit's own.
        if (threadIdx.x < 64) {
            const uint32_t lane = threadIdx.x;
            uint32_t n[4], c = 0;
            uint64_t w[4], s = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t d = 255 - 4 * lane - i;
                w[i] = sh.weights[d];
                n[i] = Few ? (uint32_t)(w[i] >> kCountShift) : sh.counts[d];
                if (Few) w[i] &= kWeight;
                if (shift == 0 && base + d == limit.order && n[i] > limit.ties)
                    w[i] = w[i] / n[i] * limit.ties, n[i] = limit.ties;
                c += n[i];
                s += w[i];
            }
            uint32_t c_before = wave_upto(c) - c;
            uint64_t s_before = wave_upto(s) - s;
            const uint64_t reached = __ballot(c_before + c >= need_count || s_before + s >= need_weight);
            const uint32_t at = reached ? (uint32_t)__ffsll((unsigned long long)reached) - 1 : 63u;
            if (lane == at) {
                uint32_t digit = 256;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (digit != 256) continue;
                    if (reached && n[i] && (c_before + n[i] >= need_count || s_before + w[i] >= need_weight))
                        digit = 255 - 4 * lane - i;
                    else c_before += n[i], s_before += w[i];
                }
                sh.digit = digit;
                sh.before_count = c_before;
                sh.before_weight = s_before;
            }
        }
        __syncthreads();
        const uint32_t digit = sh.digit;
        need_count -= need_count == kAll ? 0 : sh.before_count;
        need_weight -= need_weight == ~0ull ? 0 : sh.before_weight;
        before_weight += sh.before_weight;
        if (digit == 256) {   // not reached: all of the limit
            *kept = before_weight;
            return limit;
        }
        uint32_t n = Few ? (uint32_t)(sh.weights[digit] >> kCountShift) : sh.counts[digit];
        if (shift == 0) {
            const uint64_t one = (Few ? sh.weights[digit] & kWeight : sh.weights[digit]) / n;
            if (base + digit == limit.order) n = min(n, limit.ties);
            // ties needed for the count and for the weight, whichever is reached first
            const uint64_t ties = min(min((uint64_t)n, (uint64_t)need_count), (need_weight - 1) / one + 1);
            *kept = before_weight + ties * one;
            return Cut{base + digit, (uint32_t)ties};
        }
        base += digit << shift;
        high = base + min(high - base, (1u << shift) - 1);
        if (n > 64) continue;
        each([&](uint32_t order, uint32_t weight) LS_INLINE {
            if (!weight || order < base || order > high) return;
            const uint32_t i = atomicAdd(&sh.turn, 1u);
            sh.few[i] = (uint64_t)order << 32 | weight;
        });
        __syncthreads();
        if (threadIdx.x < 64) {
            const uint64_t own = threadIdx.x < n ? sh.few[threadIdx.x] : 0;
            const uint32_t order = (uint32_t)(own >> 32), weight = (uint32_t)own;
            uint32_t c = 0, equal = 0;
            uint64_t s = 0;
            for (uint32_t i = 0; i < n; ++i) {
                const uint32_t o = __builtin_amdgcn_readlane(order, i), w = __builtin_amdgcn_readlane(weight, i);
                if (o > order) ++c, s += w;
                equal += o == order;
            }
            if (order == limit.order) equal = min(equal, limit.ties);
            const bool reached = weight && c < need_count && s < need_weight &&
                                 (c + equal >= need_count || s + (uint64_t)equal * weight >= need_weight);
            const uint64_t at = __ballot(reached);
            if (threadIdx.x == (uint32_t)__ffsll((unsigned long long)at) - 1) {
                const uint64_t ties = min(min((uint64_t)equal, (uint64_t)(need_count - c)),
                                          (need_weight - s - 1) / weight + 1);
                sh.before_count = order;
                sh.before_weight = s + ties * weight;
                sh.turn = (uint32_t)ties;
            }
        }
        __syncthreads();
        *kept = before_weight + sh.before_weight;
        return Cut{sh.before_count, sh.turn};
    }
}

// What a chunk leaves for its row, in 8-byte words: its best token (order << 32 | ~id), the sum of exp((l - top) /
// T) with top the chunk's, the number of candidates and the largest logit that is none (-inf: there is none);
// then the candidates (order << 32 | id) in order of id, then the bins.
constexpr int kHead = 3;

template <class T>
struct Vec8 {
    typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

struct RowArgs {
    uint32_t chunks, room, words;   // of a row; candidates of a chunk; 8-byte words of a chunk's record
};

// The token of the row whose kept tokens, in order of id, are those above the cut and its first ties, with
// e >= min_p: over all of the row's logits.
template <class T>
__device__ __forceinline__ void draw_from_row(const T* logits, uint32_t vocab, float top, const Scale& scale, Cut cut,
                                              float min_p, float uniform, Shared& sh, uint32_t* token,
                                              uint64_t* total) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t stretch = ((vocab + kWaves - 1) / kWaves + 63) / 64 * 64;
    const uint32_t begin = min(wave * stretch, vocab), end = min(begin + stretch, vocab);
    uint64_t above = 0;
    uint32_t ties = 0, tie_weight = 0;
    for (uint32_t i = begin + lane; i < end; i += 64) {
        const float l = to_float(logits[i]);
        const uint32_t o = order_of(l);
        if (o < cut.order || !(scale.e(l, top) >= min_p)) continue;
        if (o == cut.order) ++ties, tie_weight = scale.weight(l, top);
        else above += scale.weight(l, top);
    }
    ties = wave_sum(ties);
    tie_weight = wave_max(tie_weight, 0u);
    above = wave_sum(above);
    __syncthreads();
    if (lane == 0) sh.wave32[wave] = ties;
    __syncthreads();
    uint32_t ties_left = cut.ties;
    for (uint32_t i = 0; i < wave; ++i) ties_left -= min(ties_left, sh.wave32[i]);
    if (lane == 0) sh.wave64[wave] = above + (uint64_t)min(ties, ties_left) * tie_weight;
    __syncthreads();
    uint64_t sum = 0, before = 0;
    for (uint32_t i = 0; i < kWaves; ++i) {
        if (i == wave) before = sum;
        sum += sh.wave64[i];
    }
    const uint64_t target = min(share(sum, uniform, false), sum - 1);
    if (target >= before && target < before + sh.wave64[wave]) {   // this wave's stretch holds the token
        for (uint32_t i0 = begin; i0 < end; i0 += 64) {
            const uint32_t i = i0 + lane;
            uint32_t w = 0;
            bool tie = false;
            if (i < end) {
                const float l = to_float(logits[i]);
                const uint32_t o = order_of(l);
                const bool in = o >= cut.order && scale.e(l, top) >= min_p;
                tie = in && o == cut.order;
                if (in) w = scale.weight(l, top);
            }
            const uint64_t tie_lanes = __ballot(tie);
            if (tie && (uint32_t)__popcll(tie_lanes & ((1ull << lane) - 1)) >= ties_left) w = 0;
            ties_left -= min(ties_left, (uint32_t)__popcll(tie_lanes));
            const uint64_t upto = wave_upto((uint64_t)w);
            const uint64_t found = __ballot(before + upto > target);
            if (found) {
                if (lane == 0) sh.token = i0 + (uint32_t)__ffsll((unsigned long long)found) - 1;
                break;
            }
            before += from_lane(upto, 63);
        }
    }
    __syncthreads();
    *token = sh.token;
    *total = sum;
}

// The token of a chunk at which the running weight of its kept tokens (units of the row's best one) passes
// `rest`; ties_before: tokens equal to the cut in earlier chunks.
template <class T, uint32_t Chunk>
__device__ __forceinline__ uint32_t draw_from_chunk(const T* logits, uint32_t vocab, uint32_t chunk, float top,
                                                    const Scale& scale, Cut cut, uint32_t ties_before, double rest,
                                                    Shared& sh) {
    constexpr uint32_t kEach = Chunk / kThreads;
    const uint32_t from = chunk * Chunk + threadIdx.x * kEach;
    float x[kEach];
    uint32_t o[kEach], ties = 0;
#pragma unroll
    for (uint32_t v = 0; v < kEach; v += 8) {
        if (from + v + 8 <= vocab) {
            const typename Vec8<T>::type y = *(const typename Vec8<T>::type*)(logits + from + v);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[v + j] = to_float(y[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[v + j] = from + v + j < vocab ? to_float(logits[from + v + j]) : -INFINITY;
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        o[j] = order_of(x[j]);
        x[j] = x[j] > -INFINITY && o[j] >= cut.order ? scale.e(x[j], top) : 0.0f;
        ties += o[j] == cut.order;
    }
    uint32_t chunk_ties;
    uint32_t tie = ties_before + block_before(ties, sh.wave32, &chunk_ties);
    double thread_sum = 0.0;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        if (o[j] == cut.order && tie++ >= cut.ties) x[j] = 0.0f;
        thread_sum += x[j];
    }
    double chunk_sum;
    double before = block_before(thread_sum, sh.wave_sum, &chunk_sum);
    // `rest` and these sums are rounded apart: the last token with weight takes what is left
    uint32_t first = kAll, last = 0;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        before += x[j];
        if (x[j] > 0.0f) {
            if (before > rest) first = min(first, from + j);
            last = from + j;
        }
    }
    first = wave_min(first, kAll);
    last = wave_max(last, 0u);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave32[threadIdx.x >> 6] = first, sh.wave64[threadIdx.x >> 6] = last;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        first = min(first, sh.wave32[i]);
        last = max(last, (uint32_t)sh.wave64[i]);
    }
    return min(first, last);
}

// A row's settings.
struct Settings {
    float temperature, top_p, min_p;
    uint32_t top_k;
    bool greedy, by_count, by_weight;
    bool filtered;   // by count, weight or chance
    bool summed;     // needs the sum of all exponentials
    bool binned;     // may need the histograms
    __device__ __forceinline__ Settings(const ls_hip_sample& a, uint32_t r) {
        temperature = a.temperature ? a.temperature[r] : 1.0f;
        const int32_t k = a.top_k ? a.top_k[r] : 0;
        top_k = k > 0 ? (uint32_t)k : kAll;
        top_p = a.top_p ? a.top_p[r] : 1.0f;
        min_p = a.min_p ? fminf(a.min_p[r], 1.0f) : 0.0f;
        greedy = !(temperature > 0.0f);
        if (greedy) temperature = 1.0f;
        by_count = top_k < a.vocab;
        by_weight = top_p < 1.0f;
        filtered = !greedy && (by_count || by_weight || min_p > 0.0f);
        summed = !greedy && !by_count && (by_weight || !filtered);
        binned = summed && by_weight;
    }
};

template <class T, int Vecs>
__global__ __launch_bounds__(kThreads) void sample_chunk_kernel(const ls_hip_sample a, const RowArgs rows) {
    constexpr uint32_t kChunk = 8 * Vecs * kThreads;
    __shared__ ChunkShared sh;
    __shared__ __align__(16) uint8_t marks[kChunk / 8];
    const uint32_t r = blockIdx.y, c = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* logits = (const T*)a.logits + (int64_t)r * a.row_stride;
    const uint32_t begin = c * kChunk, size = min(a.vocab - begin, kChunk);
    const Settings set(a, r);
    const bool greedy = set.greedy, filtered = set.filtered, summed = set.summed, binned = set.binned;
    const Scale scale(set.temperature);

    // element 8 (v kThreads + thread) + j
    float l[Vecs][8], high = -INFINITY;
#pragma unroll
    for (int v = 0; v < Vecs; ++v) {
        const uint32_t i = 8 * (v * kThreads + threadIdx.x);
        if (i + 8 <= size) {
            const typename Vec8<T>::type x = *(const typename Vec8<T>::type*)(logits + begin + i);
#pragma unroll
            for (int j = 0; j < 8; ++j) l[v][j] = to_float(x[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) l[v][j] = i + j < size ? to_float(logits[begin + i + j]) : -INFINITY;
        }
    }
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
#pragma unroll
    for (int v = 0; v < Vecs; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) high = fmaxf(high, l[v][j]);
    // the best logit, and the mean of the threads' best ones: few logits of a chunk lie above that
    float chunk_top = high, mean = high > -INFINITY ? high : 0.0f, some = high > -INFINITY ? 1.0f : 0.0f;
    chunk_top = wave_max(chunk_top, -INFINITY);
    mean = wave_sum(mean);
    some = wave_sum(some);
    if (lane == 0) sh.wave_float[wave] = chunk_top, sh.wave_mean[wave] = mean, sh.wave32[wave] = (uint32_t)some;
    __syncthreads();
    mean = 0.0f, some = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        chunk_top = fmaxf(chunk_top, sh.wave_float[i]);
        mean += sh.wave_mean[i];
        some += (float)sh.wave32[i];
    }
    mean /= some;
    if (!(mean < chunk_top)) mean = -INFINITY;   // all alike, infinite or none: any
    uint32_t best_at = kAll;
    if (high == chunk_top)   // its lowest id
#pragma unroll
        for (int v = 0; v < Vecs; ++v)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (l[v][j] == chunk_top) best_at = min(best_at, begin + 8 * (v * kThreads + threadIdx.x) + j);
    best_at = wave_min(best_at, kAll);
    __syncthreads();
    if (lane == 0) sh.wave32[wave] = best_at;

    uint64_t* record = (uint64_t*)a.workspace + ((uint64_t)r * rows.chunks + c) * rows.words;
    const int top_bin = scale.bin(chunk_top);
    double sum = 0.0;
    if (summed) {
        float mine = 0.0f;
#pragma unroll
        for (int v = 0; v < Vecs; ++v)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = l[v][j];
                if (!(x > -INFINITY)) continue;
                const float e = scale.e(x, chunk_top, 32);
                mine += e;
                const int down = top_bin - scale.bin(x);
                if (binned && down < kBins)
                    atomicAdd((unsigned long long*)&sh.bins[down], 
                              1ull << kCountShift | scale.weight_of(e, x == chunk_top));
            }
        sum = wave_sum((double)mine * 0x1p-32);
        if (lane == 0) sh.wave_sum[wave] = sum;
    } else if (!greedy && filtered) {
        // few of a wave's logits exceed the mean: they are marked first and then taken together
        uint32_t hits = 0;
#pragma unroll
        for (int v = 0; v < Vecs; ++v)
#pragma unroll
            for (int j = 0; j < 8; ++j) hits |= (uint32_t)(l[v][j] > mean) << (8 * v + j);
        while (hits) {
            const uint32_t at = __ffs(hits) - 1;
            hits &= hits - 1;
            const uint32_t from = begin + 8 * (at / 8 * kThreads + threadIdx.x) + at % 8;
            const int down = top_bin - scale.bin(to_float(logits[from]));
            if (down < kBins) atomicAdd((unsigned long long*)&sh.bins[down], 1ull << kCountShift);
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) best_at = min(best_at, sh.wave32[i]);
    const uint64_t best_of_chunk = (uint64_t)order_of(chunk_top) << 32 | (uint32_t)~best_at;
    if (summed) {
        sum = 0.0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) sum += sh.wave_sum[i];
        if (threadIdx.x == 0) record[1] = __builtin_bit_cast(uint64_t, sum);
    }
    if (!greedy && filtered) {
        // bins that fit into the record, as many as possible; where only what exceeds the mean was counted, the bins
        // wholly above it
        if (wave == 0) {
            uint32_t n = 0, fit = 0;
#pragma unroll
            for (int i = 0; i < kBins / 64; ++i) n += (uint32_t)(sh.bins[kBins / 64 * lane + i] >> kCountShift);
            uint32_t upto = wave_upto(n) - n;
#pragma unroll
            for (int i = 0; i < kBins / 64; ++i)
                fit += (upto += (uint32_t)(sh.bins[kBins / 64 * lane + i] >> kCountShift)) <= rows.room;
            fit = wave_sum(fit);
            if (lane == 0)
                sh.digit = summed || mean == -INFINITY
                               ? fit : min(fit, (uint32_t)max(0, min(top_bin - scale.bin(mean), kBins)));
        }
        __syncthreads();
        const int bins = (int)sh.digit;
        if (binned)
            for (int i = threadIdx.x; i < kBins; i += kThreads) record[kHead + rows.room + i] = sh.bins[i];
        float outside = -INFINITY;
        const float least = scale.first_of(top_bin - bins + 1);
#pragma unroll
        for (int v = 0; v < Vecs; ++v) {
            uint32_t mark = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = l[v][j];
                const bool in = x >= least && x > -INFINITY;
                mark |= (uint32_t)in << j;
                outside = fmaxf(outside, in ? -INFINITY : x);
            }
            marks[v * kThreads + threadIdx.x] = (uint8_t)mark;
        }
        outside = wave_max(outside, -INFINITY);
        if (lane == 0) sh.wave_float[wave] = outside;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWaves; ++i) outside = fmaxf(outside, sh.wave_float[i]);
        // candidates in order of id: a thread takes 32 elements' marks
        uint32_t word = threadIdx.x < kChunk / 32 ? ((const uint32_t*)marks)[threadIdx.x] : 0u, total;
        uint32_t at = block_before((uint32_t)__popc(word), sh.wave32, &total);
        // Bins beyond 2^24 (a tiny temperature) are not exact and infinite logits share the last: a chunk whose
        // candidates would not fit leaves none.
        if (total > rows.room) word = 0, total = 0, outside = chunk_top;
        while (word) {
            const uint32_t id = begin + 32 * threadIdx.x + __ffs(word) - 1;
            word &= word - 1;
            record[kHead + at++] = (uint64_t)order_of(to_float(logits[id])) << 32 | id;
        }
        if (threadIdx.x == 0) record[2] = (uint64_t)total << 32 | __float_as_uint(outside);
    }
    if (threadIdx.x == 0) record[0] = best_of_chunk;
}

template <class T, int Vecs>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(const ls_hip_sample a, const RowArgs rows) {
    constexpr uint32_t kChunk = 8 * Vecs * kThreads;
    __shared__ Shared sh;
    const uint32_t r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* logits = (const T*)a.logits + (int64_t)r * a.row_stride;
    const Settings set(a, r);
    const bool greedy = set.greedy, filtered = set.filtered, by_count = set.by_count, by_weight = set.by_weight;
    const float top_p = set.top_p, min_p = set.min_p, temperature = set.temperature;
    const Scale scale(temperature);
    const uint32_t words = rows.words;
    uint64_t* record = (uint64_t*)a.workspace + (uint64_t)r * rows.chunks * words;

    // threads 0 .. chunks - 1 hold a record each; every thread takes some of the slots for candidates
    const bool mine = threadIdx.x < rows.chunks;
    uint64_t best = mine ? record[threadIdx.x * words] : 0;
    const uint64_t tail = mine && filtered ? record[threadIdx.x * words + 2] : (uint64_t)__float_as_uint(-INFINITY);
    const double sum = mine && set.summed ? __builtin_bit_cast(double, record[threadIdx.x * words + 1]) : 0.0;
    const uint64_t own = best;
    best = wave_max(best, (uint64_t)0);
    if (lane == 0) sh.wave64[wave] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) best = max(best, sh.wave64[i]);
    const uint32_t best_id = ~(uint32_t)best;
    const float top = logit_of((uint32_t)(best >> 32));
    if (greedy || !(top > -INFINITY)) {
        if (threadIdx.x == 0) {
            const bool none = !(top > -INFINITY);
            a.tokens[r] = none ? -1 : (int32_t)best_id;
            if (a.logprob) a.logprob[r] = none ? -INFINITY : 0.0f;
        }
        return;
    }
    float outside = __uint_as_float((uint32_t)tail);
    outside = wave_max(outside, -INFINITY);
    if (lane == 0) sh.wave_float[wave] = outside;
    if (mine) {
        sh.tops[threadIdx.x] = logit_of((uint32_t)(own >> 32));
        sh.sums[threadIdx.x] = sum;
        sh.held[threadIdx.x] = (uint32_t)(tail >> 32);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) outside = fmaxf(outside, sh.wave_float[i]);

    // the row's sum, in units of its best token
    double part = 0.0;
    if (mine) part = sum * (double)scale.e(sh.tops[threadIdx.x], top);
    double row_sum;
    block_before(part, sh.wave_sum, &row_sum);
    uint32_t token;
    double kept;   // weight of the kept tokens in units of the best one
    const Cut all{0, kAll};
    // The token of the row, thread c holding the kept weight of chunk c (and the ties of earlier ones): the chunk in
    // which the running sum passes uniform * sum, then the token in it.
    auto pick = [&](double part, Cut cut, uint32_t ties_before, double* sum) LS_INLINE -> uint32_t {
        __syncthreads();
        const double before = block_before(part, sh.wave_sum, sum);
        const float u = a.uniform[r] > 0.0f ? fminf(a.uniform[r], 1.0f) : 0.0f;
        const double target = fmin((double)u * *sum, *sum * (1.0 - 0x1p-52));
        if (threadIdx.x == 0) sh.token = 0;
        __syncthreads();
        // the last chunk with weight that starts at or before the target
        if (mine && part > 0.0 && before <= target) atomicMax(&sh.token, threadIdx.x);
        __syncthreads();
        const uint32_t chunk = sh.token;
        if (threadIdx.x == chunk) sh.wave_sum[0] = target - before, sh.before_count = ties_before;
        __syncthreads();
        const double rest = sh.wave_sum[0];
        ties_before = sh.before_count;
        __syncthreads();
        return draw_from_chunk<T, kChunk>(logits, a.vocab, chunk, top, scale, cut, ties_before, rest, sh);
    };

    if (!filtered) {
        token = pick(part, all, 0, &kept);
    } else {
        // ---- candidates, in order of id: slots thread * kSlots + i
        constexpr uint32_t kSlots = kCandidates / kThreads;
        uint32_t order[kSlots], id[kSlots], weight[kSlots];
        uint64_t slots[kSlots];
        uint32_t chunk = threadIdx.x * kSlots / rows.room, at = threadIdx.x * kSlots % rows.room;
#pragma unroll
        for (uint32_t i = 0; i < kSlots; ++i) {
            slots[i] = chunk < rows.chunks && at < sh.held[chunk] ? record[chunk * words + kHead + at] : 0;
            if (++at == rows.room) at = 0, ++chunk;
        }
#pragma unroll
        for (uint32_t i = 0; i < kSlots; ++i) {
            order[i] = (uint32_t)(slots[i] >> 32);
            id[i] = (uint32_t)slots[i];
            weight[i] = slots[i] ? scale.weight(logit_of(order[i]), top) : 0;
        }
        // what is no candidate does not matter if it weighs nothing
        // orders below this weigh nothing
        const uint32_t low = order_of(top - 23.0f * temperature), high = order_of(top);
        const uint32_t edge = outside > -INFINITY && scale.weight(outside, top) ? order_of(outside) : 0;
        auto candidates = [&](auto f) LS_INLINE {
#pragma unroll
            for (uint32_t i = 0; i < kSlots; ++i) f(order[i], weight[i]);
        };
        auto everything = [&](auto f) LS_INLINE {
            for (uint32_t i = threadIdx.x; i < a.vocab; i += kThreads) {
                const float v = to_float(logits[i]);
                f(order_of(v), v > -INFINITY ? scale.weight(v, top) : 0u);
            }
        };
        auto above = [edge](Cut x) { return x.order > edge || !edge; };
        Cut cut = all;
        uint64_t total = (uint64_t)(row_sum * 4294967296.0);
        bool known = by_count || by_weight || !edge;   // every kept token is a candidate
        if (by_count) {
            cut = select<true>(candidates, max(low, edge + 1), high, cut, set.top_k, ~0ull, sh, &total);
            known = above(cut);
        }
        const bool open = !known && by_weight;   // the weight that top-p takes its share of is not known
        if (by_weight && known) {
            const uint64_t limit = share(total, top_p, true);
            cut = select<true>(candidates, max(low, edge + 1), high, cut, kAll, limit ? limit : 1, sh, &total);
            known = above(cut);
        }
        // Where the cut lies below, min-p may still leave out whatever is no candidate: it then decides alone.
        if (!known && !open && !(scale.e(outside, top) >= min_p)) known = true, cut = all;
        // Top-p by the chunks' bins: false where the bin of the cut holds more tokens than there are slots, or where
        // min-p cuts above it.
        double bin_kept = 0.0;
        auto cut_in_bins = [&]() LS_INLINE -> bool {
            const int row_bin = scale.bin(top);
            const double limit = (double)fmaxf(top_p, 0.0f) * row_sum;
            // a chunk's bins begin `shift` bins below the row's, in units of the chunk's best token
            if (mine) {
                const float its = sh.tops[threadIdx.x];
                sh.shift[threadIdx.x] = its > -INFINITY ? row_bin - scale.bin(its) : kBins;
                sh.unit[threadIdx.x] = 0x1p-32 * (double)scale.e(its, top);
            }
            __syncthreads();
            // thread b: bin b of the row, 16 chunks' loads at a time
            uint32_t n = 0;
            double w = 0.0;
            for (uint32_t c0 = 0; c0 < rows.chunks; c0 += 16) {
                uint64_t x[16];
#pragma unroll
                for (uint32_t c = 0; c < 16; ++c) {
                    const uint32_t at = min(c0 + c, rows.chunks - 1);
                    x[c] = record[at * words + kHead + rows.room + max((int)threadIdx.x - sh.shift[at], 0)];
                }
#pragma unroll
                for (uint32_t c = 0; c < 16; ++c) {
                    if (c0 + c >= rows.chunks || (int)threadIdx.x < sh.shift[c0 + c]) continue;
                    n += (uint32_t)(x[c] >> kCountShift);
                    w += (double)(x[c] & kWeight) * sh.unit[c0 + c];
                }
            }
            double all_bins;
            const double before = block_before(w, sh.wave_sum, &all_bins);
            if (threadIdx.x == 0) sh.token = kAll, sh.turn = 0;
            __syncthreads();
            if (n && before < limit && before + w >= limit) atomicMin(&sh.token, threadIdx.x);
            __syncthreads();
            const uint32_t bin = sh.token;
            if (bin == kAll) return false;
            if (threadIdx.x == bin) sh.before_weight = (uint64_t)((limit - before) * 4294967296.0), sh.before_count = n;
            __syncthreads();
            if (sh.before_count > kCandidates) return false;
            const uint64_t need = sh.before_weight;
            // The ids of its tokens, in any order, into the slots of the candidates (which are all read). A thread
            // marks what it finds among 64 logits before it takes slots: one by one, the few hits of every wave would
            // each wait for the counter.
            const float least = scale.first_of(row_bin - (int)bin), beyond = scale.first_of(row_bin - (int)bin + 1);
            auto slot_at = [&](uint32_t slot) LS_INLINE {
                return record + slot / rows.room * words + kHead + slot % rows.room;
            };
            constexpr uint32_t kDeep = 8;
            const uint32_t room = rows.room * rows.chunks, whole = a.vocab / 8;
            for (uint32_t i0 = threadIdx.x; i0 <= whole; i0 += kDeep * kThreads) {
                typename Vec8<T>::type x[kDeep];
#pragma unroll
                for (uint32_t d = 0; d < kDeep; ++d) {
                    const uint32_t i = i0 + d * kThreads;
                    if (i < whole) x[d] = *(const typename Vec8<T>::type*)(logits + 8 * i);
                    else
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[d][j] = 8 * i + j < a.vocab ? logits[8 * i + j] : (T)-INFINITY;
                }
                uint64_t hits = 0;
#pragma unroll
                for (uint32_t d = 0; d < kDeep; ++d)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float v = to_float(x[d][j]);
                        hits |= (uint64_t)(v >= least && v < beyond) << (8 * d + j);
                    }
                while (hits) {
                    const uint32_t at = __ffsll((unsigned long long)hits) - 1, slot = atomicAdd(&sh.turn, 1u);
                    hits &= hits - 1;
                    if (slot < room) *slot_at(slot) = 8 * (i0 + at / 8 * kThreads) + at % 8;
                }
            }
            __syncthreads();   // and their stores, for this workgroup
            const uint32_t held = sh.turn;
            if (held > room) return false;
            uint32_t lowest = kAll, highest = 0;
#pragma unroll
            for (uint32_t i = 0; i < kSlots; ++i) {
                const uint32_t slot = i * kThreads + threadIdx.x;
                id[i] = slot < held ? (uint32_t)*slot_at(slot) : 0;
            }
#pragma unroll
            for (uint32_t i = 0; i < kSlots; ++i) {
                const bool in = i * kThreads + threadIdx.x < held;
                const float v = in ? to_float(logits[id[i]]) : 0.0f;
                order[i] = in ? order_of(v) : 0;
                weight[i] = in ? scale.weight(v, top) : 0;
                if (weight[i]) lowest = min(lowest, order[i]), highest = max(highest, order[i]);
            }
            lowest = wave_min(lowest, kAll);
            highest = wave_max(highest, 0u);
            if (lane == 0) sh.wave32[wave] = lowest, sh.wave64[wave] = highest;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kWaves; ++i) {
                lowest = min(lowest, sh.wave32[i]);
                highest = max(highest, (uint32_t)sh.wave64[i]);
            }
            if (!highest) return false;
            uint64_t of_list;
            cut = select<true>(candidates, lowest, highest, all, kAll, need ? need : 1, sh, &of_list);
            if (!cut.order) cut = Cut{lowest, kAll};   // not reached, by a rounding of the bins' sums: all of the bin
            if (min_p > 0.0f && !(scale.e(logit_of(cut.order), top) >= min_p)) return false;
            // kept weight of every chunk: its bins above, and what the list holds of it
            __syncthreads();
            if (threadIdx.x < rows.chunks) sh.list[threadIdx.x] = 0, sh.held[threadIdx.x] = 0;
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < kSlots; ++i) {
                if (weight[i] && order[i] > cut.order)
                    atomicAdd((unsigned long long*)&sh.list[id[i] / kChunk], (unsigned long long)weight[i]);
                if (weight[i] && order[i] == cut.order) atomicAdd(&sh.held[id[i] / kChunk], 1u);
            }
            for (uint32_t c = wave; c < rows.chunks; c += kWaves) {
                const uint64_t* bins = record + c * words + kHead + rows.room;
                const int above = (int)bin - sh.shift[c];
                double x = 0.0;
#pragma unroll
                for (int b = 0; b < kBins; b += 64) {
                    const uint64_t w = bins[b + lane];
                    if (b + (int)lane < above) x += (double)(w & kWeight);
                }
                x *= sh.unit[c];
                x = wave_sum(x);
                if (lane == 0) sh.sums[c] = x;
            }
            __syncthreads();
            const uint32_t ties = mine ? sh.held[threadIdx.x] : 0;
            uint32_t all_ties;
            const uint32_t ties_before = block_before(ties, sh.wave32, &all_ties);
            double part = 0.0;
            if (mine) {
                const uint32_t admitted = min(ties, cut.ties - min(cut.ties, ties_before));
                const uint64_t tied = (uint64_t)admitted * scale.weight(logit_of(cut.order), top);
                part = sh.sums[threadIdx.x] + (double)(sh.list[threadIdx.x] + tied) * 0x1p-32;
            }
            token = pick(part, cut, ties_before, &bin_kept);
            return true;
        };
        uint64_t sum64;
        if (known) {
            uint32_t ties = 0;
#pragma unroll
            for (uint32_t i = 0; i < kSlots; ++i) {
                if (order[i] < cut.order || !(scale.e(logit_of(order[i]), top) >= min_p)) weight[i] = 0;
                ties += weight[i] && order[i] == cut.order;
            }
            uint32_t all_ties;
            __syncthreads();
            uint32_t tie = block_before(ties, sh.wave32, &all_ties);
            uint64_t thread_sum = 0;
#pragma unroll
            for (uint32_t i = 0; i < kSlots; ++i) {
                if (weight[i] && order[i] == cut.order && tie++ >= cut.ties) weight[i] = 0;
                thread_sum += weight[i];
            }
            uint64_t before = block_before(thread_sum, sh.wave64, &sum64);
            const uint64_t target = min(share(sum64, a.uniform[r], false), sum64 - 1);
            if (target >= before && target < before + thread_sum) {
#pragma unroll
                for (uint32_t i = 0; i < kSlots; ++i) {
                    if (weight[i] && target >= before && target < before + weight[i]) sh.token = id[i];
                    before += weight[i];
                }
            }
            __syncthreads();
            token = sh.token;
            kept = (double)sum64 * 0x1p-32;
        } else if (set.binned && cut_in_bins()) {
            kept = bin_kept;
        } else {
            cut = all;
            if (by_count || by_weight)
                cut = select<false>(everything, low, high, cut, by_count ? set.top_k : kAll, ~0ull, sh, &total);
            if (by_weight) {
                const uint64_t limit = share(total, top_p, true);
                cut = select<false>(everything, low, high, cut, kAll, limit ? limit : 1, sh, &total);
            }
            draw_from_row(logits, a.vocab, top, scale, cut, min_p, a.uniform[r], sh, &token, &sum64);
            kept = (double)sum64 * 0x1p-32;
        }
    }
    if (threadIdx.x == 0) {
        a.tokens[r] = (int32_t)token;
        // from the exponent itself: a small weight's rounding does not show in its logarithm
        const float v = to_float(logits[token]);
        if (a.logprob) a.logprob[r] = (v == top ? 0.0f : (v - top) / temperature) - (float)log(kept);
    }
}

bool aligned(const void* p, uintptr_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

int check(const ls_hip_sample& a) {
    if (a.rows && (!a.logits || !a.uniform || !a.tokens || !a.vocab)) return EINVAL;
    if (a.dtype > LS_TYPE_F32) return EINVAL;
    if (!aligned(a.logits, a.dtype == LS_TYPE_F32 ? 4 : 2) || a.row_stride < 0) return EINVAL;
    for (const void* p : {(const void*)a.uniform, (const void*)a.temperature, (const void*)a.top_k,
                          (const void*)a.top_p, (const void*)a.min_p, (const void*)a.tokens, (const void*)a.logprob})
        if (!aligned(p, 4)) return EINVAL;
    if (!aligned(a.workspace, 16)) return EINVAL;
    if (a.vocab > kMaxVocab || a.rows > 0x7fffffffu) return ENOTSUP;
    return 0;
}

// Chunks of 4096 logits while the rows are few (less than one workgroup a compute unit with twice as many), of 8192
// otherwise: top-p of one row of 32768 15.4 us with 4096 and 16.3 with 8192, of 131072 16.7 and 17.7; of 64 rows of
// 131072 30.0 and 26.6. A row's candidates are shared out evenly.
RowArgs plan_rows(const ls_hip_sample& a, int* vecs) {
    RowArgs p{};
    const uint32_t twice = (a.vocab + 16 * kThreads - 1) / (16 * kThreads);
    *vecs = a.vocab <= 64 * 8 * kThreads && (uint64_t)a.rows * twice < 256 ? 1 : 2;
    const uint32_t chunk = 8 * *vecs * kThreads;
    p.chunks = (a.vocab + chunk - 1) / chunk;
    p.room = std::min(kCandidates / p.chunks, kChunkCandidates);
    p.words = kHead + p.room + kBins;
    return p;
}

template <class T>
hipError_t launch(ls_hip_sample a, hipStream_t st) {
    int vecs;
    const RowArgs p = plan_rows(a, &vecs);
    const uint32_t rows = a.rows;
    for (uint32_t r = 0; r < rows; r += kRowBlock) {
        const dim3 grid(p.chunks, std::min(rows - r, kRowBlock));
        hipError_t e = launch_kernel(vecs == 1 ? sample_chunk_kernel<T, 1> : sample_chunk_kernel<T, 2>, grid, kThreads, st, a, p);
        if (e == hipSuccess)
            e = launch_kernel(vecs == 1 ? sample_row_kernel<T, 1> : sample_row_kernel<T, 2>, dim3(grid.y), kThreads, st, a, p);
        if (e != hipSuccess) return e;
        a.logits = (const T*)a.logits + (int64_t)kRowBlock * a.row_stride;
        a.uniform += kRowBlock;
        a.tokens += kRowBlock;
        if (a.temperature) a.temperature += kRowBlock;
        if (a.top_k) a.top_k += kRowBlock;
        if (a.top_p) a.top_p += kRowBlock;
        if (a.min_p) a.min_p += kRowBlock;
        if (a.logprob) a.logprob += kRowBlock;
    }
    return hipSuccess;
}

}  // namespace
}  // namespace lsamd

extern "C" uint64_t ls_hip_sample_workspace(const ls_hip_sample* a) {
    using namespace lsamd;
    if (!a || check(*a) || !a->rows) return 0;
    int vecs;
    const RowArgs p = plan_rows(*a, &vecs);
    return (uint64_t)std::min(a->rows, kRowBlock) * p.chunks * p.words * 8ull;
}

extern "C" int ls_hip_sample_enqueue(const ls_hip_sample* a, void* stream) {
    using namespace lsamd;
    if (!a) return EINVAL;
    if (const int rc = check(*a)) return rc;
    if (!a->rows) return 0;
    if (!a->workspace || a->workspace_bytes < ls_hip_sample_workspace(a)) return ENOSPC;
    const auto st = static_cast<hipStream_t>(stream);
    return static_cast<int>(a->dtype == LS_TYPE_F16    ? launch<_Float16>(*a, st)
                            : a->dtype == LS_TYPE_BF16 ? launch<__bf16>(*a, st)
                                                       : launch<float>(*a, st));
}
