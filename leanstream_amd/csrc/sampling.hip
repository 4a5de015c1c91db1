// One token a row from given random numbers: ls_hip_sample_enqueue.
//
// e_i = exp((l_i - top) / T), w_i = round(2^32 e_i). Ranked by (logit descending, id ascending) the kept
// tokens are a prefix: everything above a cut logit, and of the tokens equal to it the first few by id. The
// cut of top-k, and then that of top-p among the top k, are found by radix selection over the logits' 32-bit
// order: 8 bits a pass, with the count and the weight of every digit. Weights are whole numbers, so sums are
// exact and no order of atomics changes a result. Tokens of weight 0 can neither be drawn nor move a share,
// and are left out throughout.
#include <hip/hip_runtime.h>
#include <cerrno>
#include "leanstream_hip.h"

namespace lsamd {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr float kUnit = 4294967296.0f;   // weight of the best token
constexpr uint32_t kMaxVocab = 1u << 20; // sums stay below 2^52

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_float(__bf16 x) { return (float)x; }

// Order of the logits as unsigned numbers; -0 and +0 are equal, NaN is -inf.
__device__ __forceinline__ uint32_t order_of(float l) {
    if (!(l == l)) l = -INFINITY;
    const uint32_t u = __float_as_uint(l + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// floor (or ceil) of total * fraction, the fraction in steps of 2^-24 (total < 2^52)
__device__ __forceinline__ uint64_t share(uint64_t total, float fraction, bool up) {
    const uint64_t m = fraction > 0.0f ? (uint64_t)((double)fminf(fraction, 1.0f) * 16777216.0) : 0;
    return m * (total >> 24) + ((m * (total & 0xffffff) + (up ? 0xffffff : 0)) >> 24);
}

struct Row {
    float top, temperature;
    __device__ __forceinline__ float log_e(float l) const {
        return l == top ? 0.0f : (l - top) / temperature;   // equal: also where both are infinite
    }
    __device__ __forceinline__ float e(float l) const { return expf(log_e(l)); }
};
__device__ __forceinline__ uint64_t weight(float e) { return e == e ? (uint64_t)rintf(e * kUnit) : 0; }

// A prefix of the ranking: every order above `order`, and the first `ties` ids of those equal to it.
struct Cut {
    uint32_t order, ties;
};

struct Shared {
    uint64_t weights[256];
    uint32_t counts[256];
    uint64_t wave_weight[kWaves];
    uint32_t wave_count[kWaves];
    uint64_t before_weight;
    uint32_t before_count, digit;
};

// The shortest prefix within `limit` whose count reaches need_count or whose weight reaches need_weight; all
// of `limit` if none does. kept_weight: the weight of that prefix.
template <class T>
__device__ Cut select(const T* logits, uint32_t vocab, const Row& row, Cut limit, uint32_t need_count,
                      uint64_t need_weight, Shared& sh, uint64_t* kept_weight) {
    uint32_t prefix = 0, before_count = 0;
    uint64_t before_weight = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += kThreads) sh.weights[i] = 0, sh.counts[i] = 0;
        if (threadIdx.x == 0) sh.digit = 256;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < vocab; i += kThreads) {
            const float l = to_float(logits[i]);
            const uint32_t o = order_of(l);
            if (o < limit.order || (shift < 24 && (o >> shift >> 8) != (prefix >> shift >> 8))) continue;
            const uint64_t w = weight(row.e(l));
            if (!w) continue;
            atomicAdd(&sh.counts[o >> shift & 255], 1u);
            atomicAdd((unsigned long long*)&sh.weights[o >> shift & 255], (unsigned long long)w);
        }
        __syncthreads();
        // the first digit from above at which one of the sums is reached (at the last level a digit is one
        // logit, and of the limit's own logit only its ties count)
        if (threadIdx.x == 0) {
            uint32_t c = before_count;
            uint64_t s = before_weight;
            for (int d = 255; d >= 0; --d) {
                uint32_t n = sh.counts[d];
                uint64_t w = sh.weights[d];
                if (!n) continue;
                if (shift == 0 && (prefix | (uint32_t)d) == limit.order && n > limit.ties) w = w / n * limit.ties, n = limit.ties;
                if (c + n >= need_count || s + w >= need_weight) {
                    sh.digit = d;
                    break;
                }
                c += n;
                s += w;
            }
            sh.before_count = c;
            sh.before_weight = s;
        }
        __syncthreads();
        before_count = sh.before_count;
        before_weight = sh.before_weight;
        const uint32_t digit = sh.digit;
        if (digit == 256) {   // not reached: all of the limit
            __syncthreads();
            *kept_weight = before_weight;
            return limit;
        }
        prefix |= digit << shift;
        if (shift == 0) {
            uint32_t n = sh.counts[digit];
            const uint64_t one = sh.weights[digit] / n;
            if (prefix == limit.order) n = min(n, limit.ties);
            // ties needed for the count and for the weight, whichever is reached first
            uint64_t ties = min((uint64_t)n, (uint64_t)(need_count - before_count));
            ties = min(ties, (need_weight - before_weight - 1) / one + 1);
            __syncthreads();
            *kept_weight = before_weight + ties * one;
            return Cut{prefix, (uint32_t)ties};
        }
        __syncthreads();
    }
    return limit;
}

template <class T>
__global__ __launch_bounds__(kThreads) void sample_kernel(const ls_hip_sample a) {
    __shared__ Shared sh;
    __shared__ uint64_t best[kWaves];
    const uint32_t r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* logits = (const T*)a.logits + (int64_t)r * a.row_stride;

    // the best token: highest order, lowest id
    uint64_t mine = 0;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += kThreads)
        mine = max(mine, (uint64_t)order_of(to_float(logits[i])) << 32 | (0xffffffffu - i));
#pragma unroll
    for (int d = 32; d; d >>= 1) mine = max(mine, (uint64_t)__shfl_xor((unsigned long long)mine, d));
    if (lane == 0) best[wave] = mine;
    __syncthreads();
    for (int i = 0; i < kWaves; ++i) mine = max(mine, best[i]);
    const uint32_t best_id = 0xffffffffu - (uint32_t)mine;
    Row row{to_float(logits[best_id]), a.temperature ? a.temperature[r] : 1.0f};
    if (!(row.top > -INFINITY)) {
        if (threadIdx.x == 0) {
            a.tokens[r] = -1;
            if (a.logprob) a.logprob[r] = -INFINITY;
        }
        return;
    }
    if (!(row.temperature > 0.0f)) {
        if (threadIdx.x == 0) {
            a.tokens[r] = (int32_t)best_id;
            if (a.logprob) a.logprob[r] = 0.0f;
        }
        return;
    }

    const int32_t top_k = a.top_k ? a.top_k[r] : 0;
    const float top_p = a.top_p ? a.top_p[r] : 1.0f, min_p = a.min_p ? fminf(a.min_p[r], 1.0f) : 0.0f;
    Cut cut{0, 0xffffffffu};
    uint64_t total;
    cut = select(logits, a.vocab, row, cut, top_k > 0 ? (uint32_t)top_k : 0xffffffffu, ~0ull, sh, &total);
    if (top_p < 1.0f) {
        const uint64_t limit = share(total, top_p, true);
        cut = select(logits, a.vocab, row, cut, 0xffffffffu, limit ? limit : 1, sh, &total);
    }

    // Kept weight of each wave's stretch of the vocabulary: what lies above the cut, and its ties in order.
    const uint32_t stretch = ((a.vocab + kWaves - 1) / kWaves + 63) / 64 * 64;
    const uint32_t begin = min(wave * stretch, a.vocab), end = min(begin + stretch, a.vocab);
    uint64_t above = 0, tie_weight = 0;
    uint32_t ties = 0;
    for (uint32_t i = begin + lane; i < end; i += 64) {
        const float l = to_float(logits[i]);
        const uint32_t o = order_of(l);
        const float e = row.e(l);
        if (o < cut.order || !(e >= min_p)) continue;
        if (o == cut.order) ++ties, tie_weight = weight(e);
        else above += weight(e);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        above += __shfl_xor((unsigned long long)above, d);
        ties += __shfl_xor(ties, d);
        tie_weight = max(tie_weight, (uint64_t)__shfl_xor((unsigned long long)tie_weight, d));
    }
    if (lane == 0) sh.wave_count[wave] = ties;
    __syncthreads();
    uint32_t ties_left = cut.ties;
    for (uint32_t i = 0; i < wave; ++i) ties_left -= min(ties_left, sh.wave_count[i]);
    if (lane == 0) sh.wave_weight[wave] = above + min(ties, ties_left) * tie_weight;
    __syncthreads();
    uint64_t sum = 0, before = 0;
    for (uint32_t i = 0; i < kWaves; ++i) {
        if (i == wave) before = sum;
        sum += sh.wave_weight[i];
    }
    const uint64_t target = min(share(sum, a.uniform[r], false), sum - 1);
    if (target < before || target >= before + sh.wave_weight[wave]) return;
    // this wave's stretch holds the token
    uint64_t seen = before;
    for (uint32_t i0 = begin; i0 < end; i0 += 64) {
        const uint32_t i = i0 + lane;
        float e = 0.0f;
        bool keep = false, tie = false;
        if (i < end) {
            const float l = to_float(logits[i]);
            const uint32_t o = order_of(l);
            e = row.e(l);
            tie = o == cut.order && e >= min_p;
            keep = o > cut.order && e >= min_p;
        }
        const uint64_t tie_lanes = __ballot(tie);
        if (tie && (uint32_t)__popcll(tie_lanes & ((1ull << lane) - 1)) < ties_left) keep = true;
        ties_left -= min(ties_left, (uint32_t)__popcll(tie_lanes));
        const uint64_t w = keep ? weight(e) : 0;
        uint64_t upto = w;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t x = __shfl_up((unsigned long long)upto, d);
            if (lane >= (uint32_t)d) upto += x;
        }
        const uint64_t found = __ballot(seen + upto > target);
        if (found) {
            if (lane == (uint32_t)__ffsll((unsigned long long)found) - 1) {
                a.tokens[r] = (int32_t)i;
                // from the exponent itself: a small weight's rounding does not show in its logarithm
                if (a.logprob) a.logprob[r] = row.log_e(to_float(logits[i])) - logf((float)sum / kUnit);
            }
            return;
        }
        seen += __shfl((unsigned long long)upto, 63);
    }
}

bool aligned(const void* p, uintptr_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

int check(const ls_hip_sample& a) {
    if (!a.logits || !a.uniform || !a.tokens || !a.vocab || a.dtype > LS_TYPE_F32) return EINVAL;
    if (!aligned(a.logits, a.dtype == LS_TYPE_F32 ? 4 : 2) || a.row_stride < 0) return EINVAL;
    for (const void* p : {(const void*)a.uniform, (const void*)a.temperature, (const void*)a.top_k, (const void*)a.top_p,
                          (const void*)a.min_p, (const void*)a.tokens, (const void*)a.logprob})
        if (!aligned(p, 4)) return EINVAL;
    if (!aligned(a.workspace, 16)) return EINVAL;
    if (a.vocab > kMaxVocab || a.rows > 0x7fffffffu) return ENOTSUP;
    return 0;
}

}  // namespace
}  // namespace lsamd

extern "C" uint64_t ls_hip_sample_workspace(const ls_hip_sample*) { return 0; }

extern "C" int ls_hip_sample_enqueue(const ls_hip_sample* a, void* stream) {
    using namespace lsamd;
    if (!a) return EINVAL;
    if (const int rc = check(*a)) return rc;
    if (!a->rows) return 0;
    const auto st = static_cast<hipStream_t>(stream);
    if (a->dtype == LS_TYPE_F16) sample_kernel<_Float16><<<a->rows, kThreads, 0, st>>>(*a);
    else if (a->dtype == LS_TYPE_BF16) sample_kernel<__bf16><<<a->rows, kThreads, 0, st>>>(*a);
    else sample_kernel<float><<<a->rows, kThreads, 0, st>>>(*a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : static_cast<int>(e);
}
