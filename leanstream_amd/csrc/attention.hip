// Attention of new tokens over a paged cache: ls_hip_attention_enqueue.
//
// For a query row q and its visible keys: out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), s_j = scale
// q.k_j, in one pass over the keys with the running maximum m and sum (both fp32): when m rises, what was
// summed is scaled by e^(m_old - m_new). Exponentials are taken to base 2 with scale * log2(e) folded in.
//
// The query heads of one KV head share its keys, so the rows of a tile are (token, head of the group)
// pairs: row r of a sequence is token r / group, head r % group.
//
// P = e^(s - m) is rounded to the values' type, the only type that the matrix cores multiply with them: P in two parts
// would keep 32 bits at the price of a second product. It costs up to u |v| (u = 2^-11 in fp16, 2^-8 in bf16), as much as
// the output's own rounding: against 64 bits, relative, 2.9e-4 for 4096 tokens over 32768 keys in fp16 where fp32
// weights give 2.1e-4, and 2.2e-4 and 2.1e-4 for a single token. What is summed is the unrounded P.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cerrno>
#include <cfloat>
#include <cmath>
#include "kernel_launch.h"
#include "leanstream_hip.h"
#include "wave_ops.h"

// Closures over register arrays are inlined, or the arrays would lie in memory.
#define LS_INLINE __attribute__((always_inline))

namespace lsamd {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// A row's maximum before its first visible key: no finite score lies below it, and being finite itself it can be
// subtracted from a masked one (-inf).
constexpr float kNoKey = -FLT_MAX;

// Bit patterns of the two 16-bit types; arithmetic is in fp32 and in the matrix instructions.
struct F16 {
    typedef half8 vec8;
    static constexpr uint32_t kExponent = 0x7c00u;   // all ones: infinity or NaN
    static __device__ __forceinline__ float to_float(short x) { return (float)__builtin_bit_cast(_Float16, x); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        typedef _Float16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, v2{(_Float16)a, (_Float16)b});
    }
    // A mean of finite values is no larger than they are, but with weights that were rounded apart from their sum it may
    // be by 2^-11, which past the largest fp16 would make an infinity of it.
    static __device__ __forceinline__ float mean(float x) {
        return fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.0f), 65504.0f) : x;
    }
    static __device__ __forceinline__ f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0,
                                                      0, 0);
    }
    static __device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0,
                                                      0, 0);
    }
};
struct BF16 {
    typedef bhalf8 vec8;
    static constexpr uint32_t kExponent = 0x7f80u;
    static __device__ __forceinline__ float to_float(short x) { return (float)__builtin_bit_cast(__bf16, x); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        typedef __bf16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, v2{(__bf16)a, (__bf16)b});
    }
    static __device__ __forceinline__ float mean(float x) { return x; }   // its range is fp32's, and so is the sums'
    static __device__ __forceinline__ f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), c,
                                                       0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), c,
                                                       0, 0, 0);
    }
};

// Page tables and lengths do not change while a kernel runs: read through this view, uniform entries come over the
// scalar cache and do not queue behind vector loads.
#if defined(__HIP_DEVICE_COMPILE__)
typedef const __attribute__((address_space(4))) int32_t* Table;
#else
typedef const int32_t* Table;
#endif

struct Sequence {
    int first;    // its first row of q
    int tokens;   // new tokens
    int keys;
};

// A sequence's lengths, held against the block's bounds: what lies outside has no tokens (their place in
// q is unknown) or no keys. Ints: a pointer to int32_t or a Table.
template <class Ints>
__device__ __forceinline__ Sequence read_sequence(const ls_hip_attention& a, int s) {
    const int q0 = ((Ints)a.q_start)[s], q1 = ((Ints)a.q_start)[s + 1];
    Sequence q{q0, q1 - q0, ((Ints)a.context)[s]};
    bool bad = false;
    if (q0 < 0 || q1 < q0 || q1 > (int)a.tokens || (uint32_t)(q1 - q0) > a.max_new) {
        q.tokens = 0;
        bad = true;
    }
    if (q.keys < 0 || (uint32_t)q.keys > a.max_context) {
        q.keys = 0;
        bad = true;
    }
    if (bad && a.status) atomicOr(a.status, (uint32_t)LS_STATUS_RANGE);
    return q;
}

__device__ __forceinline__ bool sees(int key, int pos, int window, int sinks) {
    return key <= pos && (window == 0 || key > pos - window || key < sinks);
}

// Of the lanes i and i ^ 32 (i ^ 16): the larger value, the sum.
__device__ __forceinline__ float max32(float x) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}
__device__ __forceinline__ float max16(float x) {
    const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}
__device__ __forceinline__ float sum32(float x) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(both[0]) + __uint_as_float(both[1]);
}
__device__ __forceinline__ float sum16(float x) {
    const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(both[0]) + __uint_as_float(both[1]);
}

// Whether one of eight values is an infinity or NaN.
template <class T>
__device__ __forceinline__ bool not_finite(s16x8 v) {
    const u32x4 w = __builtin_bit_cast(u32x4, v);
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        odd |= (w[j] & T::kExponent) == T::kExponent || ((w[j] >> 16) & T::kExponent) == T::kExponent;
    return odd;
}

// Keys that some row between the positions p_low and p_high sees, in steps of `unit` keys: the sinks' steps,
// then those from the oldest key of a window on. Step t starts at key(t).
struct Steps {
    int unit, sink, first, count;
    int low;   // keys below it are seen as sinks only
    __device__ __forceinline__ Steps(int unit_, int p_low, int p_high, int window, int sinks) : unit(unit_) {
        low = window ? max(0, p_low + 1 - window) : 0;
        const int end = p_high < 0 ? 0 : p_high / unit + 1;
        sink = window ? min((sinks + unit - 1) / unit, end) : 0;
        first = max(low / unit, sink);
        count = end ? sink + max(0, end - first) : 0;
    }
    __device__ __forceinline__ int key(int t) const { return (t < sink ? t : first + t - sink) * unit; }
};

// ---------------------------------------------------------------------------------
// Few rows: one sequence's new tokens times the heads of a group
// ---------------------------------------------------------------------------------
// Bound by the bytes of the cache: 4.9 TB/s for 32 sequences of up to 8192 keys (64 / 8 heads of 128, 136 us), 5.5 for
// two of up to 131072 (145 us); a copy of 2 GiB reaches 4.9. 16-row products waste most of their rows on a single
// token, at 3 % of what the matrix cores could do. Keys go 32 at a time from memory straight into matrix operands, with
// no LDS: a lane of S^T = K Q^T (16 x 16 x 32) holds 16 bytes of one key, and of V a lane loads the same D / 16
// dimensions of the 8 keys whose P it multiplies, which byte permutes turn into operands. The four waves of a workgroup
// take the steps of its split in turn and are joined through LDS; the splits of a long sequence are joined by the
// workgroup that finishes last, in their order.
constexpr int kRowWaves = 4;
constexpr int kRows = 16;          // sequences of up to this many rows go this way
constexpr int kStepKeys = 32;
constexpr uint32_t kMaxSplits = 128;   // one workgroup joins them

struct SplitPlan {
    uint32_t splits;       // of the longest sequence
    uint32_t chunk;        // steps of a split, a multiple of kRowWaves
    uint32_t rows;         // of a split in the workspace
    uint64_t bytes;        // of the workspace
};

// The workspace begins with the splits' counters, at the same place for calls of every shape: they are 0
// between calls.
constexpr uint32_t kFill = 1024;   // workgroups that fill the card, 4 on each of 256 compute units
constexpr uint64_t kCounterBytes = kFill * sizeof(uint32_t);

__device__ __forceinline__ void store_agent(float* p, float a, float b) {
    __hip_atomic_store((uint64_t*)p, __builtin_bit_cast(uint64_t, f32x2{a, b}), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x2 load_agent(const float* p) {
    return __builtin_bit_cast(f32x2, __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// The 32 keys of a step: where they lie. Pages of 16 keys and more: both halves lie in one page each, their
// addresses are uniform and lanes add 32-bit offsets. Smaller ones: lane t holds the page of key t
// (one token over 777 keys 7.7 and 8.1 us, 2048 over 8192 308 and 312).
template <bool Large>
struct StepPages {
    int page[Large ? 2 : 1];
    bool ok;   // no page out of range among them
    __device__ __forceinline__ StepPages(const ls_hip_attention& a, Table table, int shift, int key0, int lane) {
        const int last = (int)a.table_width - 1;
        if constexpr (Large) {
            page[0] = table[min(key0 >> shift, last)];
            page[1] = table[min((key0 + 16) >> shift, last)];
            ok = (uint32_t)page[0] < a.pages && (uint32_t)page[1] < a.pages;
        } else {
            page[0] = table[min((key0 + (lane & 31)) >> shift, last)];
            ok = __all((uint32_t)page[0] < a.pages);
        }
    }
    // page of key0 + 16 half + row, row < 16; -1 if it is no page
    __device__ __forceinline__ int of(const ls_hip_attention& a, int half, int row) const {
        const int p = Large ? page[Large ? half : 0] : __shfl(page[0], 16 * half + row);
        return (uint32_t)p < a.pages ? p : -1;
    }
    // address of that key's row
    __device__ __forceinline__ const short* row(const ls_hip_attention& a, const void* base, int64_t page_stride,
                                                int64_t slot_stride, int shift, int key0, int half, int row) const {
        const int p = max(of(a, half, row), 0), mask = (1 << shift) - 1;
        if constexpr (Large)
            return (const short*)base + p * page_stride + ((key0 + 16 * half) & mask) * slot_stride +
                   (uint32_t)(row * (int)slot_stride);
        return (const short*)base + p * page_stride + ((key0 + 16 * half + row) & mask) * slot_stride;
    }
};

template <class T, int D, bool Large>
__global__ __launch_bounds__(64 * kRowWaves) void attention_rows_kernel(const ls_hip_attention a, uint32_t shift,
                                                                        const SplitPlan plan) {
    constexpr int kLaneDims = D / 16;
    typedef short lane_dims __attribute__((ext_vector_type(kLaneDims)));
    __shared__ __align__(16) float lds_o[kRowWaves][kRows][D + 4];
    __shared__ float lds_m[kRowWaves][kRows], lds_l[kRowWaves][kRows];
    __shared__ uint32_t lds_turn;

    const int head = blockIdx.x % a.kv_heads, split = blockIdx.x / a.kv_heads;
    const int group = a.q_heads / a.kv_heads;
    const Sequence seq = read_sequence<Table>(a, blockIdx.y);
    const int rows = seq.tokens * group;
    if (rows > kRows || rows == 0) return;
    const int base = seq.keys - seq.tokens;
    const int p_low = base, p_high = seq.keys - 1;
    const int window = (int)a.window, sinks = (int)a.sinks;
    const Steps steps(kStepKeys, p_low, p_high, window, sinks);
    const int splits = max(1, (steps.count + (int)plan.chunk - 1) / (int)plan.chunk);
    if (split >= splits) return;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i16 = lane & 15, g = lane >> 4;
    const int row = min(i16, rows - 1);
    const int pos = base + row / group;

    s16x8 q[D / 32];
    {
        const short* p = (const short*)a.q + (seq.first + row / group) * a.q_token_stride +
                         (head * group + row % group) * a.q_head_stride + 8 * g;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) q[i] = *(const s16x8*)(p + 32 * i);
    }
    f32x4 o[kLaneDims] = {};
    float m = kNoKey, l = 0.0f;
    const float scale = a.scale * kLog2e;
    const Table table = (Table)(a.page_table + blockIdx.y * a.table_stride);
    const short* k_head = (const short*)a.k_pages + head * a.k_head_stride + 8 * g;
    const short* v_head = (const short*)a.v_pages + head * a.v_head_stride + kLaneDims * i16;

    const int end = min((split + 1) * (int)plan.chunk, steps.count);
    int t = split * (int)plan.chunk + wave;
    s16x8 k[2][D / 32];
    auto load_k = [&](const StepPages<Large>& pages, int key0) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const short* p = pages.row(a, k_head, a.k_page_stride, a.k_slot_stride, shift, key0, half, i16);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) k[half][i] = *(const s16x8*)(p + 32 * i);
        }
    };
    if (t < end) {
        int key0 = steps.key(t);
        StepPages<Large> pages(a, table, shift, key0, lane);
        load_k(pages, key0);
        for (;;) {
            // key slot (g, j) of the second product: key 16 (j / 4) + 4 g + j % 4
            lane_dims v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v[j] = *(const lane_dims*)pages.row(a, v_head, a.v_page_stride, a.v_slot_stride, shift, key0, j / 4,
                                                    4 * g + j % 4);
            f32x4 s[2] = {};
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int i = 0; i < D / 32; ++i) s[half] = T::mfma16(k[half][i], q[i], s[half]);
            const int now0 = key0;
            const StepPages<Large> now = pages;
            const bool more = t + kRowWaves < end;
            t += kRowWaves;
            if (more) {
                key0 = steps.key(t);
                pages = StepPages<Large>(a, table, shift, key0, lane);
                load_k(pages, key0);
            }
            const bool full = now.ok && now0 + kStepKeys - 1 <= p_low &&
                              (window == 0 || now0 > p_high - window || now0 + kStepKeys <= sinks);
            float top = m;
            if (!full) {
                // Keys that this row does not see are masked; of keys that no row sees (or without a page) the
                // values count as 0, whatever their slots hold.
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int key = now0 + 16 * (j / 4) + 4 * g + j % 4;
                    const bool any = key <= p_high && (window == 0 || key >= steps.low || key < sinks);
                    const bool page = now.of(a, j / 4, 4 * g + j % 4) >= 0;
                    if (any && !page) {
                        s[j / 4][j % 4] = 0.0f;
                        if (a.status) atomicOr(a.status, (uint32_t)LS_STATUS_BAD_DESCRIPTOR);
                    }
                    if (!any || !page) v[j] = lane_dims{};
                    if (!sees(key, pos, window, sinks)) s[j / 4][j % 4] = -INFINITY;
                }
            }
            {   // rounded once: fused with the subtraction below, the best score's distance to itself would not be 0
#pragma clang fp contract(off)
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, s[j / 4][j % 4] *= scale);
            }
            top = max32(max16(top));
            const float keep = __builtin_amdgcn_exp2f(m - top);
            m = top;
            // P is rounded to the values' type; the sum takes it in fp32
            u32x4 p;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float x = __builtin_amdgcn_exp2f(s[j / 4][j % 4] - m);
                const float y = __builtin_amdgcn_exp2f(s[j / 4][j % 4 + 1] - m);
                sum += x + y;
                p[j / 2] = T::pack(x, y);
            }
            l = l * keep + sum;
            const s16x8 pp = __builtin_bit_cast(s16x8, p);
#pragma unroll
            for (int d = 0; d < kLaneDims; ++d) {
                // dimension kLaneDims i16 + d of the 8 keys
                s16x8 vt;
#pragma unroll
                for (int j = 0; j < 8; ++j) vt[j] = v[j][d];
                o[d] *= keep;
                if (!full && __ballot(not_finite<T>(vt))) {
                    // A value that is not finite counts as 0 in the product (0 * NaN is NaN); key by key it is then added
                    // where it is seen. What another row sees does not change the order of a row's sums.
                    s16x8 odd = {};
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (((uint32_t)vt[j] & T::kExponent) == T::kExponent) odd[j] = vt[j], vt[j] = 0;
                    o[d] = T::mfma16(vt, pp, o[d]);
                    for (int slot = 0; slot < 32; ++slot) {
                        s16x8 va = {}, pa = {};
                        if (g == slot / 8) {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if (j == slot % 8) va[j] = odd[j], pa[j] = pp[j];
                        }
                        const f32x4 one = T::mfma16(va, pa, f32x4{});
                        if (sees(now0 + 16 * (slot % 8 / 4) + 4 * (slot / 8) + slot % 4, pos, window, sinks))
                            o[d] += one;
                    }
                    continue;
                }
                o[d] = T::mfma16(vt, pp, o[d]);
            }
            if (!more) break;
        }
    }
    l = sum32(sum16(l));

    // the waves' sums, in their order
    if (g == 0) lds_m[wave][i16] = m, lds_l[wave][i16] = l;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int d = 0; d < kLaneDims; d += 4)
            *(f32x4*)&lds_o[wave][i16][(4 * g + r) * kLaneDims + d] = 
                f32x4{o[d][r], o[d + 1][r], o[d + 2][r], o[d + 3][r]};
    __syncthreads();

    // columns pairwise: thread -> (row, dims 2 c, 2 c + 1)
    const uint32_t pair = blockIdx.y * a.kv_heads + head;
    const uint32_t stride = plan.rows * (D + 2);   // floats of a split: rows of sums, then m and l of every row
    float* space = (float*)((char*)a.workspace + kCounterBytes) + (uint64_t)pair * plan.splits * stride;
    const int items = rows * (D / 2);
    auto put = [&](int r, int c, float x, float y, float top, float sum) {
        const int64_t token = seq.first + r / group, q_head = head * group + r % group;
        const float inv = sum > 0.0f ? 1.0f / sum : sum;   // NaN stays NaN
        *(uint32_t*)((short*)a.out + token * a.out_token_stride + q_head * a.out_head_stride + c) =
            T::pack(T::mean(x * inv), T::mean(y * inv));
        if (a.lse && c == 0) a.lse[token * a.q_heads + q_head] = sum == 0.0f ? -INFINITY : top * kLn2 + logf(sum);
    };
    for (int i = threadIdx.x; i < items; i += 64 * kRowWaves) {
        const int r = i / (D / 2), c = 2 * (i % (D / 2));
        float top = lds_m[0][r];
#pragma unroll
        for (int w = 1; w < kRowWaves; ++w) top = fmaxf(top, lds_m[w][r]);
        float x = 0.0f, y = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kRowWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(lds_m[w][r] - top);
            x += lds_o[w][r][c] * f;
            y += lds_o[w][r][c + 1] * f;
            sum += lds_l[w][r] * f;
        }
        if (splits > 1) {
            float* part = space + split * stride;
            store_agent(part + r * D + c, x, y);
            if (c == 0) store_agent(part + plan.rows * D + 2 * r, top, sum);
        } else {
            put(r, c, x, y, top, sum);
        }
    }
    if (splits == 1) return;

    // every store of the workgroup has been acknowledged before its turn is taken
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    uint32_t* counter = (uint32_t*)a.workspace + pair;
    if (threadIdx.x == 0) {
        lds_turn = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (lds_turn == (uint32_t)splits - 1)   // the last: ready for the next call
            __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (lds_turn != (uint32_t)splits - 1) return;
    // m and l of every split and row, then the columns pairwise, eight splits' loads at a time
    f32x2* ml = (f32x2*)&lds_o[0][0][0];
    static_assert(kMaxSplits * kRows * sizeof(f32x2) <= sizeof(lds_o), "room");
    for (int i = threadIdx.x; i < splits * rows; i += 64 * kRowWaves)
        ml[i] = load_agent(space + i / rows * stride + plan.rows * D + 2 * (i % rows));
    __syncthreads();
    for (int i = threadIdx.x; i < items; i += 64 * kRowWaves) {
        const int r = i / (D / 2), c = 2 * (i % (D / 2));
        float top = kNoKey, x = 0.0f, y = 0.0f, sum = 0.0f;
        for (int s = 0; s < splits; ++s) top = fmaxf(top, ml[s * rows + r][0]);
        for (int s0 = 0; s0 < splits; s0 += 8) {
            f32x2 part[8];
#pragma unroll
            for (int s = 0; s < 8; ++s) part[s] = load_agent(space + min(s0 + s, splits - 1) * stride + r * D + c);
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                if (s0 + s >= splits) break;
                const f32x2 its = ml[(s0 + s) * rows + r];
                const float f = __builtin_amdgcn_exp2f(its[0] - top);
                x += part[s][0] * f;
                y += part[s][1] * f;
                sum += its[1] * f;
            }
        }
        put(r, c, x, y, top, sum);
    }
}

// ---------------------------------------------------------------------------------
// Many rows
// ---------------------------------------------------------------------------------
// One workgroup: 8 (or 4) waves of 32 rows of one sequence and KV head against the keys that they see, 64 at a time
// through LDS. Products are taken transposed, S^T = K Q^T and O^T = V^T P^T (32 x 32 x 16), so that a lane holds scores
// of one row only and the P that it computed is already the second product's operand: key slots are permuted alike in P
// and V^T, which a sum over keys allows. V^T comes out of LDS by transposing reads.
//
// Bound by the matrix cores and the vector units, which are busy for 43 and 41 % of the time (16 products of 32 cycles
// and as long a stretch of exponentials, sums and roundings for 32 x 64 scores), at 2.0 to 2.1 GHz under this load: the
// scores of the next tile are multiplied while those of this one go through the softmax. Tiles come from memory without
// passing registers, two buffers each of K and V, one barrier a tile. 4096 tokens over 32768 keys, 32 / 8 heads of 128:
// 2.17 ms in fp16 (950 TFLOP/s; a product of 8192 x 8192 matrices reaches 1180), 2.06 ms in bf16 (1000 of
// 1240). 64 rows a wave halve the LDS reads, but their 512 registers leave one wave a SIMD: 3.3 ms.
//
// A prompt from its start (4096 tokens over as many keys, 16 heads of 64: 81 us, 425 TFLOP/s) has all its tiles under way
// at once, and those of early tokens see few keys: waves live for 60 % of the launch, the matrix cores are busy for 16 %
// and the vector units for 32 %. Heads of 256 (2048 tokens over 8192 keys, 16 heads: 484 us, 500 TFLOP/s) leave one
// wave a SIMD, so that nothing runs beside its waits: 20 % and 28 %.
//
// Where tiles are few, their keys are split; the parts go to the workspace in fp32 and are joined in order by
// attention_join_kernel (128 tokens over 32768 keys, 32 / 8 heads of 128: 1019 us whole, 97 in
// parts).
template <int D>
struct Tile {
    // D = 256 needs twice the registers a row; D = 64 has fewer products to a score, and two workgroups of 4 waves on a
    // compute unit overlap better than one of 8 (4096 tokens over 4096 keys, 16 heads: 81 and 102 us; D = 128, 4096
    // over 32768: 2.37 and 2.17 ms).
    static constexpr int kWaves = D == 128 ? 8 : 4;
    static constexpr uint32_t kFill = D == 64 ? 512 : 256;    // workgroups that run at once
    static constexpr int kRows = 32 * kWaves;
    static constexpr int kKeys = D == 256 ? 32 : 64;
    static constexpr int kChunks = D / 8;                     // 16-byte chunks of a row
    static constexpr int kLoads = kKeys * kChunks / (64 * kWaves);   // a wave's loads of a tile, 64 chunks each
    static constexpr int kLoadRows = 64 / kChunks;            // rows of one load
    // Chunk c of row r lies at position c ^ turn(r): the chunks that 16 lanes read of as many rows (K operands) and the
    // 64 bytes that 32 lanes read of each of 4 rows (transposing reads) lie in different banks, all 64 of them
    // (measured: no conflicts, 256 bytes a cycle). turn(r + 8) = turn(r) ^ 2 for r % 16 < 8.
    static __device__ __forceinline__ int turn(int r) {
        return D == 64 ? (r >> 1 & 1) << 2 | (r >> 2 & 3) : (r & 3) << 2 | (r >> 2 & 3);
    }
};
// A row's running maximum moves only where one of its scores (times scale log2(e)) exceeds it by more than this: until
// then P is at most 2^8 instead of 1, and the sums need no scaling.
constexpr float kSlack = 8.0f;
// A maximum below it is rounded by 2^-5 at most, which its weights and their sum share. That of one beyond it is not
// small beside 1, and scores have to be rounded alike before it is subtracted from them.
constexpr float kFar = 0x1p20f;

struct TilePlan {
    uint32_t splits;       // of a tile, at most
    // in the workspace: the steps of a split, then from kPartsAt on the parts, [split][token][q head]
    uint64_t offset;
                           // rows of D sums and then their m and l
    uint64_t bytes;
};
constexpr uint64_t kPartsAt = 256;
// Floats of a part: it begins at a multiple of 16 bytes, as it is stored in such words.
__host__ __device__ inline uint64_t part_floats(uint64_t rows, uint64_t dim) { return (rows * (dim + 2) + 3) / 4 * 4; }
constexpr uint32_t kLeastChunk = 8;    // steps: a split's part of the sums costs as much as one

// Steps of `unit` keys that rows of up to `span` neighbouring tokens of a sequence see, at most.
__host__ __device__ inline uint64_t most_steps(uint64_t keys, uint64_t unit, uint64_t span, uint64_t window,
                                               uint64_t sinks) {
    const uint64_t steps = (keys + unit - 1) / unit;
    const uint64_t some = (window + span + unit - 1) / unit + 1 + (sinks + unit - 1) / unit;
    return window && some < steps ? some : steps;
}

// The tiles of all sequences and their splits. Only the device knows the lengths, so every wave reads them, 64
// sequences at a time. `chunk`, the steps of a split, is the least that makes no more workgroups than run at once: a
// second round for a few of them costs more than it shortens the first, and so do parts of sums for tiles that fill the
// card by themselves (4096 tokens over 4096 keys, 16 heads of 64, 256 tiles: 103 us whole, 143 us split into 512).
template <int D>
struct TileWork {
    typedef Tile<D> C;
    uint32_t chunk;
    int seq, tile, split;   // of an item; seq -1: there is none
    __device__ __forceinline__ static uint32_t tiles_of(const ls_hip_attention& a, int s, uint32_t* steps) {
        const uint32_t group = a.q_heads / a.kv_heads;
        *steps = 0;
        if (s >= (int)a.sequences) return 0;
        const Sequence q = read_sequence<const int32_t*>(a, s);
        const uint32_t rows = q.tokens * group;
        if (rows <= (uint32_t)kRows) return 0;
        *steps = (uint32_t)most_steps(q.keys, C::kKeys, C::kRows / group + 2, a.window, a.sinks);
        return (rows + C::kRows - 1) / C::kRows;
    }
    __device__ __forceinline__ TileWork(const ls_hip_attention& a, const TilePlan& plan) {
        const int lane = threadIdx.x & 63;
        uint32_t total = 0, longest = 0, tiles = 0, n, steps;
        for (int s0 = 0; s0 < (int)a.sequences; s0 += 64) {
            n = tiles_of(a, s0 + lane, &steps);
            total += n * steps;
            tiles += n;
            longest = max(longest, steps);
        }
        tiles = wave_sum(tiles) * a.kv_heads;
        longest = wave_max(longest, 0u);
        chunk = max(longest, 1u);
        if (plan.splits == 1 || 2 * tiles > C::kFill) return;
        // Tiles times steps pass 32 bits only for contexts near 2^30, where the search below then begins lower.
        chunk = max((wave_sum(total) * a.kv_heads + C::kFill - 1) / C::kFill, kLeastChunk);
        chunk = max(chunk, (longest + plan.splits - 1) / plan.splits);
        for (;;) {   // twice the even share makes at most C::kFill / 2 + tiles
            uint32_t items = 0;
            for (int s0 = 0; s0 < (int)a.sequences; s0 += 64) {
                if (a.sequences > 64) n = tiles_of(a, s0 + lane, &steps);
                items += n * ((steps + chunk - 1) / chunk);
            }
            if (wave_sum(items) * a.kv_heads <= C::kFill || chunk >= longest) break;
            chunk += chunk / 8 + 1;
        }
    }
    __device__ __forceinline__ void find(const ls_hip_attention& a, uint32_t item) {
        const int lane = threadIdx.x & 63;
        uint32_t before = 0;
        seq = -1;
        for (int s0 = 0; s0 < (int)a.sequences && seq < 0; s0 += 64) {
            uint32_t steps;
            const uint32_t tiles = tiles_of(a, s0 + lane, &steps);
            const uint32_t splits = max(1u, (steps + chunk - 1) / chunk), items = tiles * splits;
            const uint32_t upto = wave_upto(items);
            const uint64_t at = __ballot(before + upto > item);
            if (at) {
                const int from = __ffsll((unsigned long long)at) - 1;
                const uint32_t i = item - before - from_lane(upto - items, from), its = from_lane(splits, from);
                seq = s0 + from;
                // the last tiles of a sequence see the most keys: they go first
                tile = from_lane(tiles, from) - 1 - i / its;
                split = i % its;
            }
            before += from_lane(upto, 63);
        }
    }
};

typedef __attribute__((address_space(3))) void* lds_void;
typedef __attribute__((address_space(3))) char* lds_bytes;
typedef const __attribute__((address_space(1))) void* global_void;

template <class T, int D, bool Large>
__global__ __launch_bounds__(64 * Tile<D>::kWaves, D == 64 ? 2 : 1) void attention_tile_kernel(
    const ls_hip_attention a, uint32_t shift, const TilePlan plan) {
    typedef Tile<D> C;
    constexpr int kKeys = C::kKeys, kSub = kKeys / 32;
    __shared__ __align__(1024) short lds_k[2][kKeys * D];
    __shared__ __align__(1024) short lds_v[2][kKeys * D];

    TileWork<D> work(a, plan);
    if (plan.splits > 1 && blockIdx.x == 0 && threadIdx.x == 0) 
        *(uint32_t*)((char*)a.workspace + plan.offset) = work.chunk;
    work.find(a, blockIdx.x / a.kv_heads);
    if (work.seq < 0) return;
    const int head = blockIdx.x % a.kv_heads, group = a.q_heads / a.kv_heads;
    const Sequence seq = read_sequence<Table>(a, work.seq);
    const int rows = seq.tokens * group, row0 = work.tile * C::kRows;
    const int row_end = min(row0 + C::kRows, rows);
    const int base = seq.keys - seq.tokens;   // position of token 0
    const int p_low = base + row0 / group, p_high = base + (row_end - 1) / group;
    const int window = (int)a.window, sinks = (int)a.sinks;
    const Steps steps(kKeys, p_low, p_high, window, sinks);
    const int begin = work.split * (int)work.chunk, end = min(begin + (int)work.chunk, steps.count);
    if (work.split && begin >= end) return;
    const bool whole = steps.count <= (int)work.chunk;   // no other split of this tile

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, h = lane >> 5;
    const int wave_row = row0 + 32 * wave;
    const bool active = wave_row < row_end;   // else the wave loads its part of the tiles and no more
    // positions of the wave's rows: what all of them see needs no masks
    const int wave_low = base + min(wave_row, row_end - 1) / group;
    const int wave_high = base + min(wave_row + 31, row_end - 1) / group;

    const int row = min(wave_row + col, row_end - 1), token = row / group, q_head = head * group + row % group;
    const int pos = base + token;
    s16x8 q[D / 16];
    {
        const short* p = (const short*)a.q + (seq.first + token) * a.q_token_stride + q_head * a.q_head_stride + 8 * h;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) q[i] = *(const s16x8*)(p + 16 * i);
    }
    const Table table = (Table)(a.page_table + work.seq * a.table_stride);
    const float scale = a.scale * kLog2e;

    // Loads of a tile: load i of a wave brings the rows kLoadRows (wave + kWaves i) + lane / kChunks. With pages of 16
    // keys and more, such a load lies in one page.
    const int load_row = lane / C::kChunks;
    const int last_page = (int)a.table_width - 1;
    struct Pages {
        int of[C::kLoads];
    };
    auto fetch = [&](int t) LS_INLINE {
        Pages pages;
        const int key0 = steps.key(t);
#pragma unroll
        for (int i = 0; i < C::kLoads; ++i) {
            const int r0 = C::kLoadRows * (wave + C::kWaves * i);
            pages.of[i] = table[min((key0 + r0 + (Large ? 0 : load_row)) >> (int)shift, last_page)];
        }
        return pages;
    };
    // A page that is none (or lies outside the cache): nobody's, or reported, and made zeros once it is here.
    auto load = [&](const void* pool, int64_t page_stride, int64_t head_stride, int64_t slot_stride, short* lds, int t,
                    const Pages& pages) LS_INLINE {
        uint32_t bad = 0;
        const int key0 = steps.key(t);
#pragma unroll
        for (int i = 0; i < C::kLoads; ++i) {
            const int r0 = C::kLoadRows * (wave + C::kWaves * i), r = r0 + load_row;
            int page = pages.of[i];
            if ((uint32_t)page >= a.pages) page = 0, bad |= 1u << i;
            const int slot = (key0 + (Large ? r0 : r)) & ((1 << shift) - 1);
            const short* src = (const short*)pool + page * page_stride + head * head_stride + slot * slot_stride;
            uint32_t at = 8 * ((lane % C::kChunks) ^ C::turn(r));
            if constexpr (Large) at += (uint32_t)(load_row * (int)slot_stride);
            __builtin_amdgcn_global_load_lds((global_void)(src + at), (lds_void)(lds + r0 * D), 16, 0, 0);
        }
        return bad;
    };
    auto some_row_sees = [&](int key) { return key <= p_high && (window == 0 || key >= steps.low || key < sinks); };
    auto clear = [&](uint32_t bad, short* lds, int key0) {
#pragma unroll
        for (int i = 0; i < C::kLoads; ++i) {
            if (!(bad >> i & 1)) continue;
            const int r = C::kLoadRows * (wave + C::kWaves * i) + load_row;
            *(s16x8*)(lds + r * D + 8 * (lane % C::kChunks)) = s16x8{};
            if (some_row_sees(key0 + r) && a.status) atomicOr(a.status, (uint32_t)LS_STATUS_BAD_DESCRIPTOR);
        }
    };
    auto load_k = [&](int t, const Pages& pages) LS_INLINE {
        return load(a.k_pages, a.k_page_stride, a.k_head_stride, a.k_slot_stride, lds_k[t & 1], t, pages);
    };
    auto load_v = [&](int t, const Pages& pages) LS_INLINE {
        return load(a.v_pages, a.v_page_stride, a.v_head_stride, a.v_slot_stride, lds_v[t & 1], t, pages);
    };
    // A lane's addresses in LDS. Rows are 2 D bytes, so the turned chunk index is a xor on the bits below them; what is
    // left of an address is a constant of the instruction.
    const uint32_t k_at = 2 * D * col + 16 * (h ^ C::turn(col));
    const int v_row = 4 * h + (lane & 15) / 4;
    const uint32_t v_at = 2 * D * v_row + 16 * ((2 * (lane >> 4 & 1) + (lane >> 1 & 1)) ^ C::turn(v_row)) +
        8 * (lane & 1);
    auto keys = [&](const lds_bytes lds, int i, s16x8 (&k)[kSub]) LS_INLINE {
        const lds_bytes at = lds + (k_at ^ (32 * i));
#pragma unroll
        for (int kt = 0; kt < kSub; ++kt) k[kt] = *(__attribute__((address_space(3))) s16x8*)(at + 2 * D * 32 * kt);
    };
    // Scores of a tile (register i of a lane is key 8 (i / 4) + 4 h + i % 4 of 32), work(i) going on beside step i: the
    // matrix cores take 32 cycles for a product that is issued in 4, and the operands of the next step are read
    // meanwhile. The barriers keep the compiler from reading everything at once, which does not fit the registers.
    auto scores = [&](f32x16 (&s)[kSub], int t, auto work) LS_INLINE {
        const lds_bytes lds = (lds_bytes)lds_k + (t & 1) * (2 * D * kKeys);
        s16x8 k[2][kSub];
#pragma unroll
        for (int kt = 0; kt < kSub; ++kt) s[kt] = f32x16{};
        keys(lds, 0, k[0]);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            if (i + 1 < D / 16) keys(lds, i + 1, k[(i + 1) & 1]);
#pragma unroll
            for (int kt = 0; kt < kSub; ++kt) s[kt] = T::mfma32(k[i & 1][kt], q[i], s[kt]);
            work(i);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // V^T operands: key slot (h, j) of step t16 is key 16 t16 + 8 (j / 4) + 4 h + j % 4
    auto values = [&](int t, int t16, int d) LS_INLINE {
        const lds_bytes lds = (lds_bytes)lds_v + (t & 1) * (2 * D * kKeys);
        typedef __attribute__((address_space(3))) s16x4* lds_ptr;
        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + (v_at ^ (64 * d)) + 2 * D * 16 * t16));
        const s16x4 v1 =
            __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(lds + (v_at ^ (64 * d) ^ 32) + 2 * D * (16 * t16 + 8)));
        return __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto sees_all = [&](int key0, int low, int high) {   // rows from position low to high see every key of a tile
        return key0 + kKeys - 1 <= low && (window == 0 || key0 > high - window || key0 + kKeys <= sinks);
    };
    auto largest = [&](const f32x16 (&s)[kSub]) {
        float top = kNoKey;   // scaled like the scores it does not exceed any of them
#pragma unroll
        for (int kt = 0; kt < kSub; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kt][i]);
        return top;
    };
    // An infinity or NaN in a value must reach only the rows that see its key, and 0 * NaN is NaN: where not every row
    // of the workgroup sees all keys of a tile, such values become 0. True if one of them belongs to a row that sees
    // it: it is then added to the result at the end.
    auto settle = [&](int t, int key0) {
        bool odd = false, seen = false;
        for (int i = lane; i < kKeys * D / 8; i += 64) odd |= not_finite<T>(*(const s16x8*)(lds_v[t & 1] + 8 * i));
        if (!__any(odd)) return false;   // every wave looks at the whole tile: all or none go on
        __syncthreads();
        for (int i = threadIdx.x; i < kKeys * D / 8; i += 64 * C::kWaves) {
            s16x8 v = *(const s16x8*)(lds_v[t & 1] + 8 * i);
            if (!not_finite<T>(v)) continue;
            seen |= some_row_sees(key0 + i / C::kChunks);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (((uint32_t)v[j] & T::kExponent) == T::kExponent) v[j] = 0;
            *(s16x8*)(lds_v[t & 1] + 8 * i) = v;
        }
        return __syncthreads_or(seen) != 0;
    };

    f32x16 o[D / 32] = {};
    float m = kNoKey, l = 0.0f;
    float offset = m, trigger = m;   // what is subtracted from scaled scores; a score above needs a look at m
    bool later = false;
    if (begin < end) {
        f32x16 s[kSub];
        Pages pages1 = fetch(begin), pages2 = fetch(begin + 1);   // of the tiles t + 1 and t + 2
        uint32_t bad_k = load_k(begin, pages1), bad_v = load_v(begin, pages1);
        __builtin_amdgcn_s_waitcnt(0);
        if (bad_k) clear(bad_k, lds_k[begin & 1], steps.key(begin));
        __syncthreads();
        bad_k = begin + 1 < end ? load_k(begin + 1, pages2) : 0;
        pages1 = pages2;
        pages2 = fetch(begin + 2);
        scores(s, begin, [](int) {});
        float top = largest(s);
        for (int t = begin; t < end; ++t) {
            const int key0 = steps.key(t);
            const bool full = sees_all(key0, wave_low, wave_high);
            // tile t of V and tile t + 1 of K are here, and every wave is done with the buffers before them
            __builtin_amdgcn_s_waitcnt(0);
            if (bad_v) clear(bad_v, lds_v[t & 1], key0);
            if (bad_k) clear(bad_k, lds_k[(t + 1) & 1], steps.key(t + 1));
            __syncthreads();
            bad_v = t + 1 < end ? load_v(t + 1, pages1) : 0;
            bad_k = t + 2 < end ? load_k(t + 2, pages2) : 0;
            pages1 = pages2;
            pages2 = fetch(t + 3);
            if (!sees_all(key0, p_low, p_high)) later |= settle(t, key0);
            if (!active) continue;

            if (!full) {
#pragma unroll
                for (int kt = 0; kt < kSub; ++kt)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!sees(key0 + 32 * kt + 8 * (i / 4) + 4 * h + i % 4, pos, window, sinks))
                            s[kt][i] = -INFINITY;
                top = largest(s);
            }
            top = max32(top) * scale;
            if (__any(top > trigger)) {
                // by a row's own scores: with the others' its roundings would hang on keys that it does not see
                const float next_m = top > m + kSlack ? top : m, keep = __builtin_amdgcn_exp2f(m - next_m);
                m = next_m;
                l *= keep;
#pragma unroll
                for (int d = 0; d < D / 32; ++d) o[d] *= keep;
                const bool far = fabsf(m) > kFar && m != kNoKey;
                offset = far ? 0.0f : m;
                trigger = far ? -INFINITY : m + kSlack;
                if (__any(far)) {
                    // rounded like the maximum before it is subtracted: fused into one step the distance could be
                    // anything
#pragma clang fp contract(off)
#pragma unroll
                    for (int kt = 0; kt < kSub; ++kt)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float scaled = s[kt][i] * scale;
                            s[kt][i] = far ? (scaled - m) / scale : s[kt][i];
                        }
                }
            }
            // The next tile's scores (after the last one: of what the buffer held before, unused), and this one's P
            // beside them: rounded to the values' type, summed in fp32.
            f32x16 next[kSub];
            u32x4 p[kKeys / 16];
            scores(next, t + 1, [&](int step) LS_INLINE {
                constexpr int kPairs = kKeys / 4, kSteps = D / 16;
#pragma unroll
                for (int pair = step * kPairs / kSteps; pair < (step + 1) * kPairs / kSteps; ++pair) {
                    const float x = __builtin_amdgcn_exp2f(fmaf(s[pair / 8][pair % 8 * 2], scale, -offset));
                    const float y = __builtin_amdgcn_exp2f(fmaf(s[pair / 8][pair % 8 * 2 + 1], scale, -offset));
                    l += x + y;
                    p[pair / 4][pair % 4] = T::pack(x, y);
                }
            });
            // the second product, and the next tile's largest scores beside it
            top = kNoKey;
            s16x8 v[2][D / 32];
#pragma unroll
            for (int d = 0; d < D / 32; ++d) v[0][d] = values(t, 0, d);
#pragma unroll
            for (int t16 = 0; t16 < kKeys / 16; ++t16) {
                if (t16 + 1 < kKeys / 16)
#pragma unroll
                    for (int d = 0; d < D / 32; ++d) v[(t16 + 1) & 1][d] = values(t, t16 + 1, d);
#pragma unroll
                for (int d = 0; d < D / 32; ++d)
                    o[d] = T::mfma32(v[t16 & 1][d], __builtin_bit_cast(s16x8, p[t16]), o[d]);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, next[t16 / 2][t16 % 2 * 8 + i]);
            }
#pragma unroll
            for (int kt = 0; kt < kSub; ++kt) s[kt] = next[kt];
        }
    }
    l = sum32(l);
    const int64_t at = (int64_t)(seq.first + token) * a.q_heads + q_head;
    const int64_t part_rows = (int64_t)a.tokens * a.q_heads;
    float* parts = (float*)((char*)a.workspace + plan.offset + kPartsAt) + work.split * part_floats(part_rows, D);
    if (wave_row + col < row_end) {
        if (whole) {
            const float inv = l > 0.0f ? 1.0f / l : l;   // NaN stays NaN
            short* out = (short*)a.out + (seq.first + token) * a.out_token_stride + q_head * a.out_head_stride + 4 * h;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *(u32x2*)(out + 32 * d + 2 * i) =
                        u32x2{T::pack(T::mean(o[d][i] * inv), T::mean(o[d][i + 1] * inv)),
                              T::pack(T::mean(o[d][i + 2] * inv), T::mean(o[d][i + 3] * inv))};
            if (a.lse && h == 0) a.lse[at] = l == 0.0f ? -INFINITY : m * kLn2 + logf(l);
        } else {
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *(f32x4*)(parts + at * D + 32 * d + 2 * i + 4 * h) =
                        f32x4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
            if (h == 0) *(f32x2*)(parts + part_rows * D + 2 * at) = f32x2{m, l};
        }
    }
    // The values that became 0: their sum takes the place of the result of every row that sees one, or is added to it
    // where values of other tiles already left it without a finite one.
    if (!later) return;
    __syncthreads();   // the results are stored
    for (int i = threadIdx.x; i < (row_end - row0) * D; i += 64 * C::kWaves) {
        const int r = row0 + i / D, c = i % D, its = r / group, its_head = head * group + r % group;
        float sum = 0.0f;
        for (int t = begin; t < end; ++t) {
            const int key0 = steps.key(t);
            if (sees_all(key0, p_low, p_high)) continue;
            for (int key = key0; key < key0 + kKeys; ++key) {
                if (!sees(key, base + its, window, sinks)) continue;
                const int page = table[min(key >> (int)shift, last_page)];
                if ((uint32_t)page >= a.pages) continue;
                const short v = ((const short*)a.v_pages)[page * a.v_page_stride + head * a.v_head_stride +
                                                         (key & ((1 << shift) - 1)) * a.v_slot_stride + c];
                if (((uint32_t)v & T::kExponent) == T::kExponent) sum += T::to_float(v);
            }
        }
        if (sum == 0.0f) continue;
        short* out = (short*)a.out + (seq.first + its) * a.out_token_stride + its_head * a.out_head_stride + c;
        float* part = parts + ((int64_t)(seq.first + its) * a.q_heads + its_head) * D + c;
        const float now = whole ? T::to_float(*out) : *part;
        if (!(fabsf(now) < INFINITY)) sum += now;
        if (whole) *out = (short)T::pack(sum, 0.0f);
        else *part = sum;
    }
}

// Joins the parts of split tiles in the order of the splits: a workgroup 16 heads of a token, a wave a row.
template <class T, int D>
__global__ __launch_bounds__(1024) void attention_join_kernel(const ls_hip_attention a, const TilePlan plan) {
    constexpr int kLane = D / 64;
    typedef float lane_sums __attribute__((ext_vector_type(kLane)));
    const int lane = threadIdx.x & 63, t = blockIdx.x, group = a.q_heads / a.kv_heads;
    // the sequence of token t: the last one that starts at or before it
    int s = 0;
    for (int s0 = 0; s0 < (int)a.sequences; s0 += 64) {
        const uint64_t before =
            __ballot(s0 + lane < (int)a.sequences && a.q_start[min(s0 + lane, (int)a.sequences - 1)] <= t);
        if (!before) break;
        s = s0 + 63 - __clzll((long long)before);
    }
    const Sequence seq = read_sequence<Table>(a, __builtin_amdgcn_readfirstlane(s));
    const int rows = seq.tokens * group, base = seq.keys - seq.tokens;
    if (rows <= kRows || t < seq.first || t >= seq.first + seq.tokens) return;
    const int chunk = *(const int*)((const char*)a.workspace + plan.offset);
    const int64_t part_rows = (int64_t)a.tokens * a.q_heads;
    const int q_head = 16 * blockIdx.y + (threadIdx.x >> 6);
    if (q_head < (int)a.q_heads) {
        const int row0 = ((t - seq.first) * group + q_head % group) / Tile<D>::kRows * Tile<D>::kRows;
        const int row_end = min(row0 + Tile<D>::kRows, rows);
        const Steps steps(Tile<D>::kKeys, base + row0 / group, base + (row_end - 1) / group, (int)a.window,
                          (int)a.sinks);
        if (steps.count <= chunk) return;   // one split: the result is written
        const int64_t at = (int64_t)t * a.q_heads + q_head;
        const float* parts = (const float*)((const char*)a.workspace + plan.offset + kPartsAt);
        lane_sums o = {};
        float m = kNoKey, l = 0.0f;
#pragma unroll 8
        for (int begin = 0; begin < steps.count; begin += chunk, parts += part_floats(part_rows, D)) {
            const f32x2 ml = *(const f32x2*)(parts + part_rows * D + 2 * at);
            const lane_sums x = *(const lane_sums*)(parts + at * D + kLane * lane);
            const float next = fmaxf(m, ml[0]), old = __builtin_amdgcn_exp2f(m - next);
            const float f = __builtin_amdgcn_exp2f(ml[0] - next);
            o = o * old + x * f;
            l = l * old + ml[1] * f;
            m = next;
        }
        const float inv = l > 0.0f ? 1.0f / l : l;   // NaN stays NaN
        short* out = (short*)a.out + (int64_t)t * a.out_token_stride + q_head * a.out_head_stride + kLane * lane;
#pragma unroll
        for (int i = 0; i < kLane; ++i) out[i] = (short)T::pack(T::mean(o[i] * inv), 0.0f);
        if (a.lse && lane == 0) a.lse[at] = l == 0.0f ? -INFINITY : m * kLn2 + logf(l);
    }
}

bool aligned(const void* p, uintptr_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

int check(const ls_hip_attention& a) {
    // the pointers of empty tensors may be NULL
    if (a.tokens && (!a.q || !a.out || !a.k_pages || !a.v_pages || !a.page_table || !a.q_start || !a.context ||
                     !a.sequences || !a.pages || !a.table_width))
        return EINVAL;
    if (!a.q_heads || !a.kv_heads || a.q_heads % a.kv_heads) return EINVAL;
    if (!a.page_size || (a.page_size & (a.page_size - 1)) || a.dtype > LS_TYPE_F32) return EINVAL;
    if (a.tokens > 0x7fffffffu || a.pages > 0x7fffffffu || a.window > 0x3fffffffu || a.sinks > 0x3fffffffu ||
        a.max_context > 0x3fffffffu || (uint64_t)a.table_width * a.page_size < a.max_context || a.max_new > a.tokens)
        return EINVAL;
    if (a.table_stride < 0 || (a.sequences > 1 && a.table_stride < (int64_t)a.table_width) ||
        !(a.scale > 0.0f && a.scale < INFINITY))
        return EINVAL;
    for (const void* p : {(const void*)a.page_table, (const void*)a.q_start, (const void*)a.context, (const void*)a.lse,
                          (const void*)a.status})
        if (!aligned(p, 4)) return EINVAL;
    if (!aligned(a.q, 16) || !aligned(a.out, 16) || !aligned(a.k_pages, 16) || !aligned(a.v_pages, 16) ||
        !aligned(a.workspace, 16))
        return EINVAL;
    const int64_t strides[] = {a.q_token_stride, a.q_head_stride, a.out_token_stride, a.out_head_stride,
                               a.k_page_stride,
                               a.k_head_stride, a.k_slot_stride, a.v_page_stride, a.v_head_stride, a.v_slot_stride};
    for (int64_t s : strides)
        if (s < 0 || s % 8) return EINVAL;
    // a page's slots are reached with 32-bit offsets
    if ((uint64_t)a.k_slot_stride * a.page_size > 0x3fffffffu || (uint64_t)a.v_slot_stride * a.page_size > 0x3fffffffu)
        return ENOTSUP;
    if (a.dtype == LS_TYPE_F32 || (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256)) return ENOTSUP;
    if ((uint64_t)a.tokens * a.q_heads > 0x3fffffffu || a.sequences > 65535) return ENOTSUP;
    return 0;
}

// Splits of the sequences that take the row kernel. Long ones make kFill workgroups (131072 keys, 16 groups: 144 us;
// with half or twice as many 150 and 154). Splits of few steps pay only up to a workgroup a compute unit (32 sequences
// of 500 keys, 256 groups: whole 15 us, in four 20), and one workgroup joins them all: with s steps, about sqrt(2 s)
// splits cost least (8000 keys of 8 KV heads: 21 splits 13 us, 63 splits 18). That is set by the join, not by the card:
// with few KV heads most of it stays idle (131072 keys of one sequence: one KV head, 94 splits, 40 us, 1.7 TB/s; two
// 42 us, 3.2; eight 105 us, 5.1). A split has a step for each of its waves.
SplitPlan plan_rows(const ls_hip_attention& a) {
    SplitPlan p{};
    p.rows = (uint32_t)std::min<uint64_t>((uint64_t)a.max_new * (a.q_heads / a.kv_heads), kRows);
    const uint64_t steps = most_steps(a.max_context, kStepKeys, kRows, a.window, a.sinks);
    const uint64_t groups = (uint64_t)a.sequences * a.kv_heads;
    const auto even = [&](uint64_t workgroups) { return (steps * groups + workgroups - 1) / workgroups; };
    uint64_t chunk = std::max(even(kFill), (steps + kMaxSplits - 1) / kMaxSplits);
    chunk = std::max(chunk, std::min<uint64_t>(even(kFill / 4), 16));
    chunk = std::max((chunk + kRowWaves - 1) / kRowWaves, (uint64_t)(std::sqrt((double)steps / 2) / kRowWaves + 0.5));
    p.chunk = (uint32_t)std::min<uint64_t>(std::max<uint64_t>(chunk, 1) * kRowWaves, 1u << 30);
    p.splits = (uint32_t)std::max<uint64_t>(1, (steps + p.chunk - 1) / p.chunk);
    if (p.splits > 1) p.bytes = kCounterBytes + groups * p.splits * p.rows * (a.head_dim + 2) * sizeof(float);
    return p;
}

// Room for the splits of the tiles, as if all tokens belonged to few chunks.
template <int D>
TilePlan plan_tiles(const ls_hip_attention& a, uint64_t offset) {
    typedef Tile<D> C;
    TilePlan p{};
    const uint64_t group = a.q_heads / a.kv_heads;
    // workgroups without splits
    const uint64_t least = std::max<uint64_t>(1, a.tokens * group / C::kRows) * a.kv_heads;
    const uint64_t steps = most_steps(a.max_context, C::kKeys, C::kRows / group + 2, a.window, a.sinks);
    p.splits = (uint32_t)std::max<uint64_t>(1, std::min(C::kFill / least, (steps + kLeastChunk - 1) / kLeastChunk));
    p.offset = (std::max(offset, kCounterBytes) + 255) / 256 * 256;   // a call of few rows may use the counters next
    const uint64_t part = part_floats((uint64_t)a.tokens * a.q_heads, a.head_dim) * sizeof(float);
    if (p.splits > 1) p.bytes = p.offset + kPartsAt + p.splits * part;
    return p;
}
// Workgroups of the tiles: every tile ends with a split that is not full.
template <int D>
uint32_t tile_grid(const ls_hip_attention& a) {
    const uint64_t rows = (uint64_t)a.tokens * (a.q_heads / a.kv_heads);
    const uint64_t tiles = rows / Tile<D>::kRows + std::min<uint64_t>(a.sequences, rows / (kRows + 1));
    return (uint32_t)((tiles + Tile<D>::kFill / a.kv_heads + 1) * a.kv_heads);
}

struct Plan {
    bool by_rows, by_tiles;
    SplitPlan rows;
    TilePlan tiles;
    uint64_t bytes;
};
Plan make_plan(const ls_hip_attention& a) {
    Plan p{};
    const uint32_t group = a.q_heads / a.kv_heads;
    p.by_rows = group <= (uint32_t)kRows;
    p.by_tiles = (uint64_t)a.max_new * group > (uint64_t)kRows;
    if (p.by_rows) p.rows = plan_rows(a);
    if (p.by_tiles)
        p.tiles = a.head_dim == 64    ? plan_tiles<64>(a, p.rows.bytes)
                  : a.head_dim == 128 ? plan_tiles<128>(a, p.rows.bytes)
                                      : plan_tiles<256>(a, p.rows.bytes);
    p.bytes = std::max(p.rows.bytes, p.tiles.bytes);
    return p;
}

template <class T, int D>
hipError_t launch(const ls_hip_attention& a, const Plan& plan, hipStream_t stream) {
    const uint32_t shift = __builtin_ctz(a.page_size);
    const bool large = a.page_size >= 16;
    hipError_t e = hipSuccess;
    if (plan.by_rows)
        e = launch_kernel(large ? attention_rows_kernel<T, D, true> : attention_rows_kernel<T, D, false>,
                          dim3(plan.rows.splits * a.kv_heads, a.sequences), 64 * kRowWaves, stream, a, shift, plan.rows);
    if (plan.by_tiles && e == hipSuccess)
        e = launch_kernel(large ? attention_tile_kernel<T, D, true> : attention_tile_kernel<T, D, false>,
                          dim3(tile_grid<D>(a)), 64 * Tile<D>::kWaves, stream, a, shift, plan.tiles);
    if (plan.by_tiles && plan.tiles.splits > 1 && e == hipSuccess)
        e = launch_kernel(attention_join_kernel<T, D>, dim3(a.tokens, (a.q_heads + 15) / 16), 1024, stream, a, plan.tiles);
    return e;
}

template <class T>
hipError_t launch(const ls_hip_attention& a, const Plan& plan, hipStream_t stream) {
    return a.head_dim == 64    ? launch<T, 64>(a, plan, stream)
           : a.head_dim == 128 ? launch<T, 128>(a, plan, stream)
                               : launch<T, 256>(a, plan, stream);
}

}  // namespace
}  // namespace lsamd

extern "C" uint64_t ls_hip_attention_workspace(const ls_hip_attention* a) {
    using namespace lsamd;
    if (!a || check(*a) || !a->tokens || !a->max_new) return 0;
    return make_plan(*a).bytes;
}

extern "C" int ls_hip_attention_enqueue(const ls_hip_attention* a, void* stream) {
    using namespace lsamd;
    if (!a) return EINVAL;
    if (const int rc = check(*a)) return rc;
    if (!a->tokens || !a->max_new) return 0;
    const Plan plan = make_plan(*a);
    if (plan.bytes && (!a->workspace || a->workspace_bytes < plan.bytes)) return ENOSPC;
    const auto st = static_cast<hipStream_t>(stream);
    return static_cast<int>(a->dtype == LS_TYPE_F16 ? launch<F16>(*a, plan, st) : launch<BF16>(*a, plan, st));
}
