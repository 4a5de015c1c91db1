// Attention of new tokens over a paged cache: ls_hip_attention_enqueue.
//
// For a query row q and its visible keys: out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), s_j = scale
// q.k_j, in one pass over the keys with the running maximum m and sum (both fp32): when m rises, what was
// summed is scaled by e^(m_old - m_new). Exponentials are taken to base 2 with scale * log2(e) folded in.
//
// The query heads of one KV head share its keys, so the rows of a tile are (token, head of the group)
// pairs: row r of a sequence is token r / group, head r % group.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cerrno>
#include <cmath>
#include "leanstream_hip.h"

namespace lsamd {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Below every score that can occur and finite: a row's maximum before its first visible key.
constexpr float kNoKey = -1e30f;

// Bit patterns of the two 16-bit types; arithmetic is in fp32 and in the matrix instructions.
struct F16 {
    typedef half8 vec8;
    static constexpr uint32_t kExponent = 0x7c00u;   // all ones: infinity or NaN
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        typedef _Float16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, v2{(_Float16)a, (_Float16)b});
    }
    static __device__ __forceinline__ f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    }
};
struct BF16 {
    typedef bhalf8 vec8;
    static constexpr uint32_t kExponent = 0x7f80u;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        typedef __bf16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, v2{(__bf16)a, (__bf16)b});
    }
    static __device__ __forceinline__ f32x16 mfma32(s16x8 a, s16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bhalf8, a), __builtin_bit_cast(bhalf8, b), c, 0, 0, 0);
    }
};

struct Sequence {
    int first;    // its first row of q
    int tokens;   // new tokens
    int keys;
};

// A sequence's lengths, held against the block's bounds: what lies outside has no tokens (their place in
// q is unknown) or no keys.
__device__ __forceinline__ Sequence read_sequence(const ls_hip_attention& a, int s) {
    const int q0 = a.q_start[s], q1 = a.q_start[s + 1];
    Sequence q{q0, q1 - q0, a.context[s]};
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
// Few rows: one sequence's new tokens times the heads of a group, 16 rows a workgroup
// ---------------------------------------------------------------------------------
// Bound by the bytes of the cache. Keys go 32 at a time from memory straight into matrix operands, with no
// LDS: a lane of S^T = K Q^T (16 x 16 x 32) holds 16 bytes of one key, and of V a lane loads the same D / 16
// dimensions of the 8 keys whose P it multiplies, which byte permutes turn into operands. The four waves of a
// workgroup take the steps of its split in turn and are joined through LDS; the splits of a long sequence are
// joined by the workgroup that finishes last, in their order.
constexpr int kRowWaves = 4;
constexpr int kRows = 16;
constexpr int kStepKeys = 32;
constexpr int kShortRows = 64;     // sequences of up to this many rows go this way

struct SplitPlan {
    uint32_t splits;       // of the longest sequence
    uint32_t chunk;        // steps of a split, a multiple of kRowWaves
    uint32_t row_blocks;
    uint32_t rows;         // of a row block in the workspace
    uint64_t bytes;        // of the workspace
};

// The workspace begins with the splits' counters, at the same place for calls of every shape: they are 0
// between calls.
constexpr uint32_t kFill = 1024;   // workgroups that fill the card, 4 on each of 256 compute units
constexpr uint64_t kCounterBytes = kFill * sizeof(uint32_t);

__device__ __forceinline__ void store_agent(float* p, float a, float b) {
    typedef float v2 __attribute__((ext_vector_type(2)));
    __hip_atomic_store((uint64_t*)p, __builtin_bit_cast(uint64_t, v2{a, b}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float load_agent(const float* p) {
    return __uint_as_float(__hip_atomic_load((const uint32_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// The 32 keys of a step: where they lie. Pages of 16 keys and more: both halves lie in one page each, their
// addresses are uniform and lanes add 32-bit offsets. Smaller ones: lane t holds the page of key t.
template <bool Large>
struct StepPages {
    int page[Large ? 2 : 1];
    bool ok;   // no page out of range among them
    __device__ __forceinline__ StepPages(const ls_hip_attention& a, const int32_t* table, int shift, int key0, int lane) {
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
    const Sequence seq = read_sequence(a, blockIdx.y);
    const int rows = seq.tokens * group, row0 = blockIdx.z * kRows;
    if (rows > kShortRows || row0 >= rows) return;
    const int row_count = min(kRows, rows - row0);
    const int base = seq.keys - seq.tokens;
    const int p_low = base + row0 / group, p_high = base + (row0 + row_count - 1) / group;
    const int window = (int)a.window, sinks = (int)a.sinks;
    const Steps steps(kStepKeys, p_low, p_high, window, sinks);
    const int splits = max(1, (steps.count + (int)plan.chunk - 1) / (int)plan.chunk);
    if (split >= splits) return;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i16 = lane & 15, g = lane >> 4;
    const int row = row0 + min(i16, row_count - 1);
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
    const int32_t* table = a.page_table + blockIdx.y * a.table_stride;
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
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, s[j / 4][j % 4] *= scale);
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float keep = __builtin_amdgcn_exp2f(m - top);
            m = top;
            // P is rounded to the values' type for the matrix product; the sum takes it in fp32
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
                    // as in attention_tile_kernel: key by key, each added where it is seen
                    for (int slot = 0; slot < 32; ++slot) {
                        s16x8 va = {}, pa = {};
                        if (g == slot / 8) {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if (j == slot % 8) va[j] = vt[j], pa[j] = pp[j];
                        }
                        const f32x4 one = T::mfma16(va, pa, f32x4{});
                        if (sees(now0 + 16 * (slot % 8 / 4) + 4 * (slot / 8) + slot % 4, pos, window, sinks)) o[d] += one;
                    }
                    continue;
                }
                o[d] = T::mfma16(vt, pp, o[d]);
            }
            if (!more) break;
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // the waves' sums, in their order
    if (g == 0) lds_m[wave][i16] = m, lds_l[wave][i16] = l;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int d = 0; d < kLaneDims; d += 4)
            *(f32x4*)&lds_o[wave][i16][(4 * g + r) * kLaneDims + d] = f32x4{o[d][r], o[d + 1][r], o[d + 2][r], o[d + 3][r]};
    __syncthreads();

    // columns pairwise: thread -> (row, dims 2 c, 2 c + 1)
    const uint32_t pair = (blockIdx.y * a.kv_heads + head) * plan.row_blocks + blockIdx.z;
    const uint32_t stride = plan.rows * (D + 2);   // floats of a split: rows of sums, then m and l of every row
    float* space = (float*)((char*)a.workspace + kCounterBytes) + (uint64_t)pair * plan.splits * stride;
    const int items = row_count * (D / 2);
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
            const int token = seq.first + (row0 + r) / group, q_head = head * group + (row0 + r) % group;
            const float inv = sum > 0.0f ? 1.0f / sum : sum;   // NaN stays NaN
            *(uint32_t*)((short*)a.out + token * a.out_token_stride + q_head * a.out_head_stride + c) = T::pack(x * inv, y * inv);
            if (a.lse && c == 0)
                a.lse[(int64_t)token * a.q_heads + q_head] = sum == 0.0f ? -INFINITY : top * kLn2 + logf(sum);
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
    for (int i = threadIdx.x; i < row_count * D; i += 64 * kRowWaves) {
        const int r = i / D, c = i % D;
        float top = kNoKey, x = 0.0f, sum = 0.0f;
        for (int s = 0; s < splits; ++s) {
            const float* part = space + s * stride;
            const float ms = load_agent(part + plan.rows * D + 2 * r);
            const float next = fmaxf(top, ms);
            const float old = __builtin_amdgcn_exp2f(top - next), f = __builtin_amdgcn_exp2f(ms - next);
            x = x * old + load_agent(part + r * D + c) * f;
            sum = sum * old + load_agent(part + plan.rows * D + 2 * r + 1) * f;
            top = next;
        }
        const int token = seq.first + (row0 + r) / group, q_head = head * group + (row0 + r) % group;
        const float inv = sum > 0.0f ? 1.0f / sum : sum;
        ((short*)a.out)[token * a.out_token_stride + q_head * a.out_head_stride + c] = (short)T::pack(x * inv, 0.0f);
        if (a.lse && c == 0)
            a.lse[(int64_t)token * a.q_heads + q_head] = sum == 0.0f ? -INFINITY : top * kLn2 + logf(sum);
    }
}

// ---------------------------------------------------------------------------------
// Many rows
// ---------------------------------------------------------------------------------
constexpr int kTileWaves = 4;
constexpr int kTileRows = 32 * kTileWaves;
constexpr int kTileKeys = 64;

// One workgroup: 128 rows of one sequence and KV head against all keys they see, 64 at a time through LDS.
// A wave owns 32 rows. Products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that a lane holds
// scores of one row only and the P that it computed is already the second product's operand: key slots are
// permuted alike in P and V^T, which a sum over keys allows.
template <class T, int D>
__global__ __launch_bounds__(64 * kTileWaves) void attention_tile_kernel(const ls_hip_attention a, uint32_t page_shift) {
    constexpr int kStride = D + 8;   // halves of an LDS row; 16 bytes of padding turn the banks
    __shared__ __align__(16) short lds_k[kTileKeys * kStride];
    __shared__ __align__(16) short lds_v[kTileKeys * kStride];

    const int head = blockIdx.x % a.kv_heads;
    const int group = a.q_heads / a.kv_heads;
    const int tile = blockIdx.x / a.kv_heads;
    const Sequence seq = read_sequence(a, blockIdx.y);
    const int rows = seq.tokens * group;
    const int row0 = tile * kTileRows;
    if (rows <= kShortRows || row0 >= rows) return;
    const int row_end = min(row0 + kTileRows, rows);
    const int base = seq.keys - seq.tokens;   // position of token 0
    const int p_low = base + row0 / group, p_high = base + (row_end - 1) / group;
    const int window = (int)a.window, sinks = (int)a.sinks;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 31, h = lane >> 5;
    const int row = min(row0 + 32 * wave + col, row_end - 1);
    const bool store = row0 + 32 * wave + col < row_end;
    const int token = row / group, q_head = head * group + row % group;
    const int pos = base + token;

    s16x8 q[D / 16];
    {
        const short* p = (const short*)a.q + (seq.first + token) * a.q_token_stride + q_head * a.q_head_stride + 8 * h;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) q[i] = *(const s16x8*)(p + 16 * i);
    }
    f32x16 o[D / 32] = {};
    float m = kNoKey, l = 0.0f;
    const float scale = a.scale * kLog2e;

    const Steps steps(kTileKeys, p_low, p_high, window, sinks);
    const int low = steps.low;

    for (int t = 0; t < steps.count; ++t) {
        const int key0 = steps.key(t);
        __syncthreads();   // every wave is done with the previous tile
        for (int i = threadIdx.x; i < kTileKeys * (D / 8); i += 64 * kTileWaves) {
            const int r = i / (D / 8), c = i % (D / 8), key = key0 + r;
            s16x8 k = {}, v = {};
            if (key <= p_high && (window == 0 || key >= low || key < sinks)) {
                const int page = a.page_table[blockIdx.y * a.table_stride + (key >> page_shift)];
                const int slot = key & ((1 << page_shift) - 1);
                if ((uint32_t)page < a.pages) {
                    k = *(const s16x8*)((const short*)a.k_pages + page * a.k_page_stride + head * a.k_head_stride +
                                        slot * a.k_slot_stride + 8 * c);
                    v = *(const s16x8*)((const short*)a.v_pages + page * a.v_page_stride + head * a.v_head_stride +
                                        slot * a.v_slot_stride + 8 * c);
                } else if (a.status) {
                    atomicOr(a.status, (uint32_t)LS_STATUS_BAD_DESCRIPTOR);
                }
            }
            *(s16x8*)(lds_k + r * kStride + 8 * c) = k;
            *(s16x8*)(lds_v + r * kStride + 8 * c) = v;
        }
        __syncthreads();
        const bool full = key0 + kTileKeys - 1 <= p_low &&
                          (window == 0 || key0 > p_high - window || key0 + kTileKeys <= sinks);

        // scores of 2 x 32 keys: register i of a lane is key 8 (i / 4) + 4 h + i % 4 of its 32
        f32x16 s[2] = {};
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
                s[kt] = T::mfma32(*(const s16x8*)(lds_k + (32 * kt + col) * kStride + 16 * i + 8 * h), q[i], s[kt]);
        float top = m;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float x = s[kt][i] * scale;
                if (!full && !sees(key0 + 32 * kt + 8 * (i / 4) + 4 * h + i % 4, pos, window, sinks)) x = -INFINITY;
                s[kt][i] = x;
                top = fmaxf(top, x);
            }
        top = fmaxf(top, __shfl_xor(top, 32));
        const float keep = __builtin_amdgcn_exp2f(m - top);
        m = top;
        float sum = 0.0f;
        // P is rounded to the values' type for the matrix product; the sum takes it in fp32
        u32x4 p[4];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float x = __builtin_amdgcn_exp2f(s[kt][i] - m), y = __builtin_amdgcn_exp2f(s[kt][i + 1] - m);
                sum += x + y;
                p[2 * kt + i / 8][i % 8 / 2] = T::pack(x, y);
            }
        l = l * keep + sum;
#pragma unroll
        for (int d = 0; d < D / 32; ++d) o[d] *= keep;

        // key slot (h, j) of product step t: key 16 t + 8 (j / 4) + 4 h + j % 4
        const int tr_row = 4 * h + (lane & 15) / 4, tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
        for (int t16 = 0; t16 < 4; ++t16)
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
                const short* at = lds_v + (16 * t16 + tr_row) * kStride + 32 * d + tr_col;
                typedef __attribute__((address_space(3))) s16x4* lds_ptr;
                const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at));
                const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at + 8 * kStride));
                const s16x8 v = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
                if (!full) {
                    // An infinity or NaN in a value must reach only the rows that see its key, and 0 * NaN is
                    // NaN: such (rare) fragments are taken key by key, each added where it is seen.
                    if (__ballot(not_finite<T>(v))) {
                        const s16x8 pp = __builtin_bit_cast(s16x8, p[t16]);
                        for (int slot = 0; slot < 16; ++slot) {
                            s16x8 va = {}, pa = {};
                            if (h == slot / 8) {
#pragma unroll
                                for (int j = 0; j < 8; ++j)
                                    if (j == slot % 8) va[j] = v[j], pa[j] = pp[j];
                            }
                            const f32x16 one = T::mfma32(va, pa, f32x16{});
                            if (sees(key0 + 16 * t16 + 8 * (slot % 8 / 4) + 4 * (slot / 8) + slot % 4, pos, window, sinks))
                                o[d] += one;
                        }
                        continue;
                    }
                }
                o[d] = T::mfma32(v, __builtin_bit_cast(s16x8, p[t16]), o[d]);
            }
    }
    l += __shfl_xor(l, 32);
    if (!store) return;
    const float inv = l > 0.0f ? 1.0f / l : l;   // NaN stays NaN
    short* out = (short*)a.out + (seq.first + token) * a.out_token_stride + q_head * a.out_head_stride + 4 * h;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            *(u32x2*)(out + 32 * d + 2 * i) =
                u32x2{T::pack(o[d][i] * inv, o[d][i + 1] * inv), T::pack(o[d][i + 2] * inv, o[d][i + 3] * inv)};
    if (a.lse && h == 0)
        a.lse[(int64_t)(seq.first + token) * a.q_heads + q_head] = l == 0.0f ? -INFINITY : m * kLn2 + logf(l);
}

bool aligned(const void* p, uintptr_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

int check(const ls_hip_attention& a) {
    if (!a.q || !a.out || !a.k_pages || !a.v_pages || !a.page_table || !a.q_start || !a.context) return EINVAL;
    if (!a.sequences || !a.q_heads || !a.kv_heads || a.q_heads % a.kv_heads || !a.pages || !a.table_width) return EINVAL;
    if (!a.page_size || (a.page_size & (a.page_size - 1)) || a.dtype > LS_TYPE_F32) return EINVAL;
    if (a.tokens > 0x7fffffffu || a.pages > 0x7fffffffu || a.window > 0x3fffffffu || a.sinks > 0x3fffffffu ||
        a.max_context > 0x3fffffffu || (uint64_t)a.table_width * a.page_size < a.max_context || a.max_new > a.tokens)
        return EINVAL;
    if (a.table_stride < 0 || (a.sequences > 1 && a.table_stride < (int64_t)a.table_width) || !(std::fabs(a.scale) < INFINITY))
        return EINVAL;
    if (!aligned(a.q, 16) || !aligned(a.out, 16) || !aligned(a.k_pages, 16) || !aligned(a.v_pages, 16) ||
        !aligned(a.workspace, 16))
        return EINVAL;
    const int64_t strides[] = {a.q_token_stride, a.q_head_stride, a.out_token_stride, a.out_head_stride, a.k_page_stride,
                               a.k_head_stride, a.k_slot_stride, a.v_page_stride, a.v_head_stride, a.v_slot_stride};
    for (int64_t s : strides)
        if (s < 0 || s % 8) return EINVAL;
    // a page's slots are reached with 32-bit offsets
    if ((uint64_t)a.k_slot_stride * a.page_size > 0x3fffffffu || (uint64_t)a.v_slot_stride * a.page_size > 0x3fffffffu)
        return ENOTSUP;
    if (a.dtype == LS_TYPE_F32 || (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256)) return ENOTSUP;
    if ((uint64_t)a.max_new * (a.q_heads / a.kv_heads) > 0x3fffffffu || a.sequences > 65535) return ENOTSUP;
    return 0;
}

// Splits of the sequences that take the row kernel: enough workgroups to fill the card, none with less than a
// step for each of its waves. Where there are kFill groups already, there is one split.
SplitPlan plan_rows(const ls_hip_attention& a) {
    const uint32_t rows = std::min<uint64_t>((uint64_t)a.max_new * (a.q_heads / a.kv_heads), kShortRows);
    SplitPlan p{};
    p.row_blocks = (rows + kRows - 1) / kRows;
    p.rows = std::min<uint32_t>(rows, kRows);
    uint64_t steps = (a.max_context + kStepKeys - 1) / kStepKeys;
    if (a.window)
        steps = std::min<uint64_t>(steps, ((uint64_t)a.window + a.max_new + kStepKeys - 1) / kStepKeys + 1 +
                                              (a.sinks + kStepKeys - 1) / kStepKeys);
    const uint64_t groups = (uint64_t)a.sequences * a.kv_heads * p.row_blocks;
    const uint64_t chunk = std::max<uint64_t>(1, (steps * groups + kFill - 1) / kFill);
    p.chunk = (uint32_t)std::min<uint64_t>((chunk + kRowWaves - 1) / kRowWaves * kRowWaves, 1u << 30);
    p.splits = (uint32_t)std::max<uint64_t>(1, (steps + p.chunk - 1) / p.chunk);
    if (p.splits > 1) p.bytes = kCounterBytes + groups * p.splits * p.rows * (a.head_dim + 2) * sizeof(float);
    return p;
}

template <class T, int D>
void launch(const ls_hip_attention& a, hipStream_t stream) {
    const uint32_t group = a.q_heads / a.kv_heads, rows = a.max_new * group, shift = __builtin_ctz(a.page_size);
    if (group <= (uint32_t)kShortRows) {
        const SplitPlan plan = plan_rows(a);
        const dim3 grid(plan.splits * a.kv_heads, a.sequences, plan.row_blocks);
        if (a.page_size >= 16) attention_rows_kernel<T, D, true><<<grid, 64 * kRowWaves, 0, stream>>>(a, shift, plan);
        else attention_rows_kernel<T, D, false><<<grid, 64 * kRowWaves, 0, stream>>>(a, shift, plan);
    }
    if (rows > (uint32_t)kShortRows) {
        const dim3 grid((rows + kTileRows - 1) / kTileRows * a.kv_heads, a.sequences);
        attention_tile_kernel<T, D><<<grid, 64 * kTileWaves, 0, stream>>>(a, shift);
    }
}

template <class T>
void launch(const ls_hip_attention& a, hipStream_t stream) {
    if (a.head_dim == 64) launch<T, 64>(a, stream);
    else if (a.head_dim == 128) launch<T, 128>(a, stream);
    else launch<T, 256>(a, stream);
}

}  // namespace
}  // namespace lsamd

extern "C" uint64_t ls_hip_attention_workspace(const ls_hip_attention* a) {
    using namespace lsamd;
    if (!a || check(*a) || !a->tokens || !a->max_new || a->q_heads / a->kv_heads > (uint32_t)kShortRows) return 0;
    return plan_rows(*a).bytes;
}

extern "C" int ls_hip_attention_enqueue(const ls_hip_attention* a, void* stream) {
    using namespace lsamd;
    if (!a) return EINVAL;
    if (const int rc = check(*a)) return rc;
    if (!a->tokens || !a->max_new) return 0;
    const uint64_t need = ls_hip_attention_workspace(a);
    if (need && (!a->workspace || a->workspace_bytes < need)) return ENOSPC;
    if (a->dtype == LS_TYPE_F16) launch<F16>(*a, static_cast<hipStream_t>(stream));
    else launch<BF16>(*a, static_cast<hipStream_t>(stream));
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : static_cast<int>(e);
}
