// The row operators around the blocks of a decode step: rotary positions and the cache's new slots
// (ls_hip_append_enqueue), and the norms and the residual between two blocks (ls_hip_block_norm_enqueue).
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <cerrno>
#include <cmath>
#include <type_traits>
#include "kernel_launch.h"
#include "leanstream_hip.h"
#include "wave_ops.h"

namespace lsamd {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxWidth = 16384;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_float(__bf16 x) { return (float)x; }

// Eight elements at any element's alignment, loaded and stored as 16-byte words.
template <class T>
struct Vec8 {
    typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    typedef T half __attribute__((ext_vector_type(4), aligned(sizeof(T))));
};

// The i-th eight of a row of `width` elements; zeros beyond its end.
template <class T>
__device__ __forceinline__ typename Vec8<T>::type load8(const T* row, uint32_t i, uint32_t width) {
    typename Vec8<T>::type v = {};
    if (8 * i + 8 <= width) v = *(const typename Vec8<T>::type*)(row + 8 * i);
    else
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (8 * i + j < width) v[j] = row[8 * i + j];
    return v;
}
template <class T>
__device__ __forceinline__ void store8(T* row, uint32_t i, uint32_t width, const float (&x)[8]) {
    typename Vec8<T>::type v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (T)x[j];
    if (8 * i + 8 <= width) *(typename Vec8<T>::type*)(row + 8 * i) = v;
    else
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (8 * i + j < width) row[8 * i + j] = v[j];
}

// Sum over the waves of a row.
template <int Waves>
__device__ __forceinline__ float row_sum(float x, float* scratch) {
    x = wave_sum(x);
    if constexpr (Waves > 1) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
        __syncthreads();
        x = 0.0f;
#pragma unroll
        for (int i = 0; i < Waves; ++i) x += scratch[i];
    }
    return x;
}

// Bound by memory: every input is read once, all of a thread's loads are under way before the first sum, and
// the row stays in registers (fp32) from there on. 8192 rows of 8192 in bf16 with a gate for every element: 120 us,
// 5.6 TB/s (through LDS and element by element: 589). One row of 4096: 3 us. Vecs: eights of a thread.
// Rows of up to 2048 columns take one wave (no barriers), four to a workgroup, longer ones the whole workgroup: 8192
// rows of 512 8.7 and 34.6 us, of 1024 14.2 and 33.2 (22.4 with registers for 2048), of 2048 27.3 and 34.8.
template <class T, int Waves, int Vecs>
__global__ __launch_bounds__(kThreads) void block_norm_kernel(const ls_hip_block_norm a) {
    __shared__ float scratch[Waves];
    constexpr uint32_t kLanes = 64 * Waves;
    const int64_t r = Waves > 1 ? blockIdx.x : blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (r >= (int64_t)a.rows) return;   // a wave of its own row: no barrier follows
    const uint32_t lane = threadIdx.x % kLanes, width = a.width;
    const T* block = (const T*)a.block + r * a.block_stride;
    const T* residual = (const T*)a.residual + r * a.residual_stride;
    const T* gate = (const T*)a.gate + r * a.gate_stride;
    const T* post = (const T*)a.post_weight;
    const T* pre = (const T*)a.pre_weight;
    const float n = (float)width;

    typename Vec8<T>::type y[Vecs], res[Vecs], gt[Vecs] = {};
#pragma unroll
    for (int v = 0; v < Vecs; ++v) y[v] = load8(block, lane + v * kLanes, width);
#pragma unroll
    for (int v = 0; v < Vecs; ++v) res[v] = load8(residual, lane + v * kLanes, width);
    if (gate)
#pragma unroll
        for (int v = 0; v < Vecs; ++v) gt[v] = load8(gate, lane + v * kLanes, width);
    // Rows of few registers hold the weights too, so that one row waits for memory once; many long rows find them in
    // the caches, and the registers are better spent on more waves.
    constexpr bool kEarly = Vecs <= 2;
    typename Vec8<T>::type before[kEarly ? Vecs : 1] = {}, after[kEarly ? Vecs : 1] = {};
    if constexpr (kEarly) {
        if (post)
#pragma unroll
            for (int v = 0; v < Vecs; ++v) before[v] = load8(post, lane + v * kLanes, width);
        if (a.normed)
#pragma unroll
            for (int v = 0; v < Vecs; ++v) after[v] = load8(pre, lane + v * kLanes, width);
    }

    float inv = 1.0f;
    if (post) {
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < Vecs; ++v)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += to_float(y[v][j]) * to_float(y[v][j]);
        inv = 1.0f / sqrtf(row_sum<Waves>(sum, scratch) / n + a.eps);
    }
    float h[Vecs][8], sum = 0.0f;
#pragma unroll
    for (int v = 0; v < Vecs; ++v) {
        typename Vec8<T>::type w = {};
        if (post) w = kEarly ? before[kEarly ? v : 0] : load8(post, lane + v * kLanes, width);
        const bool in = 8 * (lane + v * kLanes) < width;   // beyond the end 0 * inv may be NaN
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float z = to_float(y[v][j]);
            if (post) z = z * inv * (a.weight_offset + to_float(w[j]));
            if (gate) z *= to_float(gt[v][j]);
            h[v][j] = a.residual_scale * to_float(res[v][j]) + z;
            if (in && 8 * (lane + v * kLanes) + j < width) sum += h[v][j] * h[v][j];
        }
    }
    if (a.hidden)
#pragma unroll
        for (int v = 0; v < Vecs; ++v) store8((T*)a.hidden + r * a.hidden_stride, lane + v * kLanes, width, h[v]);
    if (!a.normed) return;
    inv = 1.0f / sqrtf(row_sum<Waves>(sum, scratch) / n + a.eps);
#pragma unroll
    for (int v = 0; v < Vecs; ++v) {
        const typename Vec8<T>::type w = kEarly ? after[kEarly ? v : 0] : load8(pre, lane + v * kLanes, width);
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = h[v][j] * inv * (a.weight_offset + to_float(w[j]));
        store8((T*)a.normed + r * a.normed_stride, lane + v * kLanes, width, x);
    }
}

template <class T>
hipError_t launch_norm(const ls_hip_block_norm& a, hipStream_t st) {
    const uint32_t w = a.width, packed = (a.rows + kThreads / 64 - 1) / (kThreads / 64);
    const auto kernel = w <= 512    ? block_norm_kernel<T, 1, 1>
                        : w <= 1024 ? block_norm_kernel<T, 1, 2>
                        : w <= 2048 ? block_norm_kernel<T, 1, 4>
                        : w <= 4096 ? block_norm_kernel<T, 4, 2>
                        : w <= 8192 ? block_norm_kernel<T, 4, 4>
                                    : block_norm_kernel<T, 4, 8>;
    return launch_kernel(kernel, dim3(w <= 2048 ? packed : a.rows), kThreads, st, a);
}

// Lengths and page tables do not change while a kernel runs: uniform ones come over the scalar cache.
#if defined(__HIP_DEVICE_COMPILE__)
typedef const __attribute__((address_space(4))) int32_t* Table;
#else
typedef const int32_t* Table;
#endif

// One workgroup a token: its q and k heads are rotated and its k and v put into the slot of its position.
// Bound by memory, for few tokens by the latency of q_start -> context -> page -> tables: a thread's first values are
// loaded before. Chunks of 8 dimensions go in 16-byte words where the head and the rotated part divide into them
// (Wide); otherwise dimensions go alone. 8192 tokens of 64 + 8 + 8 heads of 128: 70 us, 4.8 TB/s (alone: 114).
// Threads of a token: up to a token a compute unit the wait for its first values counts (32 tokens: 4.1 us with 512,
// 4.6 with 256), beyond it the workgroups under way (8192 tokens: 81 and 70 us).
constexpr uint32_t kAppendThreads = 512;
constexpr uint32_t kAppendFew = 256;
template <class T, bool Wide, uint32_t Threads>
__global__ __launch_bounds__(Threads) void append_kernel(const ls_hip_append a, uint32_t page_shift) {
    typedef typename Vec8<T>::type vec8;
    typedef typename Vec8<float>::half float4u;
    typedef std::conditional_t<Wide, vec8, T> Piece;
    const int64_t t = blockIdx.x;
    const uint32_t lane = threadIdx.x & 63;
    const int start = a.q_start[min(lane, a.sequences - 1)];   // of the first 64 sequences

    // Units of a token: rotated ones (q heads, then k heads), copied ones of q and k, then v. A rotated unit is a pair
    // of pieces, or with interleaved pairs in 16-byte words one piece.
    constexpr uint32_t kUnit = Wide ? 8 : 1;
    const uint32_t half = a.rot / 2, heads = a.q_heads + a.kv_heads;
    const bool lone = a.interleaved && Wide;
    const uint32_t turned = lone ? a.rot / 8 : half / kUnit, plain = (a.head_dim - a.rot) / kUnit;
    const uint32_t whole = a.head_dim / kUnit;
    const uint32_t turn_units = heads * turned, plain_units = turn_units + heads * plain;
    const uint32_t units = plain_units + a.kv_heads * whole;
    int64_t pos = -1, slot = 0;
    int page = 0;
    for (uint32_t i0 = 0; i0 < units; i0 += Threads) {
        const uint32_t i = min(i0 + threadIdx.x, units - 1);   // beyond the end: loaded only
        const bool turn = i < turn_units, value = i >= plain_units;
        const uint32_t j = turn ? i : value ? i - plain_units : i - turn_units;
        const uint32_t each = turn ? turned : value ? whole : plain;
        const uint32_t head = j / each, u = j % each;
        const bool query = !value && head < a.q_heads;
        const uint32_t kv = value || query ? head : head - a.q_heads;
        const T* src = value   ? (const T*)a.v + t * a.v_token_stride + kv * a.v_head_stride
                       : query ? (const T*)a.q + t * a.q_token_stride + kv * a.q_head_stride
                               : (const T*)a.k + t * a.k_token_stride + kv * a.k_head_stride;
        uint32_t x = kUnit * u + (turn || value ? 0 : a.rot), y = x + half;   // the dimensions of its pieces
        if (turn && !Wide && a.interleaved) x = 2 * u, y = 2 * u + 1;
        const Piece p = *(const Piece*)(src + x);
        Piece q = p;
        if (turn && !lone) q = *(const Piece*)(src + y);

        if (pos < 0) {   // once: the sequence (the last one that starts at or before t), its length, the page
            int s = 0;
            for (uint32_t s0 = 0; s0 < a.sequences; s0 += 64) {
                const int first = s0 ? a.q_start[min(s0 + lane, a.sequences - 1)] : start;
                const uint32_t count = __popcll(__ballot(s0 + lane < a.sequences && first <= t));
                if (!count) break;
                s = (int)(s0 + count) - 1;
            }
            s = __builtin_amdgcn_readfirstlane(s);
            const int first = ((Table)a.q_start)[s], end = ((Table)a.q_start)[s + 1];
            if (t < first || t >= end) return;   // no sequence's token
            pos = (int64_t)((Table)a.context)[s] - (end - t);
            if (pos < 0 || (a.rot && pos >= (int64_t)a.positions) || (pos >> page_shift) >= (int64_t)a.table_width) {
                if (threadIdx.x == 0 && a.status) atomicOr(a.status, (uint32_t)LS_STATUS_RANGE);
                return;
            }
            page = ((Table)a.page_table)[s * a.table_stride + (pos >> page_shift)];
            slot = pos & ((1 << page_shift) - 1);
            if ((uint32_t)page >= a.pages) {
                if (threadIdx.x == 0 && a.status) atomicOr(a.status, (uint32_t)LS_STATUS_BAD_DESCRIPTOR);
                return;
            }
        }
        if (i0 + threadIdx.x >= units) return;
        T* dst = value   ? (T*)a.v_pages + page * a.v_page_stride + kv * a.v_head_page_stride + slot * a.v_slot_stride
                 : query ? (T*)a.q_out + t * a.q_out_token_stride + kv * a.q_out_head_stride
                         : (T*)a.k_pages + page * a.k_page_stride + kv * a.k_head_page_stride + slot * a.k_slot_stride;
        if (!turn) {
            *(Piece*)(dst + x) = p;
            continue;
        }
        const float* cosine = a.cos + pos * half;
        const float* sine = a.sin + pos * half;
        if constexpr (!Wide) {
            const float c = cosine[u], sn = sine[u], v = to_float(p), w = to_float(q);
            dst[x] = (T)(v * c - w * sn);
            dst[y] = (T)(w * c + v * sn);
        } else if (lone) {   // four pairs
            const float4u c = *(const float4u*)(cosine + 4 * u), sn = *(const float4u*)(sine + 4 * u);
            vec8 r;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float v = to_float(p[2 * k]), w = to_float(p[2 * k + 1]);
                r[2 * k] = (T)(v * c[k] - w * sn[k]);
                r[2 * k + 1] = (T)(w * c[k] + v * sn[k]);
            }
            *(vec8*)(dst + x) = r;
        } else {   // eight pairs
            const float4u c0 = *(const float4u*)(cosine + x), c1 = *(const float4u*)(cosine + x + 4);
            const float4u s0 = *(const float4u*)(sine + x), s1 = *(const float4u*)(sine + x + 4);
            vec8 r, r2;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float v = to_float(p[k]), w = to_float(q[k]), c = k < 4 ? c0[k % 4] : c1[k % 4],
                            sn = k < 4 ? s0[k % 4] : s1[k % 4];
                r[k] = (T)(v * c - w * sn);
                r2[k] = (T)(w * c + v * sn);
            }
            *(vec8*)(dst + x) = r;
            *(vec8*)(dst + y) = r2;
        }
    }
}

bool aligned(const void* p, uintptr_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

int check(const ls_hip_block_norm& a) {
    // the pointers of empty tensors may be NULL
    if (a.rows && (!a.block || !a.residual || (!a.hidden && !a.normed) || (a.normed && !a.pre_weight))) return EINVAL;
    if (!a.width || a.dtype > LS_TYPE_F32 || !(a.eps >= 0.0f && a.eps < INFINITY)) return EINVAL;
    if (!(std::fabs(a.residual_scale) < INFINITY) || !(std::fabs(a.weight_offset) < INFINITY)) return EINVAL;
    const uintptr_t element = a.dtype == LS_TYPE_F32 ? 4 : 2;
    for (const void* p : {a.block, a.residual, a.gate, a.post_weight, a.pre_weight, (const void*)a.hidden,
         (const void*)a.normed})
        if (!aligned(p, element)) return EINVAL;
    if (a.block_stride < 0 || a.residual_stride < 0 || a.gate_stride < 0) return EINVAL;
    if (a.rows > 1 && ((a.hidden && a.hidden_stride < (int64_t)a.width) || 
                       (a.normed && a.normed_stride < (int64_t)a.width)))
        return EINVAL;   // rows of an output must not overlap
    if (a.width > kMaxWidth || a.rows > 0x7fffffffu) return ENOTSUP;
    return 0;
}

int check(const ls_hip_append& a) {
    if (a.tokens && (!a.k || !a.v || !a.k_pages || !a.v_pages || !a.page_table || !a.q_start || !a.context ||
                     !a.sequences || !a.pages || !a.table_width || (a.q_heads && (!a.q || !a.q_out)) ||
                     (a.rot && (!a.cos || !a.sin || !a.positions))))
        return EINVAL;
    if (!a.kv_heads || !a.head_dim || a.head_dim % 2 || a.rot % 2 || a.rot > a.head_dim) return EINVAL;
    if (!a.page_size || (a.page_size & (a.page_size - 1)) || a.dtype > LS_TYPE_F32) return EINVAL;
    if (a.tokens > 0x7fffffffu || a.sequences > 0x7fffffffu || a.pages > 0x7fffffffu) return EINVAL;
    if (a.table_stride < 0 || (a.sequences > 1 && a.table_stride < (int64_t)a.table_width)) return EINVAL;
    for (const void* p : {a.q, a.k, a.v, (const void*)a.q_out, (const void*)a.k_pages, (const void*)a.v_pages})
        if (!aligned(p, 2)) return EINVAL;
    for (const void* p : {(const void*)a.cos, (const void*)a.sin, (const void*)a.page_table, (const void*)a.q_start,
                          (const void*)a.context, (const void*)a.status})
        if (!aligned(p, 4)) return EINVAL;
    const int64_t strides[] = {a.q_token_stride, a.q_head_stride, a.k_token_stride, a.k_head_stride, a.v_token_stride,
                               a.v_head_stride, a.q_out_token_stride, a.q_out_head_stride, a.k_page_stride,
                               a.k_head_page_stride, a.k_slot_stride, a.v_page_stride, a.v_head_page_stride,
                               a.v_slot_stride};
    for (int64_t s : strides)
        if (s < 0) return EINVAL;
    if (a.dtype == LS_TYPE_F32) return ENOTSUP;
    if ((uint64_t)(a.q_heads + 2ull * a.kv_heads) * a.head_dim > 0x3fffffffu) return ENOTSUP;
    return 0;
}

}  // namespace
}  // namespace lsamd

extern "C" int ls_hip_block_norm_enqueue(const ls_hip_block_norm* a, void* stream) {
    using namespace lsamd;
    if (!a) return EINVAL;
    if (const int rc = check(*a)) return rc;
    if (!a->rows) return 0;
    const auto st = static_cast<hipStream_t>(stream);
    return static_cast<int>(a->dtype == LS_TYPE_F16    ? launch_norm<_Float16>(*a, st)
                            : a->dtype == LS_TYPE_BF16 ? launch_norm<__bf16>(*a, st)
                                                       : launch_norm<float>(*a, st));
}

extern "C" int ls_hip_append_enqueue(const ls_hip_append* a, void* stream) {
    using namespace lsamd;
    if (!a) return EINVAL;
    if (const int rc = check(*a)) return rc;
    if (!a->tokens) return 0;
    const auto st = static_cast<hipStream_t>(stream);
    const uint32_t shift = __builtin_ctz(a->page_size);
    const bool wide = a->head_dim % 8 == 0 && a->rot % (a->interleaved ? 8 : 16) == 0;
    const auto launch = [&](auto threads) {
        constexpr uint32_t n = decltype(threads)::value;
        const auto kernel = a->dtype == LS_TYPE_F16
                                ? wide ? append_kernel<_Float16, true, n> : append_kernel<_Float16, false, n>
                                : wide ? append_kernel<__bf16, true, n> : append_kernel<__bf16, false, n>;
        return launch_kernel(kernel, dim3(a->tokens), n, st, *a, shift);
    };
    return static_cast<int>(a->tokens <= kAppendFew ? launch(std::integral_constant<uint32_t, kAppendThreads>())
                                                    : launch(std::integral_constant<uint32_t, kAppendThreads / 2>()));
}
