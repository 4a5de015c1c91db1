// The row operators around the blocks of a decode step: rotary positions and the cache's new slots
// (ls_hip_append_enqueue), and the norms and the residual between two blocks (ls_hip_block_norm_enqueue).
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <cerrno>
#include <cmath>
#include "leanstream_hip.h"

namespace lsamd {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxWidth = 16384;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_float(__bf16 x) { return (float)x; }

__device__ __forceinline__ float block_sum(float x, float* scratch) {
#pragma unroll
    for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.0f;
    for (int i = 0; i < kThreads / 64; ++i) x += scratch[i];
    return x;
}

// One workgroup a row. The row of z, then of h, stays in LDS (fp32) between the passes.
template <class T>
__global__ __launch_bounds__(kThreads) void block_norm_kernel(const ls_hip_block_norm a) {
    extern __shared__ float row[];
    __shared__ float scratch[kThreads / 64];
    const int64_t r = blockIdx.x;
    const T* block = (const T*)a.block + r * a.block_stride;
    const T* residual = (const T*)a.residual + r * a.residual_stride;
    const T* gate = (const T*)a.gate + r * a.gate_stride;
    const T* post = (const T*)a.post_weight;
    const T* pre = (const T*)a.pre_weight;
    const float n = (float)a.width;

    float sum = 0.0f;
    for (uint32_t i = threadIdx.x; i < a.width; i += kThreads) {
        const float y = to_float(block[i]);
        row[i] = y;
        sum += y * y;
    }
    float inv = 1.0f;
    if (post) inv = 1.0f / sqrtf(block_sum(sum, scratch) / n + a.eps);
    sum = 0.0f;
    for (uint32_t i = threadIdx.x; i < a.width; i += kThreads) {
        float z = row[i];
        if (post) z = z * inv * (a.weight_offset + to_float(post[i]));
        if (a.gate) z *= to_float(gate[i]);
        const float h = a.residual_scale * to_float(residual[i]) + z;
        row[i] = h;
        sum += h * h;
    }
    if (a.normed) inv = 1.0f / sqrtf(block_sum(sum, scratch) / n + a.eps);
    else __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.width; i += kThreads) {
        const float h = row[i];
        if (a.hidden) ((T*)a.hidden)[r * a.hidden_stride + i] = (T)h;
        if (a.normed) ((T*)a.normed)[r * a.normed_stride + i] = (T)(h * inv * (a.weight_offset + to_float(pre[i])));
    }
}

// The sequence that holds row t of q: the last one that starts at or before it.
__device__ __forceinline__ int find_sequence(const int32_t* q_start, uint32_t sequences, int t) {
    int lo = 0, hi = (int)sequences;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (q_start[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// One workgroup a token: its q and k heads are rotated and its k and v put into the slot of its position.
template <class T>
__global__ __launch_bounds__(kThreads) void append_kernel(const ls_hip_append a, uint32_t page_shift) {
    const int64_t t = blockIdx.x;
    const int s = find_sequence(a.q_start, a.sequences, (int)t);
    const int first = a.q_start[s], end = a.q_start[s + 1];
    if (t < first || t >= end) return;   // no sequence's token
    const int pos = a.context[s] - (end - (int)t);
    if (pos < 0 || (a.rot && (uint32_t)pos >= a.positions) || (uint32_t)(pos >> page_shift) >= a.table_width) {
        if (threadIdx.x == 0 && a.status) atomicOr(a.status, (uint32_t)LS_STATUS_RANGE);
        return;
    }
    const int page = a.page_table[s * a.table_stride + (pos >> page_shift)];
    const int slot = pos & ((1 << page_shift) - 1);
    if ((uint32_t)page >= a.pages) {
        if (threadIdx.x == 0 && a.status) atomicOr(a.status, (uint32_t)LS_STATUS_BAD_DESCRIPTOR);
        return;
    }
    const uint32_t pairs = a.head_dim / 2, half = a.rot / 2;
    const float* cosine = a.cos + (int64_t)pos * half;
    const float* sine = a.sin + (int64_t)pos * half;
    const uint32_t heads = a.q_heads + 2 * a.kv_heads;
    for (uint32_t i = threadIdx.x; i < heads * pairs; i += kThreads) {
        const uint32_t head = i / pairs, j = i % pairs;
        const T* src;
        T* dst;
        bool turn = j < half;
        if (head < a.q_heads) {
            src = (const T*)a.q + t * a.q_token_stride + head * a.q_head_stride;
            dst = (T*)a.q_out + t * a.q_out_token_stride + head * a.q_out_head_stride;
        } else if (head < a.q_heads + a.kv_heads) {
            const uint32_t h = head - a.q_heads;
            src = (const T*)a.k + t * a.k_token_stride + h * a.k_head_stride;
            dst = (T*)a.k_pages + page * a.k_page_stride + h * a.k_head_page_stride + slot * a.k_slot_stride;
        } else {
            const uint32_t h = head - a.q_heads - a.kv_heads;
            src = (const T*)a.v + t * a.v_token_stride + h * a.v_head_stride;
            dst = (T*)a.v_pages + page * a.v_page_stride + h * a.v_head_page_stride + slot * a.v_slot_stride;
            turn = false;
        }
        // pair j: rotated (j, j + rot / 2) or (2 j, 2 j + 1); from rot on (2 j, 2 j + 1) as they are
        const bool apart = j < half && !a.interleaved;
        const uint32_t x = apart ? j : 2 * j, y = apart ? j + half : 2 * j + 1;
        const T p = src[x], q = src[y];
        if (turn) {
            const float c = cosine[j], sn = sine[j], u = to_float(p), v = to_float(q);
            dst[x] = (T)(u * c - v * sn);
            dst[y] = (T)(v * c + u * sn);
        } else {
            dst[x] = p;
            dst[y] = q;
        }
    }
}

bool aligned(const void* p, uintptr_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

int check(const ls_hip_block_norm& a) {
    if (!a.block || !a.residual || (!a.hidden && !a.normed) || (a.normed && !a.pre_weight)) return EINVAL;
    if (!a.width || a.dtype > LS_TYPE_F32 || !(a.eps >= 0.0f && a.eps < INFINITY)) return EINVAL;
    if (!(std::fabs(a.residual_scale) < INFINITY) || !(std::fabs(a.weight_offset) < INFINITY)) return EINVAL;
    const uintptr_t element = a.dtype == LS_TYPE_F32 ? 4 : 2;
    for (const void* p : {a.block, a.residual, a.gate, a.post_weight, a.pre_weight, (const void*)a.hidden, (const void*)a.normed})
        if (!aligned(p, element)) return EINVAL;
    if (a.block_stride < 0 || a.residual_stride < 0 || a.gate_stride < 0) return EINVAL;
    if (a.rows > 1 && ((a.hidden && a.hidden_stride < (int64_t)a.width) || (a.normed && a.normed_stride < (int64_t)a.width)))
        return EINVAL;   // rows of an output must not overlap
    if (a.width > kMaxWidth || a.rows > 0x7fffffffu) return ENOTSUP;
    return 0;
}

int check(const ls_hip_append& a) {
    if (!a.k || !a.v || !a.k_pages || !a.v_pages || !a.page_table || !a.q_start || !a.context) return EINVAL;
    if ((a.q_heads && (!a.q || !a.q_out)) || (a.rot && (!a.cos || !a.sin || !a.positions))) return EINVAL;
    if (!a.sequences || !a.kv_heads || !a.head_dim || a.head_dim % 2 || a.rot % 2 || a.rot > a.head_dim) return EINVAL;
    if (!a.page_size || (a.page_size & (a.page_size - 1)) || !a.pages || !a.table_width || a.dtype > LS_TYPE_F32) return EINVAL;
    if (a.tokens > 0x7fffffffu || a.sequences > 0x7fffffffu || a.pages > 0x7fffffffu) return EINVAL;
    if (a.table_stride < 0 || (a.sequences > 1 && a.table_stride < (int64_t)a.table_width)) return EINVAL;
    for (const void* p : {a.q, a.k, a.v, (const void*)a.q_out, (const void*)a.k_pages, (const void*)a.v_pages})
        if (!aligned(p, 2)) return EINVAL;
    const int64_t strides[] = {a.q_token_stride, a.q_head_stride, a.k_token_stride, a.k_head_stride, a.v_token_stride,
                               a.v_head_stride, a.q_out_token_stride, a.q_out_head_stride, a.k_page_stride,
                               a.k_head_page_stride, a.k_slot_stride, a.v_page_stride, a.v_head_page_stride, a.v_slot_stride};
    for (int64_t s : strides)
        if (s < 0) return EINVAL;
    if (a.dtype == LS_TYPE_F32) return ENOTSUP;
    if ((uint64_t)(a.q_heads + 2ull * a.kv_heads) * a.head_dim > 0x3fffffffu) return ENOTSUP;
    return 0;
}

int finish() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : static_cast<int>(e);
}

}  // namespace
}  // namespace lsamd

extern "C" int ls_hip_block_norm_enqueue(const ls_hip_block_norm* a, void* stream) {
    using namespace lsamd;
    if (!a) return EINVAL;
    if (const int rc = check(*a)) return rc;
    if (!a->rows) return 0;
    const auto st = static_cast<hipStream_t>(stream);
    const size_t lds = a->width * sizeof(float);
    if (a->dtype == LS_TYPE_F16) block_norm_kernel<_Float16><<<a->rows, kThreads, lds, st>>>(*a);
    else if (a->dtype == LS_TYPE_BF16) block_norm_kernel<__bf16><<<a->rows, kThreads, lds, st>>>(*a);
    else block_norm_kernel<float><<<a->rows, kThreads, lds, st>>>(*a);
    return finish();
}

extern "C" int ls_hip_append_enqueue(const ls_hip_append* a, void* stream) {
    using namespace lsamd;
    if (!a) return EINVAL;
    if (const int rc = check(*a)) return rc;
    if (!a->tokens) return 0;
    const auto st = static_cast<hipStream_t>(stream);
    const uint32_t shift = __builtin_ctz(a->page_size);
    if (a->dtype == LS_TYPE_F16) append_kernel<_Float16><<<a->tokens, kThreads, 0, st>>>(*a, shift);
    else append_kernel<__bf16><<<a->tokens, kThreads, 0, st>>>(*a, shift);
    return finish();
}
