// Attention of new tokens over a paged cache: ls_hip_attention_enqueue.
//
// For a query row q and its visible keys: out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), s_j = scale
// q.k_j, in one pass over the keys with the running maximum m and sum (both fp32): when m rises, what was
// summed is scaled by e^(m_old - m_new). Exponentials are taken to base 2 with scale * log2(e) folded in.
//
// The query heads of one KV head share its keys, so the rows of a tile are (token, head of the group)
// pairs: row r of a sequence is token r / group, head r % group.
#include <hip/hip_runtime.h>
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
    if (row0 >= rows) return;
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

    // keys that some row of the tile sees: [0, sink_end) and [low, p_high]
    const int low = window ? max(0, p_low + 1 - window) : 0;
    const int tiles_end = p_high < 0 ? 0 : p_high / kTileKeys + 1;
    const int sink_tiles = window ? min((int)(((uint32_t)sinks + kTileKeys - 1) / kTileKeys), tiles_end) : 0;
    const int low_tile = max(low / kTileKeys, sink_tiles);

    for (int t = sink_tiles ? 0 : low_tile; t < tiles_end; t = (t + 1 == sink_tiles ? low_tile : t + 1)) {
        const int key0 = t * kTileKeys;
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
                    const u32x4 w = __builtin_bit_cast(u32x4, v);
                    bool odd = false;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        odd |= (w[j] & T::kExponent) == T::kExponent || ((w[j] >> 16) & T::kExponent) == T::kExponent;
                    if (__ballot(odd)) {
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
    if (a.dtype == LS_TYPE_F32 || (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256)) return ENOTSUP;
    if ((uint64_t)a.max_new * (a.q_heads / a.kv_heads) > 0x3fffffffu || a.sequences > 65535) return ENOTSUP;
    return 0;
}

template <class T, int D>
void launch(const ls_hip_attention& a, hipStream_t stream) {
    const uint32_t rows = a.max_new * (a.q_heads / a.kv_heads);
    const dim3 grid((rows + kTileRows - 1) / kTileRows * a.kv_heads, a.sequences);
    attention_tile_kernel<T, D><<<grid, 64 * kTileWaves, 0, stream>>>(a, __builtin_ctz(a.page_size));
}

template <class T>
void launch(const ls_hip_attention& a, hipStream_t stream) {
    if (a.head_dim == 64) launch<T, 64>(a, stream);
    else if (a.head_dim == 128) launch<T, 128>(a, stream);
    else launch<T, 256>(a, stream);
}

}  // namespace
}  // namespace lsamd

extern "C" uint64_t ls_hip_attention_workspace(const ls_hip_attention*) { return 0; }

extern "C" int ls_hip_attention_enqueue(const ls_hip_attention* a, void* stream) {
    using namespace lsamd;
    if (!a) return EINVAL;
    if (const int rc = check(*a)) return rc;
    if (!a->tokens || !a->max_new) return 0;
    if (!a->workspace ? ls_hip_attention_workspace(a) > 0 : a->workspace_bytes < ls_hip_attention_workspace(a)) return ENOSPC;
    if (a->dtype == LS_TYPE_F16) launch<F16>(*a, static_cast<hipStream_t>(stream));
    else launch<BF16>(*a, static_cast<hipStream_t>(stream));
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : static_cast<int>(e);
}
