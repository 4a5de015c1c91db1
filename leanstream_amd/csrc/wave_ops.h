// Sums, maxima and running sums over the 64 lanes of a wave, by lane moves of the vector units (a move takes a few
// cycles; a shuffle goes through LDS and takes over a hundred). Values are of 4 or 8 bytes; all lanes take part.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lsamd {

// x of the lane that a lane-move control names; `other` where there is none or the row is masked out.
template <int Control, int RowMask, class V>
__device__ __forceinline__ V moved(V x, V other) {
    static_assert(sizeof(V) == 4 || sizeof(V) == 8, "4 or 8 bytes");
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, other), __builtin_bit_cast(int, x),
                                                                 Control, RowMask, 0xf, false));
    } else {
        struct Halves {
            int low, high;
        };
        const Halves a = __builtin_bit_cast(Halves, x), b = __builtin_bit_cast(Halves, other);
        return __builtin_bit_cast(V, Halves{__builtin_amdgcn_update_dpp(b.low, a.low, Control, RowMask, 0xf, false),
                                            __builtin_amdgcn_update_dpp(b.high, a.high, Control, RowMask, 0xf, false)});
    }
}

// Lane i: op over the lanes 0 .. i. Within rows of 16 lanes by moves of 1, 2, 4 and 8, then from row to row.
template <class V, class Op>
__device__ __forceinline__ V wave_upto(V x, V nothing, Op op) {
    x = op(moved<0x111, 0xf>(x, nothing), x);
    x = op(moved<0x112, 0xf>(x, nothing), x);
    x = op(moved<0x114, 0xf>(x, nothing), x);
    x = op(moved<0x118, 0xf>(x, nothing), x);
    x = op(moved<0x142, 0xa>(x, nothing), x);   // the last lane of rows 0 and 2 to rows 1 and 3
    x = op(moved<0x143, 0xc>(x, nothing), x);   // lane 31 to rows 2 and 3
    return x;
}
template <class V>
__device__ __forceinline__ V wave_upto(V x) {
    return wave_upto(x, V(0), [](V a, V b) { return a + b; });
}

// The value of one lane (the same number in all lanes), in all of them.
template <class V>
__device__ __forceinline__ V from_lane(V x, int lane) {
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
    } else {
        struct Halves {
            int low, high;
        };
        const Halves a = __builtin_bit_cast(Halves, x);
        return __builtin_bit_cast(V, Halves{__builtin_amdgcn_readlane(a.low, lane), __builtin_amdgcn_readlane(a.high, lane)});
    }
}

template <class V>
__device__ __forceinline__ V wave_sum(V x) {
    return from_lane(wave_upto(x), 63);
}
template <class V>
__device__ __forceinline__ V wave_max(V x, V lowest) {
    return from_lane(wave_upto(x, lowest, [](V a, V b) { return a > b ? a : b; }), 63);
}
template <class V>
__device__ __forceinline__ V wave_min(V x, V highest) {
    return from_lane(wave_upto(x, highest, [](V a, V b) { return a < b ? a : b; }), 63);
}

}  // namespace lsamd
