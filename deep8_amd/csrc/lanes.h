// Sums and maxima over lanes without LDS (row_team.h, cache.hip, attention_cache.hip).
#ifndef DEEP8_AMD_LANES_H
#define DEEP8_AMD_LANES_H

#include "common.h"

namespace d8 {

// op over a team of 16 or 32 lanes side by side, or a wave, in all of them: within quads, with the other quad of eight and the other eight of sixteen (whose lanes
// are alike by then, so that mirrored will do), then with sixteens and halves of the wave swapped.  (Shuffles through LDS, six one after the other of some 50
// cycles each: gradients of 8192 x 2048 halves' norm 33 us, 29 so.)
template <int CTRL, class N>
__device__ __forceinline__ N moved(N x) {
    return __builtin_bit_cast(N, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int LANES, class N, class F>
__device__ __forceinline__ N over_lanes(N x, F op) {
    typedef unsigned pair __attribute__((ext_vector_type(2)));
    x = op(x, moved<0xb1>(x));   // lanes 1 0 3 2 of four
    x = op(x, moved<0x4e>(x));   // 2 3 0 1
    x = op(x, moved<0x141>(x));  // eight lanes, mirrored
    x = op(x, moved<0x140>(x));  // sixteen
    if constexpr (LANES > 16) {
        const unsigned y = __builtin_bit_cast(unsigned, x);
        const pair p = __builtin_bit_cast(pair, __builtin_amdgcn_permlane16_swap(y, y, false, false));
        const unsigned p0 = p[0], p1 = p[1];
        x = op(__builtin_bit_cast(N, p0), __builtin_bit_cast(N, p1));
    }
    if constexpr (LANES > 32) {
        const unsigned y = __builtin_bit_cast(unsigned, x);
        const pair p = __builtin_bit_cast(pair, __builtin_amdgcn_permlane32_swap(y, y, false, false));
        const unsigned p0 = p[0], p1 = p[1];
        x = op(__builtin_bit_cast(N, p0), __builtin_bit_cast(N, p1));
    }
    return x;
}

// the sum over the lanes up to this one: within sixteens, then what the sixteens, and the halves, before have
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved_or_0(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ long moved_or_0(long x) {
    return (long)((unsigned long)(unsigned)moved_or_0<CTRL, ROWS>((int)(x >> 32)) << 32 | (unsigned)moved_or_0<CTRL, ROWS>((int)x));
}
template <class N>
__device__ __forceinline__ N sum_upto_lane(N x) {
    x += moved_or_0<0x111, 0xf>(x), x += moved_or_0<0x112, 0xf>(x), x += moved_or_0<0x114, 0xf>(x), x += moved_or_0<0x118, 0xf>(x);  // lanes 1, 2, 4, 8 before
    x += moved_or_0<0x142, 0xa>(x);  // the last lane of a sixteen, into all of the next: second and fourth
    x += moved_or_0<0x143, 0xc>(x);  // lane 31, into the other half
    return x;
}

}  // namespace d8

#endif
