// A cache of keys and values in 8-bit integers: what its kernels share (cache.hip, attention_cache.hip).
//
// A page holds 64 tokens of a sequence, every key head's 64 keys and values side by side:
//   keys    [page][head][token][pitch]   `pitch` the head's elements rounded up to 16: a row of keys is whole 16-byte pieces
//   values  [page][head][pitch][token]   transposed, so that sixteen tokens of one element are a piece: the second product of attention sums over tokens,
//                                        and a lane reads its operand from memory as it needs it
//   scales  [page][head]                 of keys and of values: a code stands for code * scale
// Bytes between a head's elements and its pitch, and of tokens that are not there, mean nothing: a whole number times a weight of 0 is 0.
#ifndef DEEP8_AMD_CACHE_H
#define DEEP8_AMD_CACHE_H

#include "common.h"

namespace d8 {
namespace cache {

enum { PAGE = D8_CACHE_PAGE, MOST_DIM = 256 };
constexpr float LEAST_SCALE = 7.888609052210118e-31f;  // 2^-100

typedef int i32x4 __attribute__((ext_vector_type(4)));

inline long pitch_of(int dim) { return (dim + 15L) / 16 * 16; }

struct Pages {
    signed char *k_codes, *v_codes;
    float *k_scales, *v_scales;
    const int *starts, *lengths, *table;
    int sequences, tokens, table_pages, pages, kv_heads, dim, pitch;
    __device__ __forceinline__ long tile(int page, int head) const { return ((long)page * kv_heads + head) * PAGE * pitch; }
    // the page of a sequence's tokens 64 p .. 64 p + 63, -1 if it has none
    __device__ __forceinline__ int page_of(int s, int p) const {
        if (p < 0 || p >= table_pages) return -1;
        const int page = table[(long)s * table_pages + p];
        return page >= 0 && page < pages ? page : -1;
    }
};

// a value or a mean of such; where the largest elements' codes round up past what the type holds, its largest number
template <class T>
__device__ __forceinline__ float within(float x) {
    constexpr float MOST = sizeof(T) == 2 ? 65504.f : 3.4028234663852886e38f;
    return fabsf(x) > MOST ? copysignf(MOST, x) : x;
}

int check(const Pages &p, int dtype, const char *name);

}  // namespace cache
}  // namespace d8

#endif
