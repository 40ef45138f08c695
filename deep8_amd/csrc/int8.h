// What the products in 8-bit integers share (quantize.hip, matmul_int8.hip, matmul_int8_wide.hip).
//
// A matrix of codes has its reduction axis along memory: a row of x, and a column of w, is `pitch` bytes, the codes and then zeros up to
// a multiple of 128, so that no kernel has a step of the reduction that is cut short.
#ifndef DEEP8_AMD_INT8_H
#define DEEP8_AMD_INT8_H

#include "common.h"

namespace d8 {
namespace int8 {

typedef int i32x4 __attribute__((ext_vector_type(4)));

enum { STEP = 128 };         // bytes of a row that a step of the reduction takes
enum { MOST_INNER = 131071 };  // 128 * 128 of each fit an int32
constexpr float LEAST_SCALE = 7.888609052210118e-31f;  // 2^-100

inline long pitch_of(int inner) { return ((long)inner + STEP - 1) / STEP * STEP; }

struct Args {
    const signed char *x, *w;
    const float *x_scales, *w_scales;
    void *z;
    int *part;  // partial sums [parts][rows][part_ld] of tiles whose reduction is cut into parts
    long pitch, ldz, part_ld;
    int rows, cols, steps, parts;
    int vec;  // four elements of z that lie side by side can be stored at once (8 bytes in half, 16 in single)
};

// A row's sums times its scale and those of their columns: one rounding of the sum to fp32, one of each product, and the type's.  One scale after the other: the
// scales' product may be too small or too large for fp32 where the result is not (of two scales of 2^-75 it is 0).  The row's first, which leaves nothing too small, a
// scale being 2^-100 at least; the column's first if the row's may leave too much, and then nothing is too large but what the result is.  (A branch for all of a row's:
// 8192 x 4096 x 8192 in 230 us, as without it; the smaller scale of each first 234.)
template <class T, int N, class Sum>
__device__ __forceinline__ void scale_row(const Sum &sum, float row, const float (&cols)[N], T (&out)[N]) {
    constexpr float LARGE = 7.922816251426434e28f;  // 2^96
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = (T)((float)sum[e] * row * cols[e]);
    if (__builtin_expect(__ballot(fabsf(row) > LARGE) != 0, 0)) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (fabsf(row) > LARGE) out[e] = (T)((float)sum[e] * cols[e] * row);
    }
}
template <class T>
__device__ __forceinline__ T scaled(int sum, float row, float col) {
    const int sums[1] = {sum};
    const float cols[1] = {col};
    T out[1];
    scale_row<T, 1>(sums, row, cols, out);
    return out[0];
}

// many rows and columns (matmul_int8_wide.hip)
bool wide_eligible(const Args &a);
template <class T>
int wide_launch(const Args &a, hipStream_t stream);

}  // namespace int8
}  // namespace d8

#endif
