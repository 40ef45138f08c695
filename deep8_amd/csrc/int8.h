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

// a row's sum times both scales: one rounding of the sum to fp32, one of the scales' product, one of the result, and the type's
template <class T>
__device__ __forceinline__ T scaled(int sum, float x_scale, float w_scale) { return (T)((float)sum * (x_scale * w_scale)); }

// many rows and columns (matmul_int8_wide.hip)
bool wide_eligible(const Args &a);
template <class T>
int wide_launch(const Args &a, hipStream_t stream);

}  // namespace int8
}  // namespace d8

#endif
