// Arguments of the gated product's kernels and what they share (gated.hip, gated_wide.hip).
#ifndef DEEP8_AMD_GATED_H
#define DEEP8_AMD_GATED_H

#include "attention.h"

namespace d8 {
namespace gated {

struct Args {
    const void *x, *w;
    void *pre, *h;
    const void *dh;
    void *dpre;
    int rows, inner, cols, act;
    // x and w as they lie: row strides, where the factor's columns begin, elements of a row (a half row of w) with the zeros behind it
    long ldx, ldw;
    int up, inner_there, cols_there;
    int chunk, parts;  // K of a workgroup, and how many it is cut into: few rows, or the tiles from number `whole` on
    int whole;
    float *part;       // ... their sums: few rows [parts][rows][2 cols], else [tile][part][gate, factor][rows of a tile][its columns]
    int vec;           // the way back: rows of pre, dh and dpre can be moved in 16-byte pieces
};

// Half: the hardware's reciprocal and power of two, good to 1 ulp of fp32.
template <class T>
__device__ __forceinline__ float sigmoid(float a) {
    if (sizeof(T) == 2) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * a));
    return 1.f / (1.f + expf(-a));
}
// The normal distribution's integral up to a, (1 + erf(a / sqrt 2)) / 2, from the complement: 1 + erf cancels for negative a (a formula for erf that is
// good to 1.5e-7 left 7e-2 of it at a = -5).  Half: erfc(y) = exp(-y^2) t Q(t) with t = 1 / (1 + 3 y / 8), Q of degree 6 fitted to the smallest
// largest relative error for y up to 9, 6.4e-7 (1e-6 with the roundings of fp32), without a branch.
template <class T>
__device__ __forceinline__ float normal_integral(float a) {
    if (sizeof(T) == 4) return 0.5f * erfcf(-0.70710678f * a);
    const float t = __builtin_amdgcn_rcpf(1.f + 0.26516504f * fabsf(a));
    const float q = (((((-0.135095671f * t + 0.38793692f) * t - 0.129595846f) * t + 0.283060342f) * t + 0.166665107f) * t + 0.215689063f) * t + 0.211339459f;
    const float tail = 0.5f * t * q * __builtin_amdgcn_exp2f(-0.72134752f * a * a);
    return a < 0.f ? tail : 1.f - tail;
}

template <class T>
__device__ __forceinline__ float activation(float a, int act) {
    switch (act) {
        case D8_GATE_SILU: return a * sigmoid<T>(a);
        case D8_GATE_GELU: return a * normal_integral<T>(a);
        case D8_GATE_RELU: return a > 0.f ? a : 0.f;
        default: return sigmoid<T>(a);
    }
}

// element (m, n) of both projections into h and, if it is kept, pre
template <class T>
__device__ __forceinline__ void store(const Args &a, int m, int n, float g, float u) {
    ((T *)a.h)[(long)m * a.cols + n] = (T)(activation<T>(g, a.act) * u);
    if (a.pre) {
        T *p = (T *)a.pre + (long)m * 2 * a.cols + n;
        p[0] = (T)g, p[a.cols] = (T)u;
    }
}

// many rows and columns in half (gated_wide.hip)
bool wide_eligible(const Args &a);
int wide_launch(const Args &a, hipStream_t stream);

}  // namespace gated
}  // namespace d8

#endif
