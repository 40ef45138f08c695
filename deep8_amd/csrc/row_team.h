// Rows that a team of 64, 256 or 1024 threads holds in registers: how they are loaded and stored, and which team a row takes (layer_norm.hip,
// quantize.hip).
#ifndef DEEP8_AMD_ROW_TEAM_H
#define DEEP8_AMD_ROW_TEAM_H

#include <type_traits>

#include "common.h"

namespace d8 {
namespace row_team {

// Elements of a row that a team holds (16 a thread of 1024 do not leave the gradient enough registers in single precision).
constexpr int most_held(bool vec, int bytes) { return vec && bytes == 2 ? 16384 : 8192; }

template <class T, int V>
struct Vec {
    typedef T type __attribute__((ext_vector_type(V)));
};
template <class T>
struct Vec<T, 1> {
    typedef T type;
};

// E elements of a row of T in one thread, in pieces of V: piece i is number t + TEAM * i of the row.
template <class T, int V, int TEAM, int E>
struct Held {
    static constexpr int P = E / V;
    typedef typename Vec<T, V>::type vec;
    vec raw[P];
    __device__ __forceinline__ void load(const T *row, int t, int cols) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int c = (t + TEAM * i) * V;
            if (c < cols) raw[i] = *(const vec *)(row + c);
            else raw[i] = vec{};
        }
    }
    __device__ __forceinline__ void ones() {
#pragma unroll
        for (int i = 0; i < P; ++i) raw[i] = vec{} + (T)1;
    }
    __device__ __forceinline__ float at(int e) const {
        if constexpr (V == 1) return (float)raw[e];
        else return (float)raw[e / V][e % V];
    }
    __device__ __forceinline__ void get(float (&v)[E]) const {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = at(e);
    }
    // the same values, but not to the compiler: what it made of them before is not kept
    __device__ __forceinline__ void renew() {
#pragma unroll
        for (int i = 0; i < P; ++i) asm volatile("" : "+v"(raw[i]));
    }
    static __device__ __forceinline__ void store(T *row, int t, int cols, const float (&v)[E]) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int c = (t + TEAM * i) * V;
            if (c >= cols) continue;
            vec w;
            if constexpr (V == 1) {
                w = (T)v[i];
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) w[e] = (T)v[i * V + e];
            }
            *(vec *)(row + c) = w;
        }
    }
};

// The sum of two values over a team.  Several waves: through LDS, a slot that the call before last used (two places in turn: the barrier
// of the call between keeps a wave from writing what another still reads).
template <int TEAM>
__device__ __forceinline__ void team_sum(float &a, float &b, float2 *slots, int &turn) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) a += __shfl_xor(a, d), b += __shfl_xor(b, d);
    if constexpr (TEAM > 64) {
        const int wave = threadIdx.x >> 6;
        float2 *s = slots + turn * 16;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) s[wave] = make_float2(a, b);
        __syncthreads();
        constexpr int N = TEAM / 64;
        s += wave / N * N;
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) a += s[i].x, b += s[i].y;
    }
}

// fn<V, TEAM, E> for the smallest team that holds a row; rows that do not start at multiples of 16 bytes go element by element
template <class T, class F>
void with_team(bool vec, int cols, F &&fn) {
    constexpr int V = 16 / sizeof(T);
#define D8_TEAM(V_, TEAM_, E_) fn(std::integral_constant<int, V_>(), std::integral_constant<int, TEAM_>(), std::integral_constant<int, E_>())
    if (!vec) {
        if (cols <= 1024) D8_TEAM(1, 64, 16);
        else if (cols <= 4096) D8_TEAM(1, 256, 16);
        else D8_TEAM(1, 1024, 8);
    } else if (cols <= 512) D8_TEAM(V, 64, 8);
    else if (cols <= 1024) D8_TEAM(V, 64, 16);
    else if (cols <= 2048) D8_TEAM(V, 256, 8);
    else if (cols <= 4096) D8_TEAM(V, 256, 16);
    else if (cols <= 8192) D8_TEAM(V, 1024, 8);
    else if constexpr (sizeof(T) == 2) D8_TEAM(V, 1024, 16);
#undef D8_TEAM
}


}  // namespace row_team
}  // namespace d8

#endif
