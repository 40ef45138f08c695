// Rows that a team of 16 to 1024 threads holds in registers: how they are loaded and stored, and which team a row takes (layer_norm.hip, quantize.hip).
#ifndef DEEP8_AMD_ROW_TEAM_H
#define DEEP8_AMD_ROW_TEAM_H

#include <type_traits>

#include "lanes.h"

namespace d8 {
namespace row_team {

// Elements of a row that a team holds at most, 16 a thread of 1024.
enum { MOST_HELD = 16384 };

// E elements of a row of T in one thread, in pieces of V: piece i is number t + TEAM * i of the row.  ODD: the row, of V elements at least, starts
// anywhere, and may end within a piece, for which the row's last V are read; settle() then moves them down.  (Norm of 16384 rows of 1001 in half: 15 us, 32
// element by element.  A load that branches where the row ends keeps the next row's from running ahead: gradients of 4096 rows of 4095 took 51 us
// so, and 31 with this.)
template <class T, int V, int TEAM, int E, bool ODD>
struct Held {
    static constexpr int P = E / V;
    typedef T vec __attribute__((ext_vector_type(V)));
    typedef T odd_vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    typedef std::conditional_t<ODD, odd_vec, vec> there;
    // Whether pieces beyond the row read its last V too and are cleared when used, in place of a load that may not be made: fewer registers (gradients of
    // 1024 rows of 16384 in single: 61 us, 107 without), but 2 % more time in single where there are enough.
    static constexpr bool CLAMPED = ODD || TEAM == 1024;
    vec raw[P];
    // whether element e of the thread's is one of the row's
    static __device__ __forceinline__ bool has(int e, int t, int cols) { return (t + TEAM * (e / V)) * V + (ODD ? e % V : 0) < cols; }
    __device__ __forceinline__ void load(const T *row, int t, int cols) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int c = (t + TEAM * i) * V;
            if constexpr (CLAMPED) raw[i] = *(const there *)(row + min(c, cols - V));
            else if (c < cols) raw[i] = *(const vec *)(row + c);
            else raw[i] = vec{};
        }
    }
    // after a load, before its elements are used: those beyond the row are 0
    __device__ __forceinline__ void settle(int t, int cols) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int beyond = (t + TEAM * i) * V - (cols - V);
            if (!CLAMPED || beyond <= 0) continue;
            if constexpr (ODD) {
                typedef unsigned _BitInt(8 * V * sizeof(T)) bits;
                raw[i] = beyond < V ? __builtin_bit_cast(vec, (bits)(__builtin_bit_cast(bits, raw[i]) >> (8 * (int)sizeof(T) * beyond))) : vec{};
            } else {
                raw[i] = vec{};
            }
        }
    }
    __device__ __forceinline__ void ones() {
#pragma unroll
        for (int i = 0; i < P; ++i) raw[i] = vec{} + (T)1;
    }
    __device__ __forceinline__ float at(int e) const { return (float)raw[e / V][e % V]; }
    __device__ __forceinline__ void get(float (&v)[E]) const {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = at(e);
    }
    // the same values, but not to the compiler: what it made of them before is not kept
    __device__ __forceinline__ void renew() {
#pragma unroll
        for (int i = 0; i < P; ++i)
            if constexpr (V > 1) asm volatile("" : "+v"(raw[i]));
    }
    static __device__ __forceinline__ void store(T *row, int t, int cols, const float (&v)[E]) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int c = (t + TEAM * i) * V;
            vec w;
#pragma unroll
            for (int e = 0; e < V; ++e) w[e] = (T)v[i * V + e];
            if (ODD ? c + V <= cols : c < cols) *(there *)(row + c) = w;
            else if (ODD && c < cols)
#pragma unroll
                for (int e = 0; e < V - 1; ++e)
                    if (c + e < cols) row[c + e] = w[e];
        }
    }
};

// The sum of two values over a team.  Several waves: through LDS, a slot that the call before last used (two places in turn: the barrier
// of the call between keeps a wave from writing what another still reads).
template <int TEAM>
__device__ __forceinline__ void team_sum(float &a, float &b, float2 *slots, int &turn) {
    const auto add = [](float x, float y) { return x + y; };
    a = over_lanes<TEAM>(a, add), b = over_lanes<TEAM>(b, add);
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

// fn(V, TEAM, E, ODD) for the smallest team that holds a row; whole: every row is whole pieces of 16 bytes.  Short rows share a wave (65536 of 96 in half:
// norm 9 us, 21 with a wave each); 16 elements a thread of 512 are better than 8 of 1024, of whose workgroups a compute unit has half as many to change
// between (8192 rows of 5120: 40 us and 78).
template <class T, bool GRAD, class F>
void with_team(bool whole, int cols, F &&fn) {
    constexpr int V = 16 / sizeof(T);
    if (cols < V) return fn(std::integral_constant<int, 1>(), std::integral_constant<int, 16>(), std::integral_constant<int, 8>(), std::true_type());
    auto in = [&](auto odd) {
#define D8_TEAM(TEAM_, E_) fn(std::integral_constant<int, V>(), std::integral_constant<int, TEAM_>(), std::integral_constant<int, E_>(), odd)
        if (cols <= 128) D8_TEAM(16, 8);
        else if (cols <= 256) D8_TEAM(32, 8);
        else if (cols <= 512) D8_TEAM(64, 8);
        else if (cols <= 1024) D8_TEAM(64, 16);
        else if (cols <= 2048) D8_TEAM(256, 8);
        else if (cols <= 4096) D8_TEAM(256, 16);
        else if (cols <= 8192) {
            if constexpr (GRAD && sizeof(T) == 4) D8_TEAM(1024, 8);
            else D8_TEAM(512, 16);
        }
        else D8_TEAM(1024, 16);
#undef D8_TEAM
    };
    if (whole) in(std::false_type());
    else in(std::true_type());
}

}  // namespace row_team
}  // namespace d8

#endif
