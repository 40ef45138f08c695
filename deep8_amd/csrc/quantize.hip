// Rows of x, and columns of a weight, as 8-bit integers with a scale each.
//
//   scale = max |x| / 127 in fp32, at least 2^-100;  code = x / scale to the nearest whole number, halves to the even one
//
// The code is the rounding of the exact quotient, not of a rounded one, so that it does not depend on how the quotient was come by:
// q = round(x * (1 / scale)) is off only where the product lies within 127 * 2^-23 < 1e-4 of a half, and there the sign of x - (q +- 1/2) scale, which
// one fma has exactly (scale is normal and x a number of 24 bits), says on which side the quotient is.  A row of 16384 halves meets that
// three times.  A row that holds NaN or an infinity gets the scale NaN and codes 0, so its results are NaN.
//
// Rows: bound by memory, x read once (a team of threads holds a row: row_team.h) and a byte written for each element: 8192 x 4096
// halves in 18.5 us alone and 22 before a product that reads them, 5.4 and 4.6 TB/s, where a large copy moves 5.2.  Columns are laid out once
// when a model is loaded: a workgroup goes down 64 columns twice (the second time mostly out of cache) and transposes through LDS: 4096 x 8192 halves in 367 us, bound
// by the chain of its steps on half the compute units (at a copy's rate it would be 20).
#include "int8.h"
#include "row_team.h"

namespace d8 {
namespace {

using namespace row_team;
using int8::LEAST_SCALE;

// |x| as a number that orders like it, NaN above all others
__device__ __forceinline__ unsigned size_of(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ bool finite(unsigned size) { return size < 0x7f800000u; }
__device__ __forceinline__ float scale_of(unsigned size) { return finite(size) ? fmaxf(__uint_as_float(size) / 127.f, LEAST_SCALE) : __uint_as_float(0x7fc00000u); }

// N codes (`back` = 1 / scale; 0 for a row that has none)
template <int N>
__device__ __forceinline__ void codes_of(const float (&x)[N], float scale, float back, int (&code)[N]) {
    float q[N], near = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const float t = x[e] * back;
        q[e] = rintf(t);
        near = fmaxf(near, fabsf(t - q[e]));
    }
    if (near > 0.4999f) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float above = fmaf(-(q[e] + 0.5f), scale, x[e]), below = fmaf(-(q[e] - 0.5f), scale, x[e]);
            const bool odd = (int)q[e] & 1;
            if (above > 0.f || (above == 0.f && odd)) q[e] += 1.f;
            else if (below < 0.f || (below == 0.f && odd)) q[e] -= 1.f;
        }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) code[e] = (int)q[e];
}

template <int N>
__device__ __forceinline__ void store_codes(signed char *to, const int (&code)[N]) {
    if constexpr (N == 1) {
        *to = (signed char)code[0];
    } else {
        unsigned w[N / 4];
#pragma unroll
        for (int i = 0; i < N / 4; ++i)
            w[i] = (code[4 * i] & 255) | (code[4 * i + 1] & 255) << 8 | (code[4 * i + 2] & 255) << 16 | (unsigned)code[4 * i + 3] << 24;
        if constexpr (N == 8) *(uint2 *)to = make_uint2(w[0], w[1]);
        else *(unsigned *)to = w[0];
    }
}

struct QuantizeArgs {
    const void *x;
    signed char *codes;
    float *scales;
    long ldx, pitch;
    int rows, cols;
};

template <int TEAM>
__device__ __forceinline__ unsigned team_max(unsigned m, unsigned *slots, int &turn) {
    m = over_lanes<TEAM>(m, [](unsigned x, unsigned y) { return max(x, y); });
    if constexpr (TEAM > 64) {
        unsigned *s = slots + turn * 16;
        turn ^= 1;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) s[wave] = m;
        __syncthreads();
        constexpr int N = TEAM / 64;
        s += wave / N * N;
#pragma unroll
        for (int i = 0; i < N; ++i) m = max(m, s[i]);
    }
    return m;
}

constexpr int rows_threads(int team) { return team < 256 ? 256 : team; }

template <class T, int V, int TEAM, int E, bool ODD>
__global__ __launch_bounds__(rows_threads(TEAM)) void quantize_rows_kernel(QuantizeArgs a) {
    __shared__ unsigned slots[2 * 16];
    constexpr int TEAMS = rows_threads(TEAM) / TEAM;
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    int turn = 0;
    for (long first = (long)blockIdx.x * TEAMS; first < a.rows; first += (long)gridDim.x * TEAMS) {  // (once, but for more rows than a launch has threads)
        const long row = first + team;
        Held<T, V, TEAM, E, ODD> x;
        if (row < a.rows) x.load((const T *)a.x + row * a.ldx, t, a.cols), x.settle(t, a.cols);
        unsigned size = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) size = max(size, row < a.rows ? size_of(x.at(e)) : 0u);
        size = team_max<TEAM>(size, slots, turn);
        if (row >= a.rows) continue;
        const float scale = scale_of(size), back = finite(size) ? 1.f / scale : 0.f;
        signed char *to = a.codes + row * a.pitch;
#pragma unroll
        for (int i = 0; i < E / V; ++i) {
            const int c = (t + TEAM * i) * V;
            if (c >= a.pitch) continue;
            float v[V];
            int code[V];
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = finite(size) ? x.at(i * V + e) : 0.f;
            codes_of<V>(v, scale, back, code);
            store_codes<V>(to + c, code);
        }
        if (t == 0) a.scales[row] = scale;
    }
}

template <class T>
__global__ __launch_bounds__(1024) void quantize_long_rows_kernel(QuantizeArgs a) {
    __shared__ unsigned slots[2 * 16];
    int turn = 0;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.ldx;
        unsigned size = 0;
        for (int c = threadIdx.x; c < a.cols; c += 1024) size = max(size, size_of((float)x[c]));
        size = team_max<1024>(size, slots, turn);
        const float scale = scale_of(size), back = finite(size) ? 1.f / scale : 0.f;
        for (int c = threadIdx.x; c < a.pitch; c += 1024) {
            const float v[1] = {c < a.cols && finite(size) ? (float)x[c] : 0.f};
            int code[1];
            codes_of<1>(v, scale, back, code);
            a.codes[row * a.pitch + c] = (signed char)code[0];
        }
        if (threadIdx.x == 0) a.scales[row] = scale;
    }
}

// 64 columns of x [rows][cols] (ldx apart) as 64 rows of codes, `pitch` bytes of which `rows` are codes and the rest zeros
template <class T>
__global__ __launch_bounds__(256) void quantize_columns_kernel(QuantizeArgs a) {
    __shared__ unsigned sizes[4][64];
    __shared__ unsigned tile[64][17];  // 64 codes of a column, and a word that keeps columns in different banks
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c0 = blockIdx.x * 64, c = c0 + lane;
    const T *x = (const T *)a.x + (c < a.cols ? c : 0);
    unsigned size = 0;
    if (c < a.cols)
#pragma unroll 8
        for (int r = wave; r < a.rows; r += 4) size = max(size, size_of((float)x[r * a.ldx]));
    sizes[wave][lane] = size;
    __syncthreads();
    size = max(max(sizes[0][lane], sizes[1][lane]), max(sizes[2][lane], sizes[3][lane]));
    const float scale = scale_of(size), back = finite(size) ? 1.f / scale : 0.f;
    if (wave == 0 && c < a.cols) a.scales[c] = scale;
    for (int r0 = 0; r0 < a.pitch; r0 += 64) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // four rows each of 16 of the chunk
            float v[4];
            int code[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = r0 + wave * 16 + i * 4 + e;
                v[e] = r < a.rows && c < a.cols && finite(size) ? (float)x[r * a.ldx] : 0.f;
            }
            codes_of<4>(v, scale, back, code);
            tile[lane][wave * 4 + i] = (code[0] & 255) | (code[1] & 255) << 8 | (code[2] & 255) << 16 | (unsigned)code[3] << 24;
        }
        __syncthreads();
        const int col = threadIdx.x >> 2, part = threadIdx.x & 3;  // 16 bytes a thread
        if (c0 + col < a.cols) {
            const unsigned *w = &tile[col][part * 4];
            *(uint4 *)(a.codes + (c0 + col) * a.pitch + r0 + part * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncthreads();
    }
}

template <class T>
void launch_rows(const QuantizeArgs &a, hipStream_t stream) {
    const int v = 16 / (int)sizeof(T);
    const bool whole = ((size_t)a.x & 15) == 0 && a.cols % v == 0 && a.ldx % v == 0;
    if (a.cols > MOST_HELD) {
        hipLaunchKernelGGL(quantize_long_rows_kernel<T>, dim3(a.rows < 4096 ? a.rows : 4096), dim3(1024), 0, stream, a);
        return;
    }
    with_team<T, false>(whole, a.cols, [&](auto v, auto team, auto e, auto odd) {
        constexpr int V = decltype(v)::value, TEAM = decltype(team)::value, E = decltype(e)::value, THREADS = rows_threads(TEAM);
        const long want = ((long)a.rows * TEAM + THREADS - 1) / THREADS, most = (1L << 31) / THREADS, groups = want < most ? want : most;
        hipLaunchKernelGGL((quantize_rows_kernel<T, V, TEAM, E, decltype(odd)::value>), dim3((unsigned)groups), dim3(THREADS), 0, stream, a);
    });
}

int check(const QuantizeArgs &a, int dtype, int inner, const char *name) {
    if (dtype != D8_FLOAT16 && dtype != D8_FLOAT32) return fail(D8_ERR_DTYPE, "%s: type %d is not support", name, dtype);
    D8_REQUIRE(a.rows >= 0 && a.cols >= 0 && inner >= 1, "%s: a matrix of %d x %d", name, a.rows, a.cols);
    D8_REQUIRE(inner <= int8::MOST_INNER, "%s: a sum has at most %d terms, not %d", name, (int)int8::MOST_INNER, inner);
    if (!a.rows || !a.cols) return 0;
    D8_REQUIRE(a.x && a.codes && a.scales, "%s: null tensor", name);
    D8_REQUIRE(a.ldx >= a.cols, "%s: rows of %d elements do not fit their leading dimension", name, a.cols);
    D8_REQUIRE(((size_t)a.codes & 15) == 0, "%s: codes must be 16-byte aligned", name);
    return 0;
}

}  // namespace
}  // namespace d8

using namespace d8;

extern "C" int d8_int8_pitch(int inner) { return inner < 1 || inner > int8::MOST_INNER ? 0 : (int)int8::pitch_of(inner); }

extern "C" int d8_quantize_rows(int dtype, const void *x, long ldx, int rows, int cols, signed char *codes, float *scales, void *stream) {
    QuantizeArgs a = {x, codes, scales, ldx, int8::pitch_of(cols), rows, cols};
    if (int rc = check(a, dtype, cols, "quantize_rows")) return rc;
    if (!rows) return 0;
    if (dtype == D8_FLOAT16) launch_rows<f16>(a, as_stream(stream));
    else launch_rows<float>(a, as_stream(stream));
    D8_LAUNCH_CHECK();
    return 0;
}

extern "C" int d8_quantize_columns(int dtype, const void *w, long ldw, int rows, int cols, signed char *codes, float *scales, void *stream) {
    QuantizeArgs a = {w, codes, scales, ldw, int8::pitch_of(rows), rows, cols};
    if (int rc = check(a, dtype, rows, "quantize_columns")) return rc;
    if (!cols) return 0;
    D8_REQUIRE(cols <= 1 << 29, "quantize_columns: %d columns are too many for a launch", cols);
    const dim3 grid(ceil_div(cols, 64));
    if (dtype == D8_FLOAT16) hipLaunchKernelGGL(quantize_columns_kernel<f16>, grid, dim3(256), 0, as_stream(stream), a);
    else hipLaunchKernelGGL(quantize_columns_kernel<float>, grid, dim3(256), 0, as_stream(stream), a);
    D8_LAUNCH_CHECK();
    return 0;
}
