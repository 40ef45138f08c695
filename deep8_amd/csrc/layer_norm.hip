// Norm of whole rows, and the way back.
//
//   m = mean(x),  r = 1 / sqrt(mean((x - m)^2) + epsilon),  u = (x - m) r,  y = u w + b
//   back: g = dy,  dx = r (w g - mean(w g) - u mean(w g u)),  dw = sum over rows of g u,  db = sum over rows of g
//
// Bound by memory: x is read and y written once (back: x and dy read, dx written); a row stays in the registers of its team of 16 to 1024 threads
// (row_team.h) between the sums and the result.  A thread has up to 16 elements of a row: more would leave too few waves to keep the
// loads coming.  The spread is taken about the mean that was found, not from the sum of squares, which would cancel in rows whose mean is
// far from zero, and what that mean is off by (its sum is rounded) is taken out with the same pass: sum (x - m) is it.
//
// The way back keeps the columns' sums of dw and db in registers while a workgroup goes down its rows (the next row's loads are on their
// way meanwhile), adds its teams' through LDS, and leaves one row of them in scratch; a second launch adds those in a fixed order.  Two
// workgroups of 512 threads a compute unit, so that one loads while the other adds; more would write and read more such rows.
//
// Half: 16384 x 4096 forward 53 us, 5.05 TB/s, where a large copy moves 5.2; 8192 x 4096 back 47 us (43 and 4 for the sums), 4.3 TB/s.  Single, 8192 x 4096
// forward 50 us, back 81 us: 5.4 and 5.0 TB/s.
//
// Sums are fp32; results are rounded once.
#include "row_team.h"

namespace d8 {
namespace {

using namespace row_team;

struct NormArgs {
    const void *x, *dy, *weight, *bias;
    void *out;  // y, or dx
    void *dweight, *dbias;
    float *partial;  // gradient: [groups][dw, db][cols]
    long ldx, lddy, ldout;
    int rows, cols, groups, overwrite;
    float epsilon;
};

// (E values of which those beyond the row are 0) centred in place, 0 there again; the reciprocal of the spread
template <class H, int TEAM, int E>
__device__ __forceinline__ float centre(float (&v)[E], int t, int cols, float epsilon, float2 *slots, int &turn) {
    const float n = 1.f / cols;
    float sum = 0.f, rest = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) sum += v[e];
    team_sum<TEAM>(sum, rest, slots, turn);
    const float mean = sum * n;
    float off = 0.f, squares = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        v[e] = H::has(e, t, cols) ? v[e] - mean : 0.f;
        off += v[e], squares += v[e] * v[e];
    }
    team_sum<TEAM>(off, squares, slots, turn);
    off *= n;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = H::has(e, t, cols) ? v[e] - off : 0.f;
    return 1.f / sqrtf(fmaxf(squares * n - off * off, 0.f) + epsilon);
}

constexpr int forward_threads(int team) { return team < 256 ? 256 : team; }

template <class T, int V, int TEAM, int E, bool ODD>
__global__ __launch_bounds__(forward_threads(TEAM)) void layer_norm_kernel(NormArgs a) {
    __shared__ float2 slots[2 * 16];
    constexpr int TEAMS = forward_threads(TEAM) / TEAM;
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    typedef Held<T, V, TEAM, E, ODD> H;
    float w[E], b[E];
    {
        H h;
        if (a.weight) h.load((const T *)a.weight, t, a.cols), h.settle(t, a.cols), h.get(w);
        else for (int e = 0; e < E; ++e) w[e] = 1.f;
        if (a.bias) h.load((const T *)a.bias, t, a.cols), h.settle(t, a.cols), h.get(b);
        else for (int e = 0; e < E; ++e) b[e] = 0.f;
    }
    int turn = 0;
    H x;
    long row = (long)blockIdx.x * TEAMS + team;
    const long step = (long)gridDim.x * TEAMS;
    if (row < a.rows) x.load((const T *)a.x + row * a.ldx, t, a.cols);
    for (long first = (long)blockIdx.x * TEAMS; first < a.rows; first += step, row += step) {  // (all teams take part in the barriers)
        float v[E];
        x.settle(t, a.cols), x.get(v);
        if (row + step < a.rows) x.load((const T *)a.x + (row + step) * a.ldx, t, a.cols);
        const float r = centre<H, TEAM, E>(v, t, a.cols, a.epsilon, slots, turn);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = v[e] * r * w[e] + b[e];
        if (row < a.rows) H::store((T *)a.out + row * a.ldout, t, a.cols, v);
    }
}

// Threads of a gradient workgroup, whole teams.
constexpr int grad_threads(int team) { return team == 1024 ? 1024 : 512; }
// Waves a SIMD: four where what a thread keeps (its columns' sums, weights, this row's and the next one's elements) fits in the 128 registers that leaves it.
constexpr int grad_waves(int elements, int bytes, bool odd) { return elements == 8 || (bytes == 2 && !odd) ? 4 : 1; }

template <class T, int V, int TEAM, int E, bool ODD>
__global__ __launch_bounds__(grad_threads(TEAM), grad_waves(E, sizeof(T), ODD)) void layer_norm_grad_kernel(NormArgs a) {
    constexpr int THREADS = grad_threads(TEAM), TEAMS = THREADS / TEAM;
    constexpr bool AHEAD = TEAM < 1024 || E == 8;  // the next row's loads on their way
    __shared__ float2 slots[2 * 16];
    __shared__ float sums[TEAMS > 1 ? THREADS * E : 1];
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    typedef Held<T, V, TEAM, E, ODD> H;
    H w, x, dy;
    if (a.weight) w.load((const T *)a.weight, t, a.cols), w.settle(t, a.cols);
    else w.ones();
    float dw[E], db[E];
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.f;
    int turn = 0;
    const float n = 1.f / a.cols;
    long row = (long)blockIdx.x * TEAMS + team;
    const long step = (long)gridDim.x * TEAMS;
    auto fetch = [&](long at) {
        if (at < a.rows) x.load((const T *)a.x + at * a.ldx, t, a.cols), dy.load((const T *)a.dy + at * a.lddy, t, a.cols);
    };
    fetch(row);
    for (long first = (long)blockIdx.x * TEAMS; first < a.rows; first += step, row += step) {  // (all teams take part in the barriers)
        float u[E], s0 = 0.f, s1 = 0.f;
        x.settle(t, a.cols), dy.settle(t, a.cols);
        H g = dy;
        x.get(u);
        if (AHEAD) fetch(row + step);
        const float r = centre<H, TEAM, E>(u, t, a.cols, a.epsilon, slots, turn);
        const bool mine = TEAM < 64 ? row < a.rows : __builtin_amdgcn_readfirstlane(row < a.rows);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float ge = g.at(e), wg = w.at(e) * ge;
            u[e] *= r;
            s0 += wg, s1 += wg * u[e];
            if (e % V == V - 1) asm volatile("" : "+v"(s0), "+v"(s1));  // piece by piece: one at a time is held in fp32
        }
        // (w and dy as they were loaded, converted again for each use: kept as fp32 they would take the registers of the next row)
        g.renew(), w.renew();
        if (mine) {
#pragma unroll
            for (int e = 0; e < E; ++e) dw[e] += g.at(e) * u[e], db[e] += g.at(e);
            g.renew();
        }
        team_sum<TEAM>(s0, s1, slots, turn);
        s0 *= n, s1 *= n;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            u[e] = r * (w.at(e) * g.at(e) - s0 - u[e] * s1);
            if (e % V == V - 1) asm volatile("" : "+v"(s0), "+v"(s1));
        }
        if (mine && a.out) {
            T *to = (T *)a.out + row * a.ldout;
            if (!(a.overwrite & 1)) {
                g.load(to, t, a.cols), g.settle(t, a.cols);
#pragma unroll
                for (int e = 0; e < E; ++e) u[e] += g.at(e);
            }
            H::store(to, t, a.cols, u);
        }
        if (!AHEAD) fetch(row + step);
    }
    if (!a.partial) return;  // uniform over the workgroup
    float *to = a.partial + (long)blockIdx.x * 2 * a.cols;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if constexpr (TEAMS == 1) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int c = (t + TEAM * (e / V)) * V + e % V;
                if (H::has(e, t, a.cols)) to[(long)k * a.cols + c] = k ? db[e] : dw[e];
            }
        } else {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; ++e) sums[team * (TEAM * E) + (t + TEAM * (e / V)) * V + e % V] = k ? db[e] : dw[e];
            __syncthreads();
            for (int c = threadIdx.x; c < a.cols; c += THREADS) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < TEAMS; ++i) s += sums[i * (TEAM * E) + c];
                to[(long)k * a.cols + c] = s;
            }
        }
    }
}

// ---- rows that no team holds: a workgroup a row, read as often as it takes ------------------------------------------
template <class T>
__device__ __forceinline__ void long_row(const T *x, int cols, float epsilon, float2 *slots, int &turn, float &mean, float &off, float &r) {
    float sum = 0.f, rest = 0.f;
    for (int c = threadIdx.x; c < cols; c += 1024) sum += (float)x[c];
    team_sum<1024>(sum, rest, slots, turn);
    mean = sum / cols;
    float squares = 0.f;
    off = 0.f;
    for (int c = threadIdx.x; c < cols; c += 1024) {
        const float v = (float)x[c] - mean;
        off += v, squares += v * v;
    }
    team_sum<1024>(off, squares, slots, turn);
    off /= cols;  // (kept beside the mean, whose last bit may be as large)
    r = 1.f / sqrtf(fmaxf(squares / cols - off * off, 0.f) + epsilon);
}

template <class T>
__global__ __launch_bounds__(1024) void layer_norm_long_kernel(NormArgs a) {
    __shared__ float2 slots[2 * 16];
    int turn = 0;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.ldx;
        T *y = (T *)a.out + row * a.ldout;
        float mean, off, r;
        long_row<T>(x, a.cols, a.epsilon, slots, turn, mean, off, r);
        for (int c = threadIdx.x; c < a.cols; c += 1024) {
            const float w = a.weight ? (float)((const T *)a.weight)[c] : 1.f, b = a.bias ? (float)((const T *)a.bias)[c] : 0.f;
            y[c] = (T)(((float)x[c] - mean - off) * r * w + b);
        }
    }
}

template <class T>
__global__ __launch_bounds__(1024) void layer_norm_grad_long_kernel(NormArgs a) {
    __shared__ float2 slots[2 * 16];
    int turn = 0;
    float *to = a.partial ? a.partial + (long)blockIdx.x * 2 * a.cols : nullptr;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.ldx, *dy = (const T *)a.dy + row * a.lddy, *w = (const T *)a.weight;
        T *dx = a.out ? (T *)a.out + row * a.ldout : nullptr;
        float mean, off, r, s0 = 0.f, s1 = 0.f;
        long_row<T>(x, a.cols, a.epsilon, slots, turn, mean, off, r);
        for (int c = threadIdx.x; c < a.cols; c += 1024) {
            const float u = ((float)x[c] - mean - off) * r, g = (float)dy[c], wg = w ? (float)w[c] * g : g;
            s0 += wg, s1 += wg * u;
            if (to) {  // (a column's sums belong to one thread, whichever row it is at)
                const bool fresh = row == blockIdx.x;
                to[c] = (fresh ? 0.f : to[c]) + g * u;
                to[a.cols + c] = (fresh ? 0.f : to[a.cols + c]) + g;
            }
        }
        team_sum<1024>(s0, s1, slots, turn);
        s0 /= a.cols, s1 /= a.cols;
        if (!dx) continue;
        for (int c = threadIdx.x; c < a.cols; c += 1024) {
            const float u = ((float)x[c] - mean - off) * r, g = (float)dy[c], wg = w ? (float)w[c] * g : g;
            const float d = r * (wg - s0 - u * s1);
            dx[c] = (T)(a.overwrite & 1 ? d : d + (float)dx[c]);
        }
    }
}

// C of the columns of dw (blockIdx.y 0) or db: C threads side by side add every 1024 / C-th workgroup's sums, then 1024 / C threads a column's, in a fixed order.
// 32 columns where 64 would leave compute units without any (back at 32768 x 256: 16 us for 17), 64 where there are enough (2048 x 11111: 74 for 75.5).
template <class T, int C>
__global__ __launch_bounds__(1024) void layer_norm_sums_kernel(NormArgs a) {
    constexpr int G = 1024 / C;
    __shared__ float sums[G][C + 1];
    const int c = blockIdx.x * C + threadIdx.x % C, k = blockIdx.y;
    T *to = (T *)(k ? a.dbias : a.dweight);
    if (!to) return;
    float s = 0.f;
    if (c < a.cols) {
        const float *from = a.partial + (long)k * a.cols + c;
#pragma unroll 8
        for (int g = threadIdx.x / C; g < a.groups; g += G) s += from[(long)g * 2 * a.cols];
    }
    sums[threadIdx.x / C][threadIdx.x % C] = s;
    __syncthreads();
    s = over_lanes<G>(sums[threadIdx.x % G][threadIdx.x / G], [](float x, float y) { return x + y; });
    const int own = blockIdx.x * C + threadIdx.x / G;
    if (threadIdx.x % G == 0 && own < a.cols) to[own] = (T)(a.overwrite & 2 ? s : s + (float)to[own]);
}

// ---- host -----------------------------------------------------------------------------------------------------------
bool in_pieces(const NormArgs &a, int dtype) {
    const int v = 16 / (int)dtype_bytes(dtype);
    const size_t all = (size_t)a.x | (size_t)a.dy | (size_t)a.weight | (size_t)a.bias | (size_t)a.out;
    return (all & 15) == 0 && a.cols % v == 0 && a.ldx % v == 0 && a.lddy % v == 0 && a.ldout % v == 0;
}

int check(const NormArgs &a, int dtype, bool grad) {
    const char *name = grad ? "layer_norm_grad" : "layer_norm";
    if (dtype != D8_FLOAT16 && dtype != D8_FLOAT32) return fail(D8_ERR_DTYPE, "%s: type %d is not support", name, dtype);
    D8_REQUIRE(a.rows >= 0 && a.cols >= 1 && a.cols < (1 << 30), "%s: %d rows of %d", name, a.rows, a.cols);
    D8_REQUIRE(a.epsilon >= 0.f, "%s: epsilon %g", name, (double)a.epsilon);
    if (!a.rows) return 0;
    D8_REQUIRE(a.x && (grad ? a.dy != nullptr : a.out != nullptr), "%s: null tensor", name);
    D8_REQUIRE(a.ldx >= a.cols && (!a.out || a.ldout >= a.cols) && (!grad || a.lddy >= a.cols), "%s: rows of %d elements do not fit their leading dimension", name, a.cols);
    D8_REQUIRE(a.rows == 1 || ((a.out != a.x || a.ldout == a.ldx) && (!grad || a.out != a.dy || a.ldout == a.lddy)), "%s: rows over an input lie where its rows do", name);
    return 0;
}

template <class T>
void launch_forward(const NormArgs &a, bool whole, hipStream_t stream) {
    if (a.cols > MOST_HELD) {
        hipLaunchKernelGGL(layer_norm_long_kernel<T>, dim3(a.rows < 4096 ? a.rows : 4096), dim3(1024), 0, stream, a);
        return;
    }
    with_team<T, false>(whole, a.cols, [&](auto v, auto team, auto e, auto odd) {
        constexpr int V = decltype(v)::value, TEAM = decltype(team)::value, E = decltype(e)::value, THREADS = forward_threads(TEAM);
        // four rounds of the chip's waves at most: a team that goes down several rows reads weight and bias once
        const long want = ((long)a.rows * TEAM + THREADS - 1) / THREADS, most = 2048L / THREADS * cu_count();
        hipLaunchKernelGGL((layer_norm_kernel<T, V, TEAM, E, decltype(odd)::value>), dim3((unsigned)(want < most ? want : most)), dim3(THREADS), 0, stream, a);
    });
}

template <class T>
void launch_grad(NormArgs &a, bool whole, hipStream_t stream) {
    if (a.cols > MOST_HELD) {
        a.groups = a.rows < cu_count() ? a.rows : cu_count();
        hipLaunchKernelGGL(layer_norm_grad_long_kernel<T>, dim3(a.groups), dim3(1024), 0, stream, a);
        return;
    }
    with_team<T, true>(whole, a.cols, [&](auto v, auto team, auto e, auto odd) {
        constexpr int V = decltype(v)::value, TEAM = decltype(team)::value, E = decltype(e)::value, THREADS = grad_threads(TEAM),
                      AT_ONCE = grad_waves(E, sizeof(T), decltype(odd)::value) * 256 / THREADS > 1 ? 2 : 1;
        const long want = ((long)a.rows * TEAM + THREADS - 1) / THREADS, most = (long)AT_ONCE * cu_count();
        a.groups = (int)(want < most ? want : most);
        hipLaunchKernelGGL((layer_norm_grad_kernel<T, V, TEAM, E, decltype(odd)::value>), dim3((unsigned)a.groups), dim3(THREADS), 0, stream, a);
    });
}

enum { MOST_SUMS = 1 << 27 };  // columns whose sums a launch has threads for

template <class T>
void launch_sums(const NormArgs &a, hipStream_t stream) {
    if (a.cols < 16 * cu_count()) hipLaunchKernelGGL((layer_norm_sums_kernel<T, 32>), dim3(ceil_div(a.cols, 32), 2), dim3(1024), 0, stream, a);
    else hipLaunchKernelGGL((layer_norm_sums_kernel<T, 64>), dim3(ceil_div(a.cols, 64), 2), dim3(1024), 0, stream, a);
}

}  // namespace
}  // namespace d8

using namespace d8;

extern "C" int d8_layer_norm(int dtype, const void *x, long ldx, const void *weight, const void *bias, void *y, long ldy, int rows, int cols, float epsilon,
                             void *stream) {
    NormArgs a;
    memset(&a, 0, sizeof(a));
    a.x = x, a.ldx = ldx, a.weight = weight, a.bias = bias, a.out = y, a.ldout = ldy, a.rows = rows, a.cols = cols, a.epsilon = epsilon;
    if (int rc = check(a, dtype, false)) return rc;
    if (!rows) return 0;
    if (dtype == D8_FLOAT16) launch_forward<f16>(a, in_pieces(a, dtype), as_stream(stream));
    else launch_forward<float>(a, in_pieces(a, dtype), as_stream(stream));
    D8_LAUNCH_CHECK();
    return 0;
}

extern "C" size_t d8_layer_norm_grad_scratch_bytes(int dtype, int rows, int cols) {
    if ((dtype != D8_FLOAT16 && dtype != D8_FLOAT32) || rows < 0 || cols < 1 || cols > MOST_SUMS) return 0;
    const int groups = rows < 2 * cu_count() ? rows : 2 * cu_count();
    return sizeof(float) * 2 * (size_t)(groups ? groups : 1) * cols;
}

extern "C" int d8_layer_norm_grad(int dtype, const void *x, long ldx, const void *weight, const void *dy, long lddy, void *dx, long lddx, void *dweight,
                                  void *dbias, int rows, int cols, float epsilon, int overwrite, void *scratch, size_t scratch_bytes, void *stream) {
    NormArgs a;
    memset(&a, 0, sizeof(a));
    a.x = x, a.ldx = ldx, a.weight = weight, a.dy = dy, a.lddy = lddy, a.out = dx, a.ldout = dx ? lddx : 0, a.dweight = dweight, a.dbias = dbias;
    a.rows = rows, a.cols = cols, a.epsilon = epsilon, a.overwrite = overwrite;
    if (int rc = check(a, dtype, true)) return rc;
    const bool sums = dweight || dbias;
    if (sums) {
        D8_REQUIRE(cols <= MOST_SUMS, "layer_norm_grad: weights' gradients have at most %d columns, not %d", (int)MOST_SUMS, cols);
        const size_t need = d8_layer_norm_grad_scratch_bytes(dtype, rows, cols);
        D8_REQUIRE(scratch && scratch_bytes >= need && ((size_t)scratch & 15) == 0, "layer_norm_grad: 16-byte aligned scratch of %zu bytes is needed, not %zu", need, scratch_bytes);
        a.partial = (float *)scratch;
    }
    if (rows && (sums || dx)) {
        if (dtype == D8_FLOAT16) launch_grad<f16>(a, in_pieces(a, dtype), as_stream(stream));
        else launch_grad<float>(a, in_pieces(a, dtype), as_stream(stream));
        D8_LAUNCH_CHECK();
    }
    if (sums) {  // (without a row the sums are zero)
        if (dtype == D8_FLOAT16) launch_sums<f16>(a, as_stream(stream));
        else launch_sums<float>(a, as_stream(stream));
        D8_LAUNCH_CHECK();
    }
    return 0;
}
