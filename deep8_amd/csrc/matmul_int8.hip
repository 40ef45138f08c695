// z = (x w) times a scale of each row of x and one of each column of w, x and w in 8-bit integers: sums in int32 are exact, in whatever order
// they are added, so a reduction can be cut into parts freely.
//
// Three ways, by size:
//   few rows (64 at most)      bound by memory, the weight: no LDS on its way, a wave reads 16 codes a lane straight into the operand
//                              of v_mfma_i32_16x16x64_i8 (16 or 32 columns of w as left operand, all rows of x as right one); eight waves
//                              share out the steps of the reduction and join through LDS: 4 x 4096 x 8192 in 8.5 us, 4.0 TB/s
//   many rows and columns      matmul_int8_wide.hip
//   between                    tiles of 64 x 64 through LDS, cut along the reduction where they leave compute units idle and it is long
// Where w is the left operand, a lane ends up with four columns of a row side by side.
#include <type_traits>

#include "int8.h"

namespace d8 {
namespace int8 {
namespace {

__device__ __forceinline__ void mma(i32x4 &acc, const i32x4 &a, const i32x4 &b) { acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, acc, 0, 0, 0); }

// four sums of row m, columns n .. n + 3: scaled by that row's scale and those columns' into z, or as they are into part number `part`
template <class T>
__device__ __forceinline__ void put(const Args &a, int part, int m, int n, const i32x4 &sum, float row, const float (&cols)[4]) {
    if (m >= a.rows || n >= a.cols) return;
    if (a.parts > 1) {  // (rows of parts are whole pieces)
        *(i32x4 *)(a.part + ((long)part * a.rows + m) * a.part_ld + n) = sum;
        return;
    }
    T *z = (T *)a.z + (long)m * a.ldz + n, out[4];
    scale_row<T, 4>(sum, row, cols, out);
    if (a.vec && n + 4 <= a.cols) {
        typedef T quad __attribute__((ext_vector_type(4)));
        *(quad *)z = *(const quad *)out;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < a.cols) z[e] = out[e];
    }
}
template <class T>
__device__ __forceinline__ void put(const Args &a, int part, int m, int n, const i32x4 &sum) {
    float cols[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) cols[e] = a.w_scales[min(n + e, a.cols - 1)];
    put<T>(a, part, m, n, sum, a.x_scales[min(m, a.rows - 1)], cols);
}

// the parts' sums of four columns of a row
template <class T>
__global__ __launch_bounds__(256) void int8_join_kernel(Args a) {
    const long quads = (a.cols + 3) / 4, i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= quads * a.rows) return;
    const int m = (int)(i / quads), n = (int)(i - m * quads) * 4;
    i32x4 sum = {0, 0, 0, 0};
    for (int p = 0; p < a.parts; ++p) sum += *(const i32x4 *)(a.part + ((long)p * a.rows + m) * a.part_ld + n);
    a.parts = 1;
    put<T>(a, 0, m, n, sum);
}

// ---- few rows -------------------------------------------------------------------------------------------------------
enum { ROWS_WAVES = 8 };

// RT tiles of 16 rows, CT of 16 columns
template <class T, int RT, int CT>
__global__ __launch_bounds__(ROWS_WAVES * 64) void int8_rows_kernel(Args a) {
    __shared__ i32x4 sums[ROWS_WAVES][CT * RT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = blockIdx.y, n0 = blockIdx.x * 16 * CT;
    const int first = (int)((long)a.steps * part / a.parts), end = (int)((long)a.steps * (part + 1) / a.parts);
    // a lane's 16 bytes of a step of 128: columns (rows) lane % 16 of each tile, bytes 16 (lane / 16) .. of both halves.  Beyond the last
    // column or row the last one is read again; what comes of it is not stored.
    const int r = lane & 15, at = (lane >> 4) * 16;
    const signed char *w[CT], *x[RT];
#pragma unroll
    for (int i = 0; i < CT; ++i) w[i] = a.w + (long)min(n0 + 16 * i + r, a.cols - 1) * a.pitch + at;
#pragma unroll
    for (int j = 0; j < RT; ++j) x[j] = a.x + (long)min(16 * j + r, a.rows - 1) * a.pitch + at;
    i32x4 acc[CT][RT] = {};
    // scales of what the wave stores, if any, on their way meanwhile
    static_assert(CT * RT <= ROWS_WAVES);
    const int m = 16 * (wave % RT) + r, n = n0 + 16 * (wave / RT) + (lane >> 4) * 4;
    float row = 0.f, four[4] = {};
    if (wave < CT * RT) {
        row = a.x_scales[min(m, a.rows - 1)];
#pragma unroll
        for (int e = 0; e < 4; ++e) four[e] = a.w_scales[min(n + e, a.cols - 1)];
    }
    // the loads of several steps at once (those beyond the last: it again, not multiplied)
    constexpr int U = RT == 1 ? 4 : 2;
    for (int s = first + wave; s < end; s += ROWS_WAVES * U) {
        i32x4 fw[U][CT][2], fx[U][RT][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long k = (long)min(s + ROWS_WAVES * u, end - 1) * STEP;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < CT; ++i) fw[u][i][h] = *(const i32x4 *)(w[i] + k + 64 * h);
#pragma unroll
                for (int j = 0; j < RT; ++j) fx[u][j][h] = *(const i32x4 *)(x[j] + k + 64 * h);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + ROWS_WAVES * u >= end) break;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < CT; ++i)
#pragma unroll
                    for (int j = 0; j < RT; ++j) mma(acc[i][j], fw[u][i][h], fx[u][j][h]);
        }
    }
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
        for (int j = 0; j < RT; ++j) sums[wave][i * RT + j][lane] = acc[i][j];
    __syncthreads();
    if (wave >= CT * RT) return;
    i32x4 sum = sums[0][wave][lane];
#pragma unroll
    for (int k = 1; k < ROWS_WAVES; ++k) sum += sums[k][wave][lane];
    put<T>(a, part, m, n, sum, row, four);
}

// ---- tiles ----------------------------------------------------------------------------------------------------------
// 64 x 64 of z a workgroup, four waves of 32 x 32.  Two stages of LDS; the three steps of the reduction after the next are on their way into registers: a
// workgroup alone on its compute unit would else take as long as memory answers for each (65 x 4096 x 4096: 13.2 us, 16.3 with one ahead).
// Rows of 128 bytes, 16-byte piece c of row r at position c ^ (r / 2 % 8): the 16 rows of a fragment then take all banks in turn.  Bound by LDS where
// there are many tiles: two fragments read for each two products, 880 TOP/s (1024 x 4096 x 4096 in 39 us).  Tiles of 128 x 128 on the same way through registers, of which fewer fit a compute
// unit, took 6 % longer there, and 14 us for 8.5 at 777 x 1024 x 1352.
// QUADS: w is the left operand, a lane has four columns of a row; else x is, and 16 lanes have a row's columns side by side, which is what rows of z that cannot
// be stored four elements at a time want (777 x 1000 x 1351 in single: 64 separate words a store before, 11 us for 9.2, and 8.1 with the scales loaded ahead and the tile's place in the launch's
// three axes).
enum { TILE = 64, MOST_Y = 32768 };

template <class T, bool QUADS>
__global__ __launch_bounds__(256) void int8_tile_kernel(Args a) {
    constexpr int B = TILE, F = B / 32, PIECES = B * STEP / 16 / 256;
    __shared__ __attribute__((aligned(16))) signed char lds[2][2][B * STEP];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
    // tiles of rows, of columns, parts: (x, y, z); or, where there is one part, y and z both the columns' (a launch has less than 2^16 along either)
    const int part = a.parts > 1 ? blockIdx.z : 0, m0 = blockIdx.x * B, n0 = (a.parts > 1 ? blockIdx.y : blockIdx.z * MOST_Y + blockIdx.y) * B;
    if (n0 >= a.cols) return;
    const int first = (int)((long)a.steps * part / a.parts), end = (int)((long)a.steps * (part + 1) / a.parts);
    const signed char *from[2][PIECES];
    int to[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int p = tid + 256 * i, row = p >> 3, c = p & 7;
        from[0][i] = a.w + (long)min(n0 + row, a.cols - 1) * a.pitch + c * 16;  // (rows beyond the last: it again, not stored)
        from[1][i] = a.x + (long)min(m0 + row, a.rows - 1) * a.pitch + c * 16;
        to[i] = row * STEP + ((c ^ (row >> 1 & 7)) << 4);
    }
    constexpr int D = 3;
    i32x4 ahead[D][2][PIECES], acc[F][F] = {};
    // scales of what the lane stores, on their way meanwhile (QUADS: of its row and four columns; else of its column and four rows)
    float own[F], four[F][4];
    {
        const int n = n0 + wn * (B / 2), m = m0 + wm * (B / 2), l15 = lane & 15, l4 = (lane >> 4) * 4;
#pragma unroll
        for (int i = 0; i < F; ++i) {
            own[i] = QUADS ? a.x_scales[min(m + 16 * i + l15, a.rows - 1)] : a.w_scales[min(n + 16 * i + l15, a.cols - 1)];
#pragma unroll
            for (int e = 0; e < 4; ++e) four[i][e] = QUADS ? a.w_scales[min(n + 16 * i + l4 + e, a.cols - 1)] : a.x_scales[min(m + 16 * i + l4 + e, a.rows - 1)];
        }
    }
    auto fetch = [&](i32x4 (&to)[2][PIECES], int s) {
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int i = 0; i < PIECES; ++i) to[o][i] = *(const i32x4 *)(from[o][i] + (long)s * STEP);
    };
    auto stage = [&](const i32x4 (&x)[2][PIECES], int at) {
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int i = 0; i < PIECES; ++i) *(i32x4 *)(lds[at][o] + to[i]) = x[o][i];
    };
    const int r = lane & 15, j = lane >> 4, sw = r >> 1 & 7;
    // step s, which is in LDS; step s + 1 from `next` into LDS, step s + 1 + D on its way there
    auto step = [&](int s, i32x4 (&next)[2][PIECES]) {
        const int at = (s - first) & 1;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            i32x4 fw[F], fx[F];
            const int c = ((j + 4 * h) ^ sw) << 4;
#pragma unroll
            for (int i = 0; i < F; ++i) {
                fw[i] = *(const i32x4 *)(lds[at][0] + (wn * (B / 2) + 16 * i + r) * STEP + c);
                fx[i] = *(const i32x4 *)(lds[at][1] + (wm * (B / 2) + 16 * i + r) * STEP + c);
            }
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int k = 0; k < F; ++k) mma(acc[i][k], QUADS ? fw[i] : fx[k], QUADS ? fx[k] : fw[i]);
        }
        // (steps beyond the last: it again, not computed.  Without conditions the compiler knows how many loads are on their way and waits for no more
        // than it needs.)
        stage(next, at ^ 1);
        fetch(next, min(s + 1 + D, end - 1));
        __syncthreads();
    };
    if (first < end) {
#pragma unroll
        for (int d = 0; d < D; ++d) fetch(ahead[d], min(first + d, end - 1));
        stage(ahead[0], 0);
        fetch(ahead[0], min(first + D, end - 1));
        __syncthreads();
        int s = first;
        for (; s + D <= end; s += D) step(s, ahead[1]), step(s + 1, ahead[2]), step(s + 2, ahead[0]);
        if (s < end) step(s, ahead[1]);
        if (s + 1 < end) step(s + 1, ahead[2]);
    }
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int k = 0; k < F; ++k) {
            const int m = m0 + wm * (B / 2) + 16 * k, n = n0 + wn * (B / 2) + 16 * i;
            if constexpr (QUADS) {
                put<T>(a, part, m + r, n + j * 4, acc[i][k], own[k], four[i]);
            } else {
                T *z = (T *)a.z + (long)(m + j * 4) * a.ldz + n + r;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (m + j * 4 + e < a.rows && n + r < a.cols) z[e * a.ldz] = scaled<T>(acc[i][k][e], four[k][e], own[i]);
            }
        }
}

// ---- host -----------------------------------------------------------------------------------------------------------
enum { FEW_ROWS = 64 };

// How a call runs.
struct Plan {
    bool few;
    int parts, few_cols;
    long part_ld;
    size_t bytes(int rows) const { return parts > 1 ? sizeof(int) * (size_t)parts * rows * part_ld : 0; }
};

// Parts where workgroups are fewer than compute units, of 16 steps at least: a join costs 3 us and more, as much as some ten steps take (64 x 64 tiles, one part
// and two: 512 x 1024 x 1024 6.5 and 9.3 us, 256 x 2048 x 2048 8.6 and 10.2, 65 x 4096 x 4096 13.2 and 12.2).  Few rows, whose steps eight waves share: of 64, 32
// or 16 steps for 1, 2 or 4 tiles of rows (4 x 4096 x 2048 4.8 us, 7.6 in two parts; 40 x 8192 x 1024 16 in one, 9.7 in four).
Plan plan_of(int rows, int inner, int cols) {
    Plan p;
    const long steps = pitch_of(inner) / STEP, cus = cu_count();
    p.part_ld = (cols + 3L) / 4 * 4;
    p.few = rows <= FEW_ROWS;
    const int tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;  // of 16 rows
    // 32 columns a workgroup read x half as often; 16 where those would leave half the compute units idle (16 x 4096 x 4096 6.2 us, 10.8 with 32 and two parts,
    // but 8 x 2048 x 6144 7.9 and 7.0), unless x is large (64 x 11008 x 4096 28 and 27).
    p.few_cols = tiles < 4 && 2 * ceil_div(cols, 32) <= cus ? 16 : 32;
    const long groups = p.few ? ceil_div(cols, p.few_cols) : (long)ceil_div(rows, TILE) * ceil_div(cols, TILE);
    long parts = groups >= cus ? 1 : (2 * cus) / groups;
    const long most = steps / (p.few ? 64 / tiles : 16);
    parts = parts > most ? most : parts;
    p.parts = (int)(parts < 1 ? 1 : parts);
    return p;
}

template <class T>
int launch(Args a, const Plan &p, hipStream_t stream) {
    a.parts = p.parts, a.part_ld = p.part_ld;
    a.vec = a.ldz % 4 == 0 && ((size_t)a.z & (4 * sizeof(T) - 1)) == 0;
    if (p.few) {
        const long groups = ceil_div(a.cols, p.few_cols) * (long)p.parts;
        D8_REQUIRE(groups < (1L << 23), "matmul_int8: a result of %d x %d is too large", a.rows, a.cols);
        const dim3 grid(ceil_div(a.cols, p.few_cols), p.parts), threads(ROWS_WAVES * 64);
        auto few = [&](auto rt) {
            constexpr int RT = decltype(rt)::value;
            if constexpr (RT < 4) {
                if (p.few_cols == 16) {
                    hipLaunchKernelGGL((int8_rows_kernel<T, RT, 1>), grid, threads, 0, stream, a);
                    return;
                }
            }
            hipLaunchKernelGGL((int8_rows_kernel<T, RT, 2>), grid, threads, 0, stream, a);
        };
        if (a.rows <= 16) few(std::integral_constant<int, 1>());
        else if (a.rows <= 32) few(std::integral_constant<int, 2>());
        else few(std::integral_constant<int, 4>());
    } else {
        const long groups = (long)ceil_div(a.rows, TILE) * ceil_div(a.cols, TILE) * p.parts;
        const unsigned tiles = ceil_div(a.cols, TILE);
        const dim3 grid(ceil_div(a.rows, TILE), tiles < MOST_Y ? tiles : MOST_Y, p.parts > 1 ? p.parts : ceil_div(tiles, MOST_Y));
        D8_REQUIRE(groups < (1L << 24), "matmul_int8: a result of %d x %d is too large", a.rows, a.cols);
        if (a.vec || a.parts > 1) hipLaunchKernelGGL((int8_tile_kernel<T, true>), grid, dim3(256), 0, stream, a);
        else hipLaunchKernelGGL((int8_tile_kernel<T, false>), grid, dim3(256), 0, stream, a);
    }
    D8_LAUNCH_CHECK();
    if (p.parts > 1) {
        hipLaunchKernelGGL(int8_join_kernel<T>, dim3(ceil_div((long)a.rows * ((a.cols + 3) / 4), 256)), dim3(256), 0, stream, a);
        D8_LAUNCH_CHECK();
    }
    return 0;
}

bool sizes(int rows, int inner, int cols) { return rows >= 0 && inner >= 1 && inner <= MOST_INNER && cols >= 0 && (long)rows * ceil_div(cols, 4) < (1L << 37); }

}  // namespace
}  // namespace int8
}  // namespace d8

using namespace d8;

extern "C" size_t d8_matmul_int8_scratch_bytes(int rows, int inner, int cols) {
    if (!int8::sizes(rows, inner, cols) || !rows || !cols) return 0;
    return int8::plan_of(rows, inner, cols).bytes(rows);
}

extern "C" int d8_matmul_int8(int dtype, const signed char *x, const float *x_scales, int rows, int inner, const signed char *w, const float *w_scales, int cols,
                              void *z, long ldz, void *scratch, size_t scratch_bytes, void *stream) {
    if (dtype != D8_FLOAT16 && dtype != D8_FLOAT32) return fail(D8_ERR_DTYPE, "matmul_int8: type %d is not support", dtype);
    D8_REQUIRE(rows >= 0 && inner >= 1 && cols >= 0, "matmul_int8: %d x %d times %d x %d", rows, inner, inner, cols);
    D8_REQUIRE(inner <= int8::MOST_INNER, "matmul_int8: a sum has at most %d terms, not %d", (int)int8::MOST_INNER, inner);
    if (!rows || !cols) return 0;
    D8_REQUIRE(int8::sizes(rows, inner, cols), "matmul_int8: a result of %d x %d is too large", rows, cols);
    D8_REQUIRE(x && x_scales && w && w_scales && z, "matmul_int8: null tensor");
    D8_REQUIRE(ldz >= cols, "matmul_int8: rows of %d elements do not fit their leading dimension", cols);
    D8_REQUIRE((((size_t)x | (size_t)w) & 15) == 0, "matmul_int8: codes must be 16-byte aligned");
    int8::Args a;
    memset(&a, 0, sizeof(a));
    a.x = x, a.w = w, a.x_scales = x_scales, a.w_scales = w_scales, a.z = z, a.ldz = ldz, a.rows = rows, a.cols = cols, a.parts = 1;
    a.pitch = int8::pitch_of(inner), a.steps = (int)(a.pitch / int8::STEP);
    if (int8::wide_eligible(a)) return dtype == D8_FLOAT16 ? int8::wide_launch<f16>(a, as_stream(stream)) : int8::wide_launch<float>(a, as_stream(stream));
    const int8::Plan p = int8::plan_of(rows, inner, cols);
    const size_t need = p.bytes(rows);
    D8_REQUIRE(!need || (scratch && scratch_bytes >= need && ((size_t)scratch & 15) == 0), "matmul_int8: 16-byte aligned scratch of %zu bytes is needed, not %zu", need, scratch_bytes);
    a.part = (int *)scratch;
    return dtype == D8_FLOAT16 ? int8::launch<f16>(a, p, as_stream(stream)) : int8::launch<float>(a, p, as_stream(stream));
}
