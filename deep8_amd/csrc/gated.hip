// A gated feed-forward product and the way back:  pre = x w,  h = act(pre_g) * pre_u  with  w [inner][2 cols], pre_g the first `cols`
// columns of pre and pre_u the others.
//
// Both projections, the activation and the product are one kernel: a workgroup has the same columns of both halves, a lane's
// accumulators hold the gate and the factor of the same elements, and h is formed from the fp32 sums.  pre is written
// (rounded once) only where the way back will need it.
//
// Three kernels: many rows and columns in half on 256 x 256 tiles (gated_wide.hip); few rows, where reading w is the work (below:
// gated_rows_kernel); everything else on tiles of 64 or 128 rows.  All move operands in 16-byte pieces; operands whose rows do not start at
// multiples of 16 bytes are copied to rows that do, into scratch, first (single precision moved by elements, without copies, was no faster: 777 x
// 1000 times 1000 x 2 * 1351 69.4 us against 67.6).
#include "gated.h"

namespace d8 {
namespace gated {
namespace {

using attention::desc_t;
using attention::load_to_lds;
using attention::swizzle;

// the sigmoid of a and what it is short of 1, the sigmoid of -a (a difference would leave none of its bits far above 0)
__device__ __forceinline__ void both_sigmoids(float a, float &s, float &rest) {
    const float power = expf(-fabsf(a)), large = 1.f / (1.f + power), small = power * large;
    s = a < 0.f ? small : large, rest = a < 0.f ? large : small;
}

// activation and its slope
template <class T>
__device__ __forceinline__ void activation_slope(float a, int act, float &f, float &df) {
    float s, rest;
    switch (act) {
        case D8_GATE_SILU:
            both_sigmoids(a, s, rest);
            f = a * s, df = s * (1.f + a * rest);
            break;
        case D8_GATE_GELU: {
            const float p = normal_integral<T>(a);
            f = a * p, df = p + a * 0.39894228f * expf(-0.5f * a * a);
            break;
        }
        case D8_GATE_RELU:
            f = a > 0.f ? a : 0.f, df = a > 0.f ? 1.f : 0.f;
            break;
        default:
            both_sigmoids(a, s, rest);
            f = s, df = s * rest;
    }
}

// The columns of one workgroup on their way into a tile of `rows of w` x PB bytes: the gate's in the first half of a row, the factor's in the second.
template <class T, int PB>
struct WeightLoader {
    static constexpr int V = attention::Type<T>::V, ROWS = 1024 / PB, HALF = PB / 32;  // rows of a load, pieces of half a row
    int lane_row, lane_pos, left;  // left: pieces of the columns that are there
    unsigned stride, up;
    __device__ __forceinline__ void init(const Args &a, int n0, int lane) {
        lane_row = lane / (PB / 16), lane_pos = lane % (PB / 16), left = (a.cols_there - n0) / V;
        stride = (unsigned)a.ldw * (unsigned)sizeof(T), up = (unsigned)a.up * (unsigned)sizeof(T);
    }
    // row k0's column n0 of w on, `rows` rows
    __device__ __forceinline__ desc_t desc(const Args &a, int k0, int n0, int rows) const {
        const unsigned long p = (unsigned long)((const T *)a.w + (long)k0 * a.ldw + n0);
        const unsigned bytes = rows > 0 ? (unsigned)(rows - 1) * stride + up + (unsigned)(a.cols_there - n0) * (unsigned)sizeof(T) : 0u;
        return desc_t{(unsigned)__builtin_amdgcn_readfirstlane((int)p), (unsigned)__builtin_amdgcn_readfirstlane((int)(p >> 32)) & 0xffffu,
                      (unsigned)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
    }
    __device__ __forceinline__ void load(const desc_t &d, int t, unsigned tile) const {
        const int row = t * ROWS + lane_row, c = lane_pos ^ swizzle<PB>(row), second = c >= HALF, piece = c - (second ? HALF : 0);
        load_to_lds(d, piece < left ? row * stride + (second ? up : 0u) + piece * 16 : 0x80000000u, __builtin_amdgcn_readfirstlane(tile + t * 1024));
    }
};

// columns c0 .. c0 + 31 of a tile of w as an operand fragment whose k is in the order of read_rows
template <class T, int PB>
__device__ __forceinline__ typename attention::Type<T>::frag weight_frag(const char *tile, int r0, int c0, int lane) {
    if constexpr (sizeof(T) == 2) {
        typedef attention::tr_f16x4 tr;
        const int i = lane & 15, j = lane >> 4, row = r0 + 8 * (j >> 1) + (i >> 2), at = c0 * 2 + 32 * (j & 1) + 8 * (i & 3);
        const char *lo = tile + row * PB + ((((at >> 4) ^ swizzle<PB>(row)) << 4) | (at & 15));
        const char *hi = tile + (row + 4) * PB + ((((at >> 4) ^ swizzle<PB>(row + 4)) << 4) | (at & 15));
        const tr x = __builtin_amdgcn_ds_read_tr16_b64_v4f16(ATTN_LDS(tr, lo)), y = __builtin_amdgcn_ds_read_tr16_b64_v4f16(ATTN_LDS(tr, hi));
        return __builtin_bit_cast(f16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
        return attention::cols_frag<T, PB>(tile, r0, c0, lane);
    }
}

// K in steps of 128 bytes of x, both tiles straight into a stage of LDS, the next steps' while this one is worked on.  A workgroup's
// tile by SHAPE: TALL 128 rows x 64 columns of both halves, a wave 64 x 32 of each; SQUARE 64 x 64, a wave 32 x 32 of each; SMALL 64 x 32, a wave
// 32 x 32 of one half, and gate and factor meet through LDS at the end.  Single, 777 x 1000 x 2 * 1351: 57 us of SMALL, 74 TFLOP/s of 150 that a large
// product reaches: 559 tiles are 2.2 a compute unit, and a step's 1024 cycles of products take 1800 with one workgroup on it.  Half,
// 1024 x 4096 x 2 * 5632: 133 us of TALL, 710 TFLOP/s.
enum Shape { TALL, SQUARE, SMALL };
constexpr int tile_rows(int shape) { return shape == TALL ? 128 : 64; }
constexpr int tile_cols(int shape) { return shape == SMALL ? 32 : 64; }

template <class T, int SHAPE>
__global__ __launch_bounds__(256, 2) void gated_tile_kernel(Args a) {
    typedef attention::Type<T> M;
    typedef typename M::frag frag;
    constexpr int BM = tile_rows(SHAPE), BN = tile_cols(SHAPE), R = SHAPE == TALL ? 2 : 1, H = SHAPE == SMALL ? 1 : 2;  // row blocks, halves of a wave
    constexpr int PX = 128, BK = PX / (int)sizeof(T), PW = 2 * BN * (int)sizeof(T), TX = BM * PX, TW = BK * PW;
    // (half, small tiles: a third stage, since two hold too little work to wait for loads behind, 300 x 2048 x 2 * 2816 29 -> 24 us.  Larger tiles
    // would then share a compute unit with one less: 64 x 64 39 -> 48 us at 2000 x 2048 x 2 * 1408.  Single: no gain.)
    constexpr int STAGES = SHAPE == SMALL && sizeof(T) == 2 ? 3 : 2, LOADS = (TX + TW) / 4096;
    __shared__ __attribute__((aligned(1024))) char lds[STAGES * (TX + TW)];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    // (the workgroups of an XCD, ids congruent mod 8, have a run of row tiles by columns: what they share stays in its L2)
    const int tiles_m = (a.rows + BM - 1) / BM, unit = (int)blockIdx.x - a.whole;  // (unit: of the tiles in parts)
    int id = blockIdx.x;
    if (unit >= 0) id = a.whole + unit / a.parts;
    else if (a.whole % 8 == 0) id = id % 8 * (a.whole / 8) + id / 8;
    const int m0 = id % tiles_m * BM, n0 = id / tiles_m * BN;
    const int begin = unit >= 0 ? unit % a.parts * a.chunk : 0, end = unit >= 0 ? min(a.inner, begin + a.chunk) : a.inner;
    const int wm = (wave >> 1) * 32 * R, wn = SHAPE == SMALL ? 0 : (wave & 1) * 32, half = SHAPE == SMALL ? wave & 1 : 0;
    attention::TileLoader<T, PX> lx;
    lx.init(a.ldx, a.inner, lane);
    WeightLoader<T, PW> lw;
    lw.init(a, n0, lane);
    const unsigned lds0 = attention::lds_address(lds);
    auto fetch = [&](int k0, int stage) {
        const unsigned to = lds0 + stage * (TX + TW);
        lx.pieces = (a.inner_there - k0) / M::V;
        const desc_t dx = lx.desc((const T *)a.x + (long)m0 * a.ldx + k0, min(BM, a.rows - m0), a.ldx, a.inner_there - k0);
        const desc_t dw = lw.desc(a, k0, n0, min(BK, end - k0));
#pragma unroll
        for (int i = 0; i < TX / 4096; ++i) lx.load(dx, wave * (TX / 4096) + i, to);
#pragma unroll
        for (int i = 0; i < TW / 4096; ++i) lw.load(dw, wave * (TW / 4096) + i, to + TX);
    };
    f32x16 acc[R][H];
#pragma unroll
    for (int i = 0; i < R * H; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i / H][i % H][e] = 0.f;
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
        if (begin + i * BK < end) fetch(begin + i * BK, i);
    for (int k0 = begin, stage = 0; k0 < end; k0 += BK, stage = STAGES == 2 ? stage ^ 1 : stage == STAGES - 1 ? 0 : stage + 1) {
        // this step's tiles have landed; those of the steps after it may be on their way
        if (STAGES > 2 && k0 + (STAGES - 2) * BK < end) ATTN_VMCNT((STAGES - 2) * LOADS);
        else ATTN_VMCNT(0);
        attention::lds_reads_done();
        __syncthreads();
        const int ahead = k0 + (STAGES - 1) * BK;
        if (ahead < end) fetch(ahead, STAGES == 2 ? stage ^ 1 : stage == 0 ? STAGES - 1 : stage - 1);
        const char *tx = lds + stage * (TX + TW), *tw = tx + TX;
#pragma unroll
        for (int u = 0; u < BK / M::STEP; ++u) {
            frag xf[R], wf[H];
#pragma unroll
            for (int i = 0; i < R; ++i) xf[i] = attention::rows_frag<T, PX>(tx, wm + i * 32, u, lane);
#pragma unroll
            for (int j = 0; j < H; ++j) wf[j] = weight_frag<T, PW>(tw, u * M::STEP, (half + j) * BN + wn, lane);
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int j = 0; j < H; ++j) M::mma(acc[i][j], xf[i], wf[j]);
        }
    }
    const int n = n0 + wn + (lane & 31);
    if (unit >= 0) {
        float *to = a.part + ((long)unit * 2 + half) * BM * BN + wn + (lane & 31);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < H; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) to[(j * BM + wm + i * 32 + 8 * (e >> 2) + 4 * h + (e & 3)) * BN] = acc[i][j][e];
        return;
    }
    if constexpr (SHAPE == SMALL) {
        __syncthreads();
        float *to = (float *)lds + (wave >> 1) * 1024 + lane;
        if (half) {
#pragma unroll
            for (int e = 0; e < 16; ++e) to[e * 64] = acc[0][0][e];
        }
        __syncthreads();
        if (half || n >= a.cols) return;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int m = m0 + wm + 8 * (e >> 2) + 4 * h + (e & 3);
            if (m < a.rows) store<T>(a, m, n, acc[0][0][e], to[e * 64]);
        }
    } else {
        if (n >= a.cols) return;
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int m = m0 + wm + i * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
                if (m < a.rows) store<T>(a, m, n, acc[i][0][e], acc[i][H - 1][e]);
            }
    }
}

// the tiles in parts: a part's sums added up in order
template <class T, int SHAPE>
__global__ __launch_bounds__(256) void gated_parts_kernel(Args a) {
    constexpr int BM = tile_rows(SHAPE), BN = tile_cols(SHAPE), N = BM * BN;
    const int tiles_m = (a.rows + BM - 1) / BM, tile = blockIdx.x / (N / 256), at = blockIdx.x % (N / 256) * 256 + threadIdx.x, id = a.whole + tile;
    const int m = id % tiles_m * BM + at / BN, n = id / tiles_m * BN + at % BN;
    if (m >= a.rows || n >= a.cols) return;
    float g = 0.f, u = 0.f;
    const float *from = a.part + (long)tile * a.parts * 2 * N + at;
    for (int p = 0; p < a.parts; ++p, from += 2 * N) g += from[0], u += from[N];
    store<T>(a, m, n, g, u);
}

// Few rows.  A workgroup has 128 bytes of columns of both halves and a chunk of K, of which its four waves take every fourth tile of 32 rows of w,
// each with two stages of LDS of its own and no barrier; all rows of x (32 RB at most) are the other operand.  The waves' sums are
// joined through LDS; those of several chunks go through scratch (gated_join_kernel).  Bound by the bytes of w: half, 4 x 4096 x 2 * 8192, 134 MB
// in 25 us = 5.3 TB/s, 4 for the join.
template <class T, int RB>
__global__ __launch_bounds__(256, (RB == 1 && sizeof(T) == 2 ? 2 : 1)) void gated_rows_kernel(Args a) {
    typedef attention::Type<T> M;
    typedef typename M::frag frag;
    constexpr int PB = 256, BK = 32, TILE = BK * PB, LOADS = TILE / 1024, COLS = 128 / (int)sizeof(T), N = 2 * COLS / 32, UNITS = BK / M::STEP;
    constexpr int PX = BK * (int)sizeof(T), TX = RB * 32 * PX, LOADS_X = TX / 1024, STAGE = TILE + TX;
    constexpr int JOIN = 4 * N * RB * 16 * 64 * 4, STAGES = 4 * 2 * STAGE;
    __shared__ __attribute__((aligned(1024))) char lds[JOIN > STAGES ? JOIN : STAGES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int blocks = (a.cols + COLS - 1) / COLS, n0 = blockIdx.x % blocks * COLS, part = blockIdx.x / blocks;
    const int begin = part * a.chunk, end = min(a.inner, begin + a.chunk);
    WeightLoader<T, PB> lw;
    lw.init(a, n0, lane);
    attention::TileLoader<T, PX> lx;
    lx.init(a.ldx, a.inner, lane);
    const unsigned to = attention::lds_address(lds) + wave * 2 * STAGE;
    const int there = min((end + M::V - 1) / M::V * M::V, a.inner_there);  // of a row of x (chunks are whole pieces; zeros behind the last)
    auto fetch = [&](int k0, int stage) {
        const desc_t d = lw.desc(a, k0, n0, min(BK, end - k0)), dx = lx.desc((const T *)a.x + k0, a.rows, a.ldx, there - k0);
        lx.pieces = (there - k0) / M::V;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) lw.load(d, i, to + stage * STAGE);
#pragma unroll
        for (int i = 0; i < LOADS_X; ++i) lx.load(dx, i, to + stage * STAGE + TILE);
    };
    f32x16 acc[N][RB];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[n][r][e] = 0.f;
    int k0 = begin + wave * BK;
    if (k0 < end) fetch(k0, 0);
    for (int stage = 0; k0 < end; k0 += 4 * BK, stage ^= 1) {
        if (k0 + 4 * BK < end) {
            fetch(k0 + 4 * BK, stage ^ 1);
            ATTN_VMCNT(LOADS + LOADS_X);  // everything but the next tile has landed
        } else {
            ATTN_VMCNT(0);
        }
        asm volatile("" ::: "memory");
        const char *tw = lds + wave * 2 * STAGE + stage * STAGE, *tx = tw + TILE;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            frag xf[RB];
#pragma unroll
            for (int r = 0; r < RB; ++r) xf[r] = attention::rows_frag<T, PX>(tx, r * 32, u, lane);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const frag wf = weight_frag<T, PB>(tw, u * M::STEP, n * 32, lane);
#pragma unroll
                for (int r = 0; r < RB; ++r) M::mma(acc[n][r], wf, xf[r]);
            }
        }
        attention::lds_reads_done();
    }
    // element (column i, row j) of block (n, r) lies in lane j + 32 h, register e, i = 8 (e / 4) + 4 h + e % 4
    __syncthreads();
    float *all = (float *)lds;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int e = 0; e < 16; ++e) all[((wave * N + n) * RB + r) * 1024 + e * 64 + lane] = acc[n][r][e];
    __syncthreads();
    // a thread has a column of the block for every so many rows
    for (int i = tid; i < COLS * a.rows; i += 256) {
        const int c = i % COLS, row = i / COLS, n = n0 + c;
        if (n >= a.cols) continue;
        const int at = ((c >> 5) * RB + (row >> 5)) * 1024 + (((c & 31) >> 3) * 4 + (c & 3)) * 64 + (row & 31) + 32 * ((c >> 2) & 1);
        float g = 0.f, u = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) g += all[w * N * RB * 1024 + at], u += all[(w * N + N / 2) * RB * 1024 + at];
        if (a.parts == 1) {
            store<T>(a, row, n, g, u);
        } else {
            float *p = a.part + ((long)part * a.rows + row) * 2 * a.cols + n;
            p[0] = g, p[a.cols] = u;
        }
    }
}

template <class T>
__global__ __launch_bounds__(256) void gated_join_kernel(Args a) {
    const long n = (long)a.rows * a.cols, i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int row = (int)(i / a.cols), c = (int)(i - (long)row * a.cols);
    float g = 0.f, u = 0.f;
    for (int p = 0; p < a.parts; ++p) {
        const float *from = a.part + ((long)p * a.rows + row) * 2 * a.cols + c;
        g += from[0], u += from[a.cols];
    }
    store<T>(a, row, c, g, u);
}

// rows of `from` (width elements, `gap` elements after every `width`, as two halves where there are two) to rows that start at multiples of 16
// bytes, zeros behind them
template <class T>
__global__ __launch_bounds__(256) void gated_copy_kernel(const T *from, T *to, long rows, int width, int padded) {
    typedef typename attention::Type<T>::frag frag;
    constexpr int V = attention::Type<T>::V;
    const int per_row = padded / V;
    const long n = rows * per_row;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
        const long row = i / per_row;
        const int c = (int)(i - row * per_row) * V;
        *(frag *)(to + row * padded + c) = attention::load_piece<T>(from + row * width, c, width, true, 0);
    }
}

// dpre = (dh pre_u act'(pre_g), dh act(pre_g)), rounded to the type: the two products that follow are the framework's, which take half operands (2.9
// for 2.1 10^-4 of error in dx and dw); a thread has 16 bytes of each half.  Bound by bytes: 4096 x 2 * 5632 halves, 231 MB in 38 us = 6.1 TB/s
template <class T>
__global__ __launch_bounds__(256) void gated_slope_kernel(Args a) {
    typedef typename attention::Type<T>::frag frag;
    constexpr int V = attention::Type<T>::V;
    const int per_row = (a.cols + V - 1) / V;
    const long n = (long)a.rows * per_row;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
        const long row = i / per_row;
        const int c = (int)(i - row * per_row) * V;
        const T *pre = (const T *)a.pre + row * 2 * a.cols;
        const frag g = attention::load_piece<T>(pre, c, a.cols, true, a.vec), u = attention::load_piece<T>(pre + a.cols, c, a.cols, true, a.vec);
        const frag d = attention::load_piece<T>((const T *)a.dh + row * a.cols, c, a.cols, true, a.vec);
        frag dg, du;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float f, df;
            activation_slope<T>((float)g[e], a.act, f, df);
            dg[e] = (T)((float)d[e] * (float)u[e] * df), du[e] = (T)((float)d[e] * f);
        }
        T *to = (T *)a.dpre + row * 2 * a.cols;
        if (a.vec) {
            *(frag *)(to + c) = dg, *(frag *)(to + a.cols + c) = du;
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (c + e < a.cols) to[c + e] = dg[e], to[a.cols + c + e] = du[e];
        }
    }
}

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

int check(int dtype, int rows, int inner, int cols, int act, const char *name) {
    if (dtype != D8_FLOAT16 && dtype != D8_FLOAT32) return fail(D8_ERR_DTYPE, "%s: type %d is not support", name, dtype);
    D8_REQUIRE(rows >= 1 && inner >= 1 && cols >= 1 && cols < (1 << 28) && inner < (1 << 28), "%s: %d x %d times %d x 2 * %d", name, rows, inner, inner, cols);
    D8_REQUIRE(act >= D8_GATE_SILU && act <= D8_GATE_SIGMOID, "%s: activation %d is not support", name, act);
    return 0;
}

enum { FEW_ROWS = 64 };
// Offsets into a tile are 32 bits, and 2^31 stands for what is not there: the rows of x that a tile has, at most 128, and the 32 (half, more
// than FEW_ROWS rows: 64) rows of w of a step must not be more bytes than that.  (gated_wide.hip asks for less than 2^31 of each whole operand.)
bool fits(int dtype, long rows, long inner, long cols) {
    const long es = (long)dtype_bytes(dtype), v = 16 / es, step = rows > FEW_ROWS && dtype == D8_FLOAT16 ? 64 : 32;
    const long x_row = (inner + v - 1) / v * 16, w_row = 2 * ((cols + v - 1) / v * 16);
    return (rows < 128 ? rows : 128) * x_row <= (1L << 31) && step * w_row <= (1L << 31);
}
// What a 32 x 32 block of both products takes a compute unit per element of K (microseconds): alone on it, where a workgroup waits for its
// loads and barriers, and beside others; and what a second launch takes.  Measured with one and with eight tiles a compute unit, calls of K = 2056 (half)
// and 1032 (single), launch included, in nanoseconds: half TALL 2.3 and 1.6, SQUARE 3.3 and 1.7, SMALL 5.0 and 3.0; single 11.0 and 8.9, 13.5 and 9.0,
// 16.4 and 9.7.  The constants times `cost` are near these; K = 8200 (4104) has 1.7, 2.6, 3.3 (9.2, 11.7, 13.2) alone.  Over twelve sizes of 96 to 2000
// rows the choice by them was the best of all shapes and parts or up to 8 % slower, and 13 and 18 % at 1024 x 4104 x 2 * 5632 and 1000 x 1024 x 2 * 1352.
constexpr float ALONE[2] = {0.0029f, 0.0135f}, TOGETHER[2] = {0.00135f, 0.0095f}, JOIN_US = 4.f;  // half, single

// How a forward call runs and what it takes of the scratch: copies of x and w (bytes, 0: read as they lie), partial sums.
struct Plan {
    enum { ROWS, TILES } way;
    int shape, parts, chunk, whole;
    size_t x_copy, w_copy, part;
    size_t bytes() const { return x_copy + w_copy + part; }
};

Plan plan_of(int dtype, int rows, int inner, int cols, bool x_aligned, bool w_aligned) {
    Plan p;
    memset(&p, 0, sizeof(p));
    const size_t es = dtype_bytes(dtype);
    const int v = 16 / (int)es;
    const long inner_p = (inner + v - 1L) / v * v, cols_p = (cols + v - 1L) / v * v;
    if (!x_aligned || inner % v) p.x_copy = round256(es * rows * inner_p);
    if (!w_aligned || cols % v) p.w_copy = round256(es * inner * 2 * cols_p);
    if (rows <= FEW_ROWS) {
        // two workgroups a compute unit, chunks of K of at least four tiles a wave's
        p.way = Plan::ROWS;
        const long blocks = (cols * (long)es + 127) / 128, most = (inner + 511) / 512;
        long parts = blocks >= 2 * cu_count() ? 1 : (2 * cu_count() + blocks - 1) / blocks;
        parts = parts > most ? most : parts;
        p.chunk = (int)(((inner + parts - 1) / parts + 127) / 128 * 128);
        p.parts = (int)((inner + p.chunk - 1L) / p.chunk);
        if (p.parts > 1) p.part = round256(sizeof(float) * p.parts * (size_t)rows * 2 * cols);
        return p;
    }
    p.way = Plan::TILES;
    // The shape whose busiest compute unit is through first: blocks of 32 x 32 products, weighed with what a block costs in it.  The tiles that
    // are left when every compute unit has had as many as all others may be cut along K into parts, so that they too go over the whole chip,
    // where that saves more than the second launch and the partial sums' way through memory cost.  Single, 777 x 1000 x 2 * 1351 (559 tiles of
    // 64 x 32, 47 of them in five parts): 76 -> 68 us; half, 128 x 4096 x 2 * 2048 (all 64 tiles of 64 x 64 in four): 37 -> 19 us.
    static const float cost[2][3] = {{1.f, 1.25f, 1.6f}, {1.f, 1.05f, 1.1f}};  // half, single
    const int single = dtype == D8_FLOAT32, bk = 128 / (int)es;
    const long cus = cu_count();
    float best = 0.f;
    for (int s = TALL; s <= SMALL; ++s) {
        const long tiles = (long)ceil_div(rows, tile_rows(s)) * ceil_div(cols, tile_cols(s)), rest = tiles % cus;
        const float tile = (float)inner * (tile_rows(s) / 32) * (tile_cols(s) / 32) * cost[single][s];
        for (int want = 1; want <= (rest ? 16 : 1); ++want) {
            const int chunk = (int)(((inner + want - 1L) / want + bk - 1) / bk * bk), parts = (inner + chunk - 1) / chunk;
            if (want > 1 && (parts < want || chunk < 4 * bk)) continue;
            const float share = parts == 1 ? 1.f : (float)chunk / inner;  // of a tile, what a part is
            const float longest = tiles >= cus ? 1.f : share, load = (float)(tiles / cus) + (float)((rest * parts + cus - 1) / cus) * share;
            const float join = parts == 1 ? 0.f : JOIN_US + (float)rest * (parts + 1) * tile_rows(s) * tile_cols(s) * 16.f / 4e6f;
            const float t = tile * fmaxf(ALONE[single] * longest, TOGETHER[single] * load) + join;
            if ((s == TALL && want == 1) || t < (p.parts == 1 ? 0.95f : 1.f) * best) best = t, p.shape = s, p.parts = parts, p.chunk = parts == 1 ? inner : chunk, p.whole = (int)(parts == 1 ? tiles : tiles - rest);
        }
    }
    if (p.parts > 1) {
        const long rest = (long)ceil_div(rows, tile_rows(p.shape)) * ceil_div(cols, tile_cols(p.shape)) - p.whole;
        p.part = round256(sizeof(float) * 2 * (size_t)rest * p.parts * tile_rows(p.shape) * tile_cols(p.shape));
    }
    return p;
}

}  // namespace
}  // namespace gated
}  // namespace d8

using namespace d8;

extern "C" size_t d8_matmul_gated_scratch_bytes(int dtype, int which, int rows, int inner, int cols) {
    if ((dtype != D8_FLOAT16 && dtype != D8_FLOAT32) || rows < 1 || inner < 1 || cols < 1 || cols >= (1 << 28) || inner >= (1 << 28)) return 0;
    if (which != 1) return !gated::fits(dtype, rows, inner, cols) ? 0 : gated::plan_of(dtype, rows, inner, cols, which != 2, which != 2).bytes();
    return gated::round256(dtype_bytes(dtype) * 2 * (size_t)rows * cols) + d8_matmul_scratch_bytes(dtype, 3, 1, rows, inner, 1, inner, 2 * cols);
}

namespace d8 {
namespace gated {
namespace {

template <class T>
int copy_rows(const void *from, void *to, long rows, int width, int padded, hipStream_t stream) {
    const long groups = (rows * (padded / attention::Type<T>::V) + 255) / 256;
    hipLaunchKernelGGL(gated_copy_kernel<T>, dim3((unsigned)(groups < 8192 ? groups : 8192)), dim3(256), 0, stream, (const T *)from, (T *)to, rows, width, padded);
    D8_LAUNCH_CHECK();
    return 0;
}

template <class T, int SHAPE>
int launch_tiles(const Args &a, hipStream_t stream) {
    const long tiles = (long)ceil_div(a.rows, tile_rows(SHAPE)) * ceil_div(a.cols, tile_cols(SHAPE));
    D8_REQUIRE(tiles < (1L << 30), "matmul_gated: too many rows");
    const long rest = tiles - a.whole;
    hipLaunchKernelGGL((gated_tile_kernel<T, SHAPE>), dim3((unsigned)(a.whole + rest * a.parts)), dim3(256), 0, stream, a);
    D8_LAUNCH_CHECK();
    if (!rest) return 0;
    hipLaunchKernelGGL((gated_parts_kernel<T, SHAPE>), dim3((unsigned)(rest * (tile_rows(SHAPE) * tile_cols(SHAPE) / 256))), dim3(256), 0, stream, a);
    D8_LAUNCH_CHECK();
    return 0;
}

template <class T>
int forward(Args a, const Plan &p, char *scratch, hipStream_t stream) {
    constexpr int V = attention::Type<T>::V;
    a.ldx = a.inner_there = a.inner, a.ldw = 2L * a.cols, a.up = a.cols_there = a.cols;
    if (p.x_copy) {
        a.ldx = a.inner_there = (a.inner + V - 1) / V * V;
        if (int rc = copy_rows<T>(a.x, scratch, a.rows, a.inner, a.inner_there, stream)) return rc;
        a.x = scratch, scratch += p.x_copy;
    }
    if (p.w_copy) {  // (a row of w is two rows of `cols`)
        a.up = a.cols_there = (a.cols + V - 1) / V * V, a.ldw = 2L * a.up;
        if (int rc = copy_rows<T>(a.w, scratch, 2L * a.inner, a.cols, a.cols_there, stream)) return rc;
        a.w = scratch, scratch += p.w_copy;
    }
    a.part = (float *)scratch, a.parts = p.parts, a.chunk = p.chunk, a.whole = p.whole;
    if (p.way == Plan::ROWS) {
        const dim3 grid((unsigned)ceil_div((long)a.cols * sizeof(T), 128) * p.parts);
        if (a.rows <= 32) hipLaunchKernelGGL((gated_rows_kernel<T, 1>), grid, dim3(256), 0, stream, a);
        else hipLaunchKernelGGL((gated_rows_kernel<T, 2>), grid, dim3(256), 0, stream, a);
        D8_LAUNCH_CHECK();
        if (p.parts == 1) return 0;
        hipLaunchKernelGGL(gated_join_kernel<T>, dim3(ceil_div((long)a.rows * a.cols, 256)), dim3(256), 0, stream, a);
        D8_LAUNCH_CHECK();
        return 0;
    }
    switch (p.shape) {
        case TALL: return launch_tiles<T, TALL>(a, stream);
        case SQUARE: return launch_tiles<T, SQUARE>(a, stream);
        default: return launch_tiles<T, SMALL>(a, stream);
    }
}

}  // namespace
}  // namespace gated
}  // namespace d8

extern "C" int d8_matmul_gated(int dtype, const void *x, int rows, int inner, const void *w, int cols, int act, void *pre, void *h, void *scratch,
                               size_t scratch_bytes, void *stream) {
    if (int rc = gated::check(dtype, rows, inner, cols, act, "matmul_gated")) return rc;
    D8_REQUIRE(gated::fits(dtype, rows, inner, cols), "matmul_gated: rows of %d and 2 * %d elements are too long", inner, cols);
    D8_REQUIRE(x && w && h, "matmul_gated: null tensor");
    gated::Args a;
    memset(&a, 0, sizeof(a));
    a.x = x, a.w = w, a.pre = pre, a.h = h, a.rows = rows, a.inner = inner, a.cols = cols, a.act = act;
    if (dtype == D8_FLOAT16 && gated::wide_eligible(a)) return gated::wide_launch(a, as_stream(stream));
    const gated::Plan p = gated::plan_of(dtype, rows, inner, cols, ((size_t)x & 15) == 0, ((size_t)w & 15) == 0);
    const size_t need = p.bytes();
    D8_REQUIRE(!need || (scratch && scratch_bytes >= need && ((size_t)scratch & 15) == 0), "matmul_gated: 16-byte aligned scratch of %zu bytes is needed, not %zu", need, scratch_bytes);
    return dtype == D8_FLOAT16 ? gated::forward<f16>(a, p, (char *)scratch, as_stream(stream)) : gated::forward<float>(a, p, (char *)scratch, as_stream(stream));
}

extern "C" int d8_matmul_gated_grad(int dtype, const void *x, void *dx, int rows, int inner, const void *w, void *dw, int cols, int act, const void *pre,
                                    const void *dh, int overwrite, void *scratch, size_t scratch_bytes, void *stream) {
    if (int rc = gated::check(dtype, rows, inner, cols, act, "matmul_gated_grad")) return rc;
    D8_REQUIRE(x && w && dx && dw && pre && dh, "matmul_gated_grad: null tensor");
    const size_t need = d8_matmul_gated_scratch_bytes(dtype, 1, rows, inner, cols), own = gated::round256(dtype_bytes(dtype) * 2 * (size_t)rows * cols);
    D8_REQUIRE(scratch && scratch_bytes >= need && ((size_t)scratch & 15) == 0, "matmul_gated_grad: 16-byte aligned scratch of %zu bytes is needed, not %zu", need, scratch_bytes);
    gated::Args a;
    memset(&a, 0, sizeof(a));
    a.pre = (void *)pre, a.dh = dh, a.dpre = scratch, a.rows = rows, a.inner = inner, a.cols = cols, a.act = act;
    const int v = 16 / (int)dtype_bytes(dtype);
    a.vec = cols % v == 0 && (((size_t)pre | (size_t)dh) & 15) == 0;
    const long threads = (long)rows * ceil_div(cols, v);
    const dim3 grid((unsigned)((threads + 255) / 256 < 16384 ? (threads + 255) / 256 : 16384));
    if (dtype == D8_FLOAT16) hipLaunchKernelGGL(gated::gated_slope_kernel<f16>, grid, dim3(256), 0, as_stream(stream), a);
    else hipLaunchKernelGGL(gated::gated_slope_kernel<float>, grid, dim3(256), 0, as_stream(stream), a);
    D8_LAUNCH_CHECK();
    void *rest = scratch_bytes > own ? (char *)scratch + own : nullptr;
    return d8_matmul_grad_xy(dtype, x, dx, 1, rows, inner, w, dw, 1, inner, 2 * cols, scratch, overwrite, rest, scratch_bytes - own, stream);
}
