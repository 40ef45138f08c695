// The gated product (gated.hip) of many rows and columns in half: the 256 x 256 tile loop of gemm_wide_kernel.h, whose 256 columns of w
// are 128 of the gate and the same 128 of the factor, arranged so that each wave has 64 of both: what a wave's lanes fetch decides it,
// LDS layout, fragments and the order of the products are the plain product's.  The epilogue forms h from the accumulators.
//
// Bound by the matrix pipe's power like the plain product: 8192 x 4096 x 2 * 8192 in 840 us at the least = 1310 TFLOP/s (a large plain product 1320), 890
// in the mean of 40 calls in a row, at 1.86 GHz.  The
// epilogue reads no memory and writes h, and g and u for training, 16 bytes a lane in whole 128-byte lines.
#include "gated.h"
#include "gemm_wide_kernel.h"

namespace d8 {
namespace gated {

struct WideArgs {
    const f16 *x, *w;
    f16 *pre, *h;
    int rows, inner, cols, tilesM, tilesN, total;
    // the plain product that the tile loop knows: 2 cols columns, a tile's first column, halved, is its first column of either half
    __device__ __forceinline__ wide::Launch product() const {
        wide::Launch L;
        wide::Product &p = L.p[0];
        p.A = x, p.B = w, p.C = nullptr, p.bias = nullptr, p.M = rows, p.N = 2 * cols, p.K = inner, p.lda = inner, p.ldb = 2 * cols, p.ldc = 0;
        p.sA = p.sB = p.sC = 0, p.tilesM = tilesM, p.tilesN = tilesN, p.tiles = total, p.form = wide::FORM_NN, p.beta = 0.f, p.relu = 0;
        L.n = 1, L.total = total, L.rec = nullptr;
        return L;
    }
};

typedef wide::TileOperands<true, false> WideOperands;

// The operands of the tile at `w`: a lane's pieces of w moved to where its columns come from.  Piece c of a row of the tile (8 columns) belongs
// to wave column c / 16, to the factor if c / 8 is odd, and is piece c % 8 of those 64 columns.
__device__ __forceinline__ void wide_operands(WideOperands &T, const WideArgs &all, const wide::Where &w, int wave, int lane) {
    WideArgs a = all;
    asm volatile("" : "+s"(a.rows), "+s"(a.inner), "+s"(a.cols), "+v"(lane));  // per tile, not once and kept: scalar registers are short
    T.init<wide::Shipped>(a.product().p[0], w, wave, lane);
    const int kr = wave * 2 + (lane >> 5), pos = lane & 31;
#pragma unroll
    for (int par = 0; par < 2; ++par) {
        const int c = pos ^ (((kr & 3) | (par << 2)) << 1);
        T.ob.voff[par] = 2u * ((unsigned)kr * 2u * (unsigned)a.cols + (unsigned)((c >> 4) * 64 + (c & 7) * 8) + ((c >> 3) & 1 ? (unsigned)a.cols : 0u));
    }
    T.b_org = (unsigned)w.n0;  // 2 bytes times n0 / 2 columns
}

// A finished tile on its way out, 16 rows at a time through the wave's patch of LDS (gemm_wide_kernel.h: store_tile); a lane has eight columns
// of both halves in two of the rows.
template <bool INTERIOR, bool KEEP, int ACT>
__device__ __forceinline__ void store_gated(const WideArgs &all, const wide::Where &w, float *patch, int wave, int lane, f32x4 (&acc)[8][8]) {
    WideArgs a = all;
    asm volatile("" : "+s"(a.cols), "+v"(lane));
    const int wm = wave >> 1, wn = wave & 1;
    const int l15 = lane & 15, l4 = lane >> 4, chunk = lane & 7, up_row = lane >> 3;
    const int n = w.n0 / 2 + wn * 64 + chunk * 8;
    unsigned wr[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) wr[q] = (unsigned)(size_t)WIDE_LDS(float, patch) + 4u * ((4 * l4) * 128 + ((q ^ l4) * 16 + l15));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        wide::write_slab<0>(wr, acc[i]);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int row = t * 8 + up_row, at = (chunk * 8) ^ ((row >> 2) * 16), m = w.m0 + wm * 128 + i * 16 + row;
            float g[8], u[8];
            *(f32x4 *)&g[0] = *(const f32x4 *)(patch + row * 128 + at);
            *(f32x4 *)&g[4] = *(const f32x4 *)(patch + row * 128 + at + 4);
            *(f32x4 *)&u[0] = *(const f32x4 *)(patch + row * 128 + 64 + at);
            *(f32x4 *)&u[4] = *(const f32x4 *)(patch + row * 128 + 64 + at + 4);
            if (!INTERIOR && (m < w.m_own || n < w.n_own / 2)) continue;
            f16x8 h;
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = (f16)(activation<f16>(g[e], ACT) * u[e]);
            __builtin_nontemporal_store(h, (f16x8 *)(a.h + (long)m * a.cols + n));
            if (KEEP) {
                f16x8 g16, u16;
#pragma unroll
                for (int e = 0; e < 8; ++e) g16[e] = (f16)g[e], u16[e] = (f16)u[e];
                f16 *p = a.pre + (long)m * 2 * a.cols + n;
                __builtin_nontemporal_store(g16, (f16x8 *)p);
                __builtin_nontemporal_store(u16, (f16x8 *)(p + a.cols));
            }
        }
    }
}

template <bool KEEP, int ACT>
__global__ __launch_bounds__(256) void gated_wide_kernel(WideArgs a) {
    using namespace wide;
    __shared__ __attribute__((aligned(1024))) char lds[LDS_BYTES];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    float *patch = (float *)(lds + 2 * STAGE_BYTES) + wave * (16 * 128);
    const unsigned wave_base = (unsigned)(size_t)WIDE_LDS(const char, lds) + wave * 1024;
    f32x4 acc[8][8];
    int idx = blockIdx.x;
    Where cur = locate(a.product(), idx);
    {
        WideOperands T;
        wide_operands(T, a, cur, wave, lane);
        T.issue_first_steps(wave_base);
    }
    __builtin_amdgcn_s_waitcnt(0x4f70);  // vmcnt(16): the first stage has landed
    __syncthreads();
    for (;;) {
        const int nidx = idx + gridDim.x;
        const bool more = nidx < a.total;
        const Where nxt = more ? locate(a.product(), nidx) : cur;
        {
            WideOperands T;
            wide_operands(T, a, cur, wave, lane);
            k_loop<Shipped, true, false>(T, lds, wave_base, acc);
        }
        if (more) {  // the next tile's first two steps set out before this tile's epilogue: 32 loads a wave
            WideOperands T;
            wide_operands(T, a, nxt, wave, lane);
            T.issue_first_steps(wave_base);
        }
        const bool interior = cur.m0 == cur.m_own && cur.n0 == cur.n_own;
        if (interior) store_gated<true, KEEP, ACT>(a, cur, patch, wave, lane, acc);
        else store_gated<false, KEEP, ACT>(a, cur, patch, wave, lane, acc);
        if (!more) break;
        // an interior tile's epilogue has issued 16 stores (48 with g and u) after those 32 loads, and vector-memory instructions
        // complete in order: at most 16 outstanding, and the loads have landed
        if (interior) __builtin_amdgcn_s_waitcnt(0x4f70);
        else __builtin_amdgcn_s_waitcnt(0x0f70);
        __syncthreads();
        cur = nxt, idx = nidx;
    }
}

template <int ACT>
int launch_act(const WideArgs &a, int grid, hipStream_t stream) {
    if (a.pre) hipLaunchKernelGGL((gated_wide_kernel<true, ACT>), dim3(grid), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((gated_wide_kernel<false, ACT>), dim3(grid), dim3(256), 0, stream, a);
    D8_LAUNCH_CHECK();
    return 0;
}

bool wide_eligible(const Args &a) {
    if (a.rows < 256 || a.cols < 128 || a.inner < 64 || a.inner % 64 || a.cols % 8) return false;
    if (((size_t)a.x | (size_t)a.w | (size_t)a.h | (size_t)a.pre) & 15) return false;
    if (2L * a.rows * a.inner >= (1L << 31) || 4L * a.inner * a.cols >= (1L << 31)) return false;
    const long tiles = (long)ceil_div(a.rows, 256) * ceil_div(a.cols, 128);
    return 4 * tiles >= 3L * cu_count() && tiles < (1L << 30);
}

// x and w as they lie: no copies (whole pieces by wide_eligible)
int wide_launch(const Args &args, hipStream_t stream) {
    WideArgs a;
    a.x = (const f16 *)args.x, a.w = (const f16 *)args.w, a.pre = (f16 *)args.pre, a.h = (f16 *)args.h;
    a.rows = args.rows, a.inner = args.inner, a.cols = args.cols;
    a.tilesM = ceil_div(a.rows, 256), a.tilesN = ceil_div(a.cols, 128), a.total = a.tilesM * a.tilesN;
    const int cus = cu_count(), grid = a.total <= cus ? a.total : cus >= 8 ? cus - cus % 8 : cus;
    switch (args.act) {  // (a kernel each: a switch around every element of an unrolled epilogue would be most of the code)
        case D8_GATE_SILU: return launch_act<D8_GATE_SILU>(a, grid, stream);
        case D8_GATE_GELU: return launch_act<D8_GATE_GELU>(a, grid, stream);
        case D8_GATE_RELU: return launch_act<D8_GATE_RELU>(a, grid, stream);
        default: return launch_act<D8_GATE_SIGMOID>(a, grid, stream);
    }
}

}  // namespace gated
}  // namespace d8
