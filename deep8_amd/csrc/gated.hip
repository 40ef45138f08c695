// A gated feed-forward product and the way back:  pre = x w,  h = act(pre_g) * pre_u  with  w [inner][2 cols], pre_g the first `cols`
// columns of pre and pre_u the others.
//
// Both projections, the activation and the product are one kernel: a workgroup has the same columns of both halves, a lane's
// accumulators hold the gate and the factor of the same elements, and h is formed from the fp32 sums.  pre is written
// (rounded once) only where the way back will need it.
#include "attention.h"

namespace d8 {
namespace gated {
namespace {

struct Args {
    const void *x, *w;
    void *pre, *h;
    const void *dh;
    void *dpre;
    int rows, inner, cols, act;
    int vec_x, vec_w;
};

__device__ __forceinline__ float activation(float a, int act) {
    switch (act) {
        case D8_GATE_SILU: return a / (1.f + expf(-a));
        case D8_GATE_GELU: return 0.5f * a * (1.f + erff(a * 0.70710678f));
        case D8_GATE_RELU: return a > 0.f ? a : 0.f;
        default: return 1.f / (1.f + expf(-a));
    }
}

// activation and its slope
__device__ __forceinline__ void activation_slope(float a, int act, float &f, float &df) {
    switch (act) {
        case D8_GATE_SILU: {
            const float s = 1.f / (1.f + expf(-a));
            f = a * s, df = s * (1.f + a * (1.f - s));
            break;
        }
        case D8_GATE_GELU: {
            const float p = 0.5f * (1.f + erff(a * 0.70710678f));
            f = a * p, df = p + a * 0.39894228f * expf(-0.5f * a * a);
            break;
        }
        case D8_GATE_RELU:
            f = a > 0.f ? a : 0.f, df = a > 0.f ? 1.f : 0.f;
            break;
        default: {
            const float s = 1.f / (1.f + expf(-a));
            f = s, df = s * (1.f - s);
        }
    }
}

enum { BM = 128, BN = 64 };

// 128 rows x 64 columns of both halves a workgroup, a wave 64 x 32 of each
template <class T>
__global__ __launch_bounds__(256) void gated_tile_kernel(Args a) {
    typedef attention::Type<T> M;
    typedef typename M::frag frag;
    constexpr int BK = 2 * M::STEP, PX = BK * (int)sizeof(T) + 16, PW = 2 * BN * (int)sizeof(T) + 16;
    __shared__ __attribute__((aligned(16))) char tile_x[BM * PX], tile_w[BK * PW];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int m0 = blockIdx.y * BM, n0 = blockIdx.x * BN, wm = (wave >> 1) * 64, wn = (wave & 1) * 32;
    const T *x = (const T *)a.x, *w = (const T *)a.w;
    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i >> 1][i & 1][e] = 0.f;
    for (int k0 = 0; k0 < a.inner; k0 += BK) {
        __syncthreads();
        for (int p = tid; p < BM * BK / M::V; p += 256) {
            const int r = p / (BK / M::V), c = p % (BK / M::V) * M::V;
            const bool in = m0 + r < a.rows;
            *(frag *)(tile_x + r * PX + c * (int)sizeof(T)) = attention::load_piece<T>(x + (long)(in ? m0 + r : 0) * a.inner, k0 + c, a.inner, in, a.vec_x);
        }
        for (int p = tid; p < BK * 2 * BN / M::V; p += 256) {
            const int r = p / (2 * BN / M::V), c = p % (2 * BN / M::V) * M::V, up = c >= BN;
            const bool in = k0 + r < a.inner;
            *(frag *)(tile_w + r * PW + c * (int)sizeof(T)) =
                attention::load_piece<T>(w + (long)(in ? k0 + r : 0) * 2 * a.cols + (up ? a.cols : 0), n0 + c - (up ? BN : 0), a.cols, in, a.vec_w);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < BK / M::STEP; ++u) {
            frag xf[2], wf[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                xf[i] = attention::read_rows<T>(tile_x + (wm + i * 32) * PX, PX, u, lane);
                wf[i] = M::template read_cols<true>(tile_w, PW, u * M::STEP, i * BN + wn, lane);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) M::mma(acc[i][j], xf[i], wf[j]);
        }
    }
    const int n = n0 + wn + (lane & 31);
    if (n >= a.cols) return;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int m = m0 + wm + i * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
            if (m >= a.rows) continue;
            const float g = acc[i][0][e], u = acc[i][1][e];
            ((T *)a.h)[(long)m * a.cols + n] = (T)(activation(g, a.act) * u);
            if (a.pre) {
                T *p = (T *)a.pre + (long)m * 2 * a.cols + n;
                p[0] = (T)g, p[a.cols] = (T)u;
            }
        }
}

// dpre = (dh pre_u act'(pre_g), dh act(pre_g)); a thread has 16 bytes of each half
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
        const frag g = attention::load_piece<T>(pre, c, a.cols, true, a.vec_w), u = attention::load_piece<T>(pre + a.cols, c, a.cols, true, a.vec_w);
        const frag d = attention::load_piece<T>((const T *)a.dh + row * a.cols, c, a.cols, true, a.vec_w);
        frag dg, du;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float f, df;
            activation_slope((float)g[e], a.act, f, df);
            dg[e] = (T)((float)d[e] * (float)u[e] * df), du[e] = (T)((float)d[e] * f);
        }
        T *to = (T *)a.dpre + row * 2 * a.cols;
        if (a.vec_w) {
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
    D8_REQUIRE(rows >= 1 && inner >= 1 && cols >= 1 && cols < (1 << 30), "%s: %d x %d times %d x 2 * %d", name, rows, inner, inner, cols);
    D8_REQUIRE(act >= D8_GATE_SILU && act <= D8_GATE_SIGMOID, "%s: activation %d is not support", name, act);
    return 0;
}

}  // namespace
}  // namespace gated
}  // namespace d8

using namespace d8;

extern "C" size_t d8_matmul_gated_scratch_bytes(int dtype, int which, int rows, int inner, int cols) {
    if ((dtype != D8_FLOAT16 && dtype != D8_FLOAT32) || rows < 1 || inner < 1 || cols < 1 || cols >= (1 << 30)) return 0;
    if (which != 1) return 0;
    return gated::round256(dtype_bytes(dtype) * 2 * (size_t)rows * cols) + d8_matmul_scratch_bytes(dtype, 3, 1, rows, inner, 1, inner, 2 * cols);
}

extern "C" int d8_matmul_gated(int dtype, const void *x, int rows, int inner, const void *w, int cols, int act, void *pre, void *h, void *scratch,
                               size_t scratch_bytes, void *stream) {
    if (int rc = gated::check(dtype, rows, inner, cols, act, "matmul_gated")) return rc;
    D8_REQUIRE(x && w && h, "matmul_gated: null tensor");
    (void)scratch, (void)scratch_bytes;
    gated::Args a;
    memset(&a, 0, sizeof(a));
    a.x = x, a.w = w, a.pre = pre, a.h = h, a.rows = rows, a.inner = inner, a.cols = cols, a.act = act;
    const int v = 16 / (int)dtype_bytes(dtype);
    a.vec_x = inner % v == 0 && ((size_t)x & 15) == 0, a.vec_w = cols % v == 0 && ((size_t)w & 15) == 0;
    const dim3 grid(ceil_div(cols, gated::BN), ceil_div(rows, gated::BM));
    D8_REQUIRE(grid.y < 65536u, "matmul_gated: too many rows");
    if (dtype == D8_FLOAT16) hipLaunchKernelGGL(gated::gated_tile_kernel<f16>, grid, dim3(256), 0, as_stream(stream), a);
    else hipLaunchKernelGGL(gated::gated_tile_kernel<float>, grid, dim3(256), 0, as_stream(stream), a);
    D8_LAUNCH_CHECK();
    return 0;
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
    a.vec_w = cols % v == 0 && (((size_t)pre | (size_t)dh) & 15) == 0;
    const long threads = (long)rows * ceil_div(cols, v);
    const dim3 grid((unsigned)((threads + 255) / 256 < 16384 ? (threads + 255) / 256 : 16384));
    if (dtype == D8_FLOAT16) hipLaunchKernelGGL(gated::gated_slope_kernel<f16>, grid, dim3(256), 0, as_stream(stream), a);
    else hipLaunchKernelGGL(gated::gated_slope_kernel<float>, grid, dim3(256), 0, as_stream(stream), a);
    D8_LAUNCH_CHECK();
    void *rest = scratch_bytes > own ? (char *)scratch + own : nullptr;
    return d8_matmul_grad_xy(dtype, x, dx, 1, rows, inner, w, dw, 1, inner, 2 * cols, scratch, overwrite, rest, scratch_bytes - own, stream);
}
