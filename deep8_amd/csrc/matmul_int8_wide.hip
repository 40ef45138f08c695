// The product in 8-bit integers of many rows and columns: the 256 x 256 tile loop of gemm_wide_kernel.h on the same bytes.  Two codes take the place
// of one half, so a step of 64 halves is one of 128 codes, a fragment of 16 x 32 halves one of 16 x 64 codes, and only the matrix
// instruction is another (v_mfma_i32_16x16x64_i8, twice the products in the same cycles, sums in int32).  The epilogue scales.  Bound by the matrix units and what power lets
// them do: 8192 x 4096 x 8192 in 210 to 234 us, 2.6 to 2.35 POP/s (as the clock is: the first of a row of calls, and many of them), where the library's product of the same bytes takes 246.
#include "gemm_wide_kernel.h"
#include "int8.h"

namespace d8 {
namespace wide {

struct Int8 : Shipped {};
template <>
__device__ __forceinline__ void mfma<Int8>(f32x4 &acc, const f16x8 &a, const f16x8 &b) {
    asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}
template <>
__device__ __forceinline__ void mfma_first<Int8>(f32x4 &acc, const f16x8 &a, const f16x8 &b) {
    asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, 0" : "=a"(acc) : "v"(a), "v"(b));
}

}  // namespace wide

namespace int8 {

struct WideArgs {
    Args a;
    int tilesM, tilesN, total;
    // the product that the tile loop knows, in units of two codes
    __device__ __forceinline__ wide::Launch product() const {
        wide::Launch L;
        wide::Product &p = L.p[0];
        p.A = (const f16 *)a.x, p.B = (const f16 *)a.w, p.C = nullptr, p.bias = nullptr, p.M = a.rows, p.N = a.cols, p.K = a.steps * (STEP / 2);
        p.lda = p.ldb = (int)(a.pitch / 2), p.ldc = 0, p.sA = p.sB = p.sC = 0, p.tilesM = tilesM, p.tilesN = tilesN, p.tiles = total;
        p.form = wide::FORM_NT, p.beta = 0.f, p.relu = 0;
        L.n = 1, L.total = total, L.rec = nullptr;
        return L;
    }
};

typedef wide::TileOperands<true, true> WideOperands;

// The operands of the tile at `w`, from arguments that the compiler takes for new ones: per tile, not once and kept.  Scalar registers are short, and
// one that is brought back from a vector register right before a load into LDS, which is asm, comes too late for it (the built code is tested for that).
__device__ __forceinline__ void wide_operands(WideOperands &T, const WideArgs &all, const wide::Where &w, int wave, int lane) {
    WideArgs a = all;
    asm volatile("" : "+s"(a.a.rows), "+s"(a.a.cols), "+s"(a.a.steps), "+s"(a.a.pitch), "+v"(lane));
    T.init<wide::Int8>(a.product().p[0], w, wave, lane);
}

// The eight columns of a row that a lane stores, of a wave's 128: half, eight side by side, 16 bytes; single, four and the four 64 further on, so that
// in either a store instruction has whole lines.
template <class T>
__device__ __forceinline__ int column(int l15, int e) {
    return sizeof(T) == 2 ? l15 * 8 + e : l15 * 4 + (e >> 2) * 64 + (e & 3);
}

// The scales of what a lane stores: its columns', and its 32 rows' (row 16 i + 4 t + lane / 16 of the wave's 128).
template <class T>
struct Scales {
    float w[8], x[32];
    __device__ __forceinline__ void load(const Args &a, const wide::Where &at, int wave, int lane) {
        const int n = at.n0 + (wave & 1) * 128, m = at.m0 + (wave >> 1) * 128 + (lane >> 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = a.w_scales[n + column<T>(lane & 15, e)];
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = a.x_scales[m + e * 4];
    }
    // Used here, so that the compiler waits for them here and not behind loads that it does not see (they come back in order).
    __device__ __forceinline__ void arrive() {
#pragma unroll
        for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(w[e]));
#pragma unroll
        for (int e = 0; e < 32; ++e) asm volatile("" : "+v"(x[e]));
    }
};

// A finished tile on its way out, as wide::store_tile.  INTERIOR: every lane stores all its 32 pieces (single precision: 64).  Else element by element, 16
// lanes along a row.
template <class T, bool INTERIOR>
__device__ __forceinline__ void store_scaled(const Args &a, const wide::Where &w, const Scales<T> &by, float *patch, int wave, int lane, f32x4 (&acc)[8][8]) {
    asm volatile("" : "+v"(lane));
    const int wm = wave >> 1, wn = wave & 1, l15 = lane & 15, l4 = lane >> 4;
    const int n = w.n0 + wn * 128;
    unsigned wr[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) wr[q] = (unsigned)(size_t)WIDE_LDS(float, patch) + 4u * ((4 * l4) * 128 + ((q ^ l4) * 16 + l15));
    float along[8];  // scales of columns lane % 16 + 16 k
#pragma unroll
    for (int k = 0; k < 8; ++k) along[k] = INTERIOR ? 0.f : a.w_scales[n + l15 + k * 16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        wide::write_slab<0>(wr, acc[i]);
        if (INTERIOR) {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int row = t * 4 + l4, m = w.m0 + wm * 128 + i * 16 + row;
                i32x4 part[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) part[h] = *(const i32x4 *)(patch + row * 128 + (column<T>(l15, 4 * h) ^ (t * 16)));
                T out[8];
                scale_row<T, 8>(__builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7), by.x[i * 4 + t], by.w, out);
                typedef T piece __attribute__((ext_vector_type(16 / sizeof(T))));
                T *z = (T *)a.z + (long)m * a.ldz + n;
#pragma unroll
                for (int e = 0; e < 8; e += 16 / sizeof(T)) __builtin_nontemporal_store(*(const piece *)(out + e), (piece *)(z + column<T>(l15, e)));
            }
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int row = t * 4 + l4, m = w.m0 + wm * 128 + i * 16 + row;
                int sums[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) sums[k] = __float_as_int(patch[row * 128 + ((k * 16 + l15) ^ (t * 16))]);
                T *z = (T *)a.z + (long)m * a.ldz + n + l15, out[8];
                scale_row<T, 8>(sums, by.x[i * 4 + t], along, out);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (m >= w.m_own && n + l15 + k * 16 >= w.n_own) z[k * 16] = out[k];
            }
        }
    }
}

template <class T>
__global__ __launch_bounds__(256) void int8_wide_kernel(WideArgs wa) {
    using namespace wide;
    __shared__ __attribute__((aligned(1024))) char lds[LDS_BYTES];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    float *patch = (float *)(lds + 2 * STAGE_BYTES) + wave * (16 * 128);
    const unsigned wave_base = (unsigned)(size_t)WIDE_LDS(const char, lds) + wave * 1024;
    f32x4 acc[8][8];
    int idx = blockIdx.x;
    Where cur = locate(wa.product(), idx);
    {
        WideOperands T_;
        wide_operands(T_, wa, cur, wave, lane);
        T_.issue_first_steps(wave_base);
    }
    __builtin_amdgcn_s_waitcnt(0x4f70);  // vmcnt(16): the first stage has landed
    __syncthreads();
    for (;;) {
        const int nidx = idx + gridDim.x;
        const bool more = nidx < wa.total;
        const Where nxt = more ? locate(wa.product(), nidx) : cur;
        Scales<T> by;  // on their way during the loop
        by.load(wa.a, cur, wave, lane);
        {
            WideOperands T_;
            wide_operands(T_, wa, cur, wave, lane);
            k_loop<Int8, true, true>(T_, lds, wave_base, acc);
        }
        by.arrive();
        if (more) {  // the next tile's first two steps set out before this tile's epilogue: 32 loads a wave
            WideOperands T_;
            wide_operands(T_, wa, nxt, wave, lane);
            T_.issue_first_steps(wave_base);
        }
        const bool interior = wa.a.vec && cur.m0 == cur.m_own && cur.n0 == cur.n_own;
        if (interior) store_scaled<T, true>(wa.a, cur, by, patch, wave, lane, acc);
        else store_scaled<T, false>(wa.a, cur, by, patch, wave, lane, acc);
        if (!more) break;
        // an interior tile's epilogue has issued 32 stores or more after those 32 loads, and vector-memory instructions complete in order: at
        // most 32 outstanding, and the loads have landed
        if (interior) __builtin_amdgcn_s_waitcnt(0x8f70);
        else __builtin_amdgcn_s_waitcnt(0x0f70);
        __syncthreads();
        cur = nxt, idx = nidx;
    }
}

// Where these tiles are estimated to be through before those of 64 x 64: a step of 128 codes takes 1.05 us, a call 8 us beside them; the others go at 1000 TOP/s
// after 5 us.  (us here / there: 1024 x 4096 x 4096 41 / 39, 2048 x 4096 x 4096 43 / 67, 4096 x 1024 x 4096 21 / 43, 2048 x 2048 x 2048 25 / 20, 3000 x 256 x 1024 14.5 / 6.4.)
bool wide_eligible(const Args &a) {
    if (a.rows < 256 || a.cols < 256) return false;
    if (a.rows * a.pitch >= (1L << 31) || a.cols * a.pitch >= (1L << 31)) return false;
    const long tiles = (long)ceil_div(a.rows, 256) * ceil_div(a.cols, 256), cus = cu_count();
    const float here = 8.f + 1.05f * a.steps * ((tiles + cus - 1) / cus), there = 5.f + 2e-9f * a.rows * a.cols * a.steps * STEP;
    return here < there && tiles < (1L << 30);
}

template <class T>
int wide_launch(const Args &a, hipStream_t stream) {
    WideArgs w;
    w.a = a;
    w.a.vec = a.cols % 8 == 0 && a.ldz % 8 == 0 && ((size_t)a.z & 15) == 0;
    w.tilesM = ceil_div(a.rows, 256), w.tilesN = ceil_div(a.cols, 256), w.total = w.tilesM * w.tilesN;
    const int cus = cu_count(), grid = w.total <= cus ? w.total : cus >= 8 ? cus - cus % 8 : cus;
    hipLaunchKernelGGL(int8_wide_kernel<T>, dim3(grid), dim3(256), 0, stream, w);
    D8_LAUNCH_CHECK();
    return 0;
}
template int wide_launch<f16>(const Args &, hipStream_t);
template int wide_launch<float>(const Args &, hipStream_t);

}  // namespace int8
}  // namespace d8
