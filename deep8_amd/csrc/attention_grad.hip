// The way back through attention (attention.hip).  With p = exp(s - lse), recomputed from q, k and the forward pass's lse:
//
//   dv = p^T do,  dp = do v^T,  ds = p (dp - delta) with delta = rowsum(do o) = rowsum(p dp),  dq = scale ds k,  dk = scale ds^T q
//
// Three launches: delta of every row; dk and dv, a workgroup for 128 keys that walks the rows that see them (those of all heads that
// share the keys, so that the sums over shared heads stay in its registers); dq, a workgroup for 128 rows that walks the keys.  The
// scores are computed twice, seven products for the five that the formulas have, and in return no two workgroups add to one
// place: no atomics, the same bits every time.
//
// In half, p and ds are rounded to half for the products that follow.  p is scaled by 2^15 (it is at most 1) and ds by a power of two
// that a bound on it allows, |dp - delta| <= 2 max |do_i| max |v_j| over all rows, so that small probabilities of long rows keep
// their bits: a probability of 10^-5 would otherwise be a subnormal half.  The scales are taken out again in fp32.
#include "attention.h"

namespace d8 {
namespace attention {
namespace {

enum { KEYS = 128, ROWS = 128, TILE = 32 };
enum { NORM_GROUPS = 512 };  // workgroups of the first launch: entries of each list of norms
constexpr float P_SHIFT = 15.f;

template <class T>
constexpr bool scaled() { return sizeof(T) == 2; }

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

// delta[head][token] = sum of do o; a wave has a row.  In half also the largest squared norms of the rows of do and of v.
template <class T>
__global__ __launch_bounds__(256) void attention_delta_kernel(Args a) {
    __shared__ float most[2][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float top_do = 0.f, top_v = 0.f;
    const long rows = (long)a.q_tokens * a.heads;
    for (long r = (long)blockIdx.x * 4 + wave; r < rows; r += (long)gridDim.x * 4) {
        const long t = r / a.heads;
        const int head = (int)(r - t * a.heads);
        const T *g = (const T *)a.dout + t * a.lddo + (long)head * a.dim, *o = (const T *)a.o + t * a.ldo + (long)head * a.dim;
        float dot = 0.f, sq = 0.f;
        for (int d = lane; d < a.dim; d += 64) {
            const float x = (float)g[d];
            dot += x * (float)o[d], sq += x * x;
        }
        dot = wave_sum(dot);
        if (lane == 0) a.delta[(long)head * a.q_tokens + t] = dot;
        if (scaled<T>()) top_do = fmaxf(top_do, wave_sum(sq));
    }
    if (!scaled<T>()) return;
    const long krows = (long)a.k_tokens * a.kv_heads;
    for (long r = (long)blockIdx.x * 4 + wave; r < krows; r += (long)gridDim.x * 4) {
        const long t = r / a.kv_heads;
        const T *v = (const T *)a.v + t * a.ldv + (r - t * a.kv_heads) * a.dim;
        float sq = 0.f;
        for (int d = lane; d < a.dim; d += 64) sq += (float)v[d] * (float)v[d];
        top_v = fmaxf(top_v, wave_sum(sq));
    }
    if (lane == 0) most[0][wave] = top_do, most[1][wave] = top_v;
    __syncthreads();
    if (threadIdx.x < 2) {
        const float *m = most[threadIdx.x];
        a.norms[threadIdx.x * NORM_GROUPS + blockIdx.x] = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
    }
}

// 2^-e with |dp - delta| < 2^e for every row and key of the call (1 where there is no such bound); every wave computes it
template <class T>
__device__ __forceinline__ float ds_scale(const Args &a) {
    if (!scaled<T>()) return 1.f;
    const int lane = threadIdx.x & 63;
    float d = 0.f, v = 0.f;
    for (int i = lane; i < NORM_GROUPS; i += 64) d = fmaxf(d, a.norms[i]), v = fmaxf(v, a.norms[NORM_GROUPS + i]);
    const float bound = 2.f * sqrtf(wave_max(d)) * sqrtf(wave_max(v));
    if (!(bound > 0.f) || bound > 3e38f) return 1.f;
    return exp2f(-(float)(ilogbf(bound) + 1));
}

// dk and dv
template <class T, int DP>
__global__ __launch_bounds__(256) void attention_grad_kv_kernel(Args a) {
    typedef Type<T> M;
    typedef typename M::frag frag;
    constexpr int PITCH = pitch_of<DP, T>(), UNITS = DP / M::STEP, PIECES = DP / M::V;
    __shared__ __attribute__((aligned(16))) char tile_q[TILE * PITCH], tile_g[TILE * PITCH];
    __shared__ __attribute__((aligned(16))) float row_lse[TILE], row_delta[TILE];
    __shared__ __attribute__((aligned(16))) int row_last[TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int hk = blockIdx.x % a.kv_heads;
    Span sp;
    int seq, block;
    if (!locate(a, blockIdx.x / a.kv_heads, sp, seq, block, [](const Span &s) { return (s.nk + KEYS - 1) / KEYS; })) return;
    const int group = a.group, rows = sp.nq * group, back = sp.nk - sp.nq;
    const float mult = ds_scale<T>(a), c = a.scale * LOG2E, shift = scaled<T>() ? P_SHIFT : 0.f;
    const int j = block * KEYS + wave * 32 + (lane & 31);  // the lane's key
    const bool there = j < sp.nk;
    const long key = sp.k0 + (there ? j : 0);
    frag kf[UNITS], vf[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        kf[u] = load_piece<T>((const T *)a.k + key * a.ldk + (long)hk * a.dim, u * M::STEP + h * M::V, a.dim, there, a.vec);
        vf[u] = load_piece<T>((const T *)a.v + key * a.ldv + (long)hk * a.dim, u * M::STEP + h * M::V, a.dim, there, a.vec);
    }
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[b][e] = dv[b][e] = 0.f;
    // the first row that sees a key of the block (its query is the block's first key less nk - nq)
    const long first = a.causal ? (long)max(0, block * KEYS - back) * group : 0;
    for (long r0 = first / TILE * TILE; r0 < rows; r0 += TILE) {
        __syncthreads();
        for (int p = tid; p < TILE * PIECES; p += 256) {
            const int row = p / PIECES, d = (p - row * PIECES) * M::V;
            const int r = (int)r0 + row;
            const bool in = r < rows;
            const int t = in ? r / group : 0, head = hk * group + (in ? r - t * group : 0);
            *(frag *)(tile_q + row * PITCH + d * (int)sizeof(T)) = load_piece<T>((const T *)a.q + (long)(sp.q0 + t) * a.ldq + (long)head * a.dim, d, a.dim, in, a.vec);
            *(frag *)(tile_g + row * PITCH + d * (int)sizeof(T)) = load_piece<T>((const T *)a.dout + (long)(sp.q0 + t) * a.lddo + (long)head * a.dim, d, a.dim, in, a.vec);
        }
        if (tid < TILE) {
            const int r = (int)r0 + tid;
            const bool in = r < rows;
            const int t = in ? r / group : 0, head = hk * group + (in ? r - t * group : 0);
            const long at = (long)head * a.q_tokens + sp.q0 + t;
            row_lse[tid] = in ? a.lse[at] * LOG2E - shift : INFINITY;
            row_delta[tid] = in ? a.delta[at] : 0.f;
            row_last[tid] = !in ? -1 : a.causal ? t + back : sp.nk - 1;
        }
        __syncthreads();
        f32x16 s, w;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = w[e] = 0.f;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            M::mma(s, read_rows<T>(tile_q, PITCH, u, lane), kf[u]);
            M::mma(w, read_rows<T>(tile_g, PITCH, u, lane), vf[u]);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int row = 8 * (e >> 2) + 4 * h + (e & 3);
            const bool seen = j <= row_last[row] && there;
            s[e] = seen ? exp2f(s[e] * c - row_lse[row]) : 0.f;
            w[e] = seen ? s[e] * ((w[e] - row_delta[row]) * mult) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < TILE / M::STEP; ++u) {
            const frag p = M::pack(s, u), d = M::pack(w, u);
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) {
                M::mma(dv[b], M::read_cols(tile_g, PITCH, u * M::STEP, b * 32, lane), p);
                M::mma(dk[b], M::read_cols(tile_q, PITCH, u * M::STEP, b * 32, lane), d);
            }
        }
    }
    if (!there) return;
    const float unshift = exp2f(-shift), by = a.scale * unshift / mult;
    T *pk = (T *)a.dk + key * a.lddk + (long)hk * a.dim, *pv = (T *)a.dv + key * a.lddv + (long)hk * a.dim;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int d = b * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
            if (d >= a.dim) continue;
            const float x = dk[b][e] * by, y = dv[b][e] * unshift;
            pk[d] = (T)((a.overwrite & 2) ? x : x + (float)pk[d]);
            pv[d] = (T)((a.overwrite & 4) ? y : y + (float)pv[d]);
        }
}

// dq
template <class T, int DP>
__global__ __launch_bounds__(256) void attention_grad_q_kernel(Args a) {
    typedef Type<T> M;
    typedef typename M::frag frag;
    constexpr int PITCH = pitch_of<DP, T>(), UNITS = DP / M::STEP, PIECES = DP / M::V;
    __shared__ __attribute__((aligned(16))) char tile_k[TILE * PITCH], tile_v[TILE * PITCH];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int hk = blockIdx.x % a.kv_heads;
    Span sp;
    int seq, tile;
    auto tiles_of = [&](const Span &s) { return (int)(((long)s.nq * a.group + ROWS - 1) / ROWS); };
    if (!locate(a, blockIdx.x / a.kv_heads, sp, seq, tile, tiles_of)) return;
    const int group = a.group, rows = sp.nq * group, back = sp.nk - sp.nq;
    tile = tiles_of(sp) - 1 - tile;
    const float mult = ds_scale<T>(a), c = a.scale * LOG2E, shift = scaled<T>() ? P_SHIFT : 0.f;
    const int r = tile * ROWS + wave * 32 + (lane & 31);
    const bool there = r < rows;
    const int t = there ? r / group : 0, head = hk * group + (there ? r - t * group : 0);
    frag qf[UNITS], gf[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        qf[u] = load_piece<T>((const T *)a.q + (long)(sp.q0 + t) * a.ldq + (long)head * a.dim, u * M::STEP + h * M::V, a.dim, there, a.vec);
        gf[u] = load_piece<T>((const T *)a.dout + (long)(sp.q0 + t) * a.lddo + (long)head * a.dim, u * M::STEP + h * M::V, a.dim, there, a.vec);
    }
    const long at = (long)head * a.q_tokens + sp.q0 + t;
    const float lse = there ? a.lse[at] * LOG2E - shift : INFINITY, delta = there ? a.delta[at] : 0.f;
    const int last = !there ? -1 : a.causal ? min(sp.nk - 1, t + back) : sp.nk - 1;
    const int t_end = (min(rows, (tile + 1) * ROWS) - 1) / group;
    const int end = a.causal ? min(sp.nk, t_end + back + 1) : sp.nk;
    f32x16 dq[DP / 32];
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) dq[b][e] = 0.f;
    for (int j0 = 0; j0 < end; j0 += TILE) {
        __syncthreads();
        for (int p = tid; p < TILE * PIECES; p += 256) {
            const int row = p / PIECES, d = (p - row * PIECES) * M::V;
            const bool in = j0 + row < sp.nk;
            const long k = sp.k0 + (in ? j0 + row : 0);
            *(frag *)(tile_k + row * PITCH + d * (int)sizeof(T)) = load_piece<T>((const T *)a.k + k * a.ldk + (long)hk * a.dim, d, a.dim, in, a.vec);
            *(frag *)(tile_v + row * PITCH + d * (int)sizeof(T)) = load_piece<T>((const T *)a.v + k * a.ldv + (long)hk * a.dim, d, a.dim, in, a.vec);
        }
        __syncthreads();
        f32x16 s, w;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = w[e] = 0.f;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            M::mma(s, read_rows<T>(tile_k, PITCH, u, lane), qf[u]);
            M::mma(w, read_rows<T>(tile_v, PITCH, u, lane), gf[u]);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const bool seen = j0 + 8 * (e >> 2) + 4 * h + (e & 3) <= last;
            w[e] = seen ? exp2f(s[e] * c - lse) * ((w[e] - delta) * mult) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < TILE / M::STEP; ++u) {
            const frag d = M::pack(w, u);
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) M::mma(dq[b], M::read_cols(tile_k, PITCH, u * M::STEP, b * 32, lane), d);
        }
    }
    if (!there) return;
    const float by = a.scale * exp2f(-shift) / mult;
    T *p = (T *)a.dq + (long)(sp.q0 + t) * a.lddq + (long)head * a.dim;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int d = b * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
            if (d >= a.dim) continue;
            const float x = dq[b][e] * by;
            p[d] = (T)((a.overwrite & 1) ? x : x + (float)p[d]);
        }
}

template <class T, int DP>
int launch_dim(const Args &a, int key_blocks, hipStream_t stream) {
    if (key_blocks) {
        hipLaunchKernelGGL((attention_grad_kv_kernel<T, DP>), dim3((unsigned)key_blocks * a.kv_heads), dim3(256), 0, stream, a);
        D8_LAUNCH_CHECK();
    }
    if (a.tiles) {
        hipLaunchKernelGGL((attention_grad_q_kernel<T, DP>), dim3((unsigned)a.tiles * a.kv_heads), dim3(256), 0, stream, a);
        D8_LAUNCH_CHECK();
    }
    return 0;
}

template <class T>
int launch(const Args &a, int key_blocks, hipStream_t stream) {
    hipLaunchKernelGGL(attention_delta_kernel<T>, dim3(NORM_GROUPS), dim3(256), 0, stream, a);
    D8_LAUNCH_CHECK();
    if (a.dim <= 32) return launch_dim<T, 32>(a, key_blocks, stream);
    if (a.dim <= 64) return launch_dim<T, 64>(a, key_blocks, stream);
    if (a.dim <= 128) return launch_dim<T, 128>(a, key_blocks, stream);
    return launch_dim<T, 256>(a, key_blocks, stream);
}

}  // namespace

size_t grad_scratch_bytes(int q_tokens, int heads) {
    return sizeof(float) * (2 * NORM_GROUPS + (size_t)q_tokens * heads);
}

}  // namespace attention
}  // namespace d8

using namespace d8;

extern "C" int d8_attention_grad(int dtype, const void *q, long ldq, const void *k, long ldk, const void *v, long ldv, const void *o, long ldo,
                                 const float *lse, const void *dout, long lddo, void *dq, long lddq, void *dk, long lddk, void *dv, long lddv,
                                 const int *q_starts, const int *k_starts, int sequences, int q_tokens, int k_tokens, int heads, int kv_heads,
                                 int dim, float scale, int causal, int overwrite, void *scratch, size_t scratch_bytes, void *stream) {
    attention::Args a;
    memset(&a, 0, sizeof(a));
    a.q = q, a.k = k, a.v = v, a.o = (void *)o, a.lse = (float *)lse, a.dout = dout, a.dq = dq, a.dk = dk, a.dv = dv;
    a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldo = ldo, a.lddo = lddo, a.lddq = lddq, a.lddk = lddk, a.lddv = lddv;
    a.q_starts = q_starts, a.k_starts = k_starts, a.sequences = sequences, a.q_tokens = q_tokens, a.k_tokens = k_tokens;
    a.heads = heads, a.kv_heads = kv_heads, a.dim = dim, a.scale = scale, a.causal = causal != 0, a.overwrite = overwrite;
    if (int rc = attention::check(a, dtype, "attention_grad")) return rc;
    const long qrow = (long)heads * dim, krow = (long)kv_heads * dim;
    D8_REQUIRE(lddo >= qrow && lddq >= qrow && lddk >= krow && lddv >= krow, "attention_grad: rows of %ld and %ld elements do not fit their leading dimensions", qrow, krow);
    if (!sequences || (!q_tokens && !k_tokens)) return 0;
    D8_REQUIRE(q_starts && k_starts && (!q_tokens || (q && o && lse && dout && dq)) && (!k_tokens || (k && v && dk && dv)), "attention_grad: null tensor");
    const size_t need = attention::grad_scratch_bytes(q_tokens, heads);
    D8_REQUIRE(scratch && scratch_bytes >= need && ((size_t)scratch & 15) == 0, "attention_grad: 16-byte aligned scratch of %zu bytes is needed, not %zu", need, scratch_bytes);
    a.norms = (float *)scratch, a.delta = a.norms + 2 * attention::NORM_GROUPS;
    a.group = heads / kv_heads;
    a.vec = attention::in_pieces(dtype, dim, {q, k, v, dout}, {ldq, ldk, ldv, lddo});
    const long tiles = q_tokens ? ((long)q_tokens * a.group + attention::ROWS - 1) / attention::ROWS + sequences : 0;
    const long blocks = k_tokens ? ((long)k_tokens + attention::KEYS - 1) / attention::KEYS + sequences : 0;
    D8_REQUIRE((tiles + blocks) * kv_heads < (1L << 31), "attention_grad: too many sequences");
    a.tiles = (int)tiles;
    return dtype == D8_FLOAT16 ? attention::launch<f16>(a, (int)blocks, as_stream(stream)) : attention::launch<float>(a, (int)blocks, as_stream(stream));
}
