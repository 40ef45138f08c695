// Attention over packed sequences of different lengths, heads sharing keys and values, forward.
//
//   s = scale q k^T (query t of a sequence with nq queries and nk keys sees keys j <= t + nk - nq, or all),  o = softmax(s) v,
//   lse = log(sum exp s);  a row that sees nothing: o = 0, lse = -inf
//
// One pass over the keys with the running maximum and sum of the softmax (fp32).  A workgroup has 128 rows, each of its four waves
// 32 of them; the scores are computed transposed (keys x rows), so that a row's scores lie in one lane (and its partner 32 lanes on),
// maximum and sum are lane arithmetic, and the probabilities are the right operand of the product with the values where they are.
// In half the probabilities, at most 1 relative to the running maximum, are rounded to half for that product: an error of 2^-12 a
// term, which the terms' different signs and the division by a sum of the unrounded ones leave below the rounding of o itself.
#include "attention.h"

namespace d8 {
namespace attention {
namespace {

enum { ROWS = 128, KEYS = 32 };

template <class T, int DP>
__global__ __launch_bounds__(256) void attention_kernel(Args a) {
    typedef Type<T> M;
    typedef typename M::frag frag;
    constexpr int PITCH = pitch_of<DP, T>(), UNITS = DP / M::STEP, PIECES = DP / M::V;
    __shared__ __attribute__((aligned(16))) char tile_k[KEYS * PITCH], tile_v[KEYS * PITCH];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int hk = blockIdx.x % a.kv_heads;
    Span sp;
    int seq, tile;
    auto tiles_of = [&](const Span &s) { return (int)(((long)s.nq * a.group + ROWS - 1) / ROWS); };
    if (!locate(a, blockIdx.x / a.kv_heads, sp, seq, tile, tiles_of)) return;
    const int group = a.group, rows = sp.nq * group;
    tile = tiles_of(sp) - 1 - tile;  // the rows that see most keys first
    const int r = tile * ROWS + wave * 32 + (lane & 31);
    const int t = r / group, head = hk * group + r - t * group;
    const bool there = r < rows;
    const T *q = (const T *)a.q + (long)(sp.q0 + (there ? t : 0)) * a.ldq + (long)head * a.dim;
    frag qf[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) qf[u] = load_piece<T>(q, u * M::STEP + h * M::V, a.dim, there, a.vec);
    const int back = sp.nk - sp.nq;
    const int last = a.causal ? min(sp.nk - 1, t + back) : sp.nk - 1;  // last key that the lane's row sees
    const int t_end = (min(rows, (tile + 1) * ROWS) - 1) / group;
    const int end = a.causal ? min(sp.nk, t_end + back + 1) : sp.nk;
    const float c = a.scale * LOG2E;
    f32x16 acc[DP / 32];
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[b][e] = 0.f;
    float m = -INFINITY, l = 0.f;
    for (int j0 = 0; j0 < end; j0 += KEYS) {
        __syncthreads();
        for (int p = tid; p < KEYS * PIECES; p += 256) {
            const int row = p / PIECES, d = (p - row * PIECES) * M::V;
            const bool in = j0 + row < sp.nk;
            const long at = sp.k0 + (in ? j0 + row : 0);
            *(frag *)(tile_k + row * PITCH + d * (int)sizeof(T)) = load_piece<T>((const T *)a.k + at * a.ldk + (long)hk * a.dim, d, a.dim, in, a.vec);
            *(frag *)(tile_v + row * PITCH + d * (int)sizeof(T)) = load_piece<T>((const T *)a.v + at * a.ldv + (long)hk * a.dim, d, a.dim, in, a.vec);
        }
        __syncthreads();
        f32x16 s;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) M::mma(s, read_rows<T>(tile_k, PITCH, u, lane), qf[u]);
        float top = m;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int j = j0 + 8 * (e >> 2) + 4 * h + (e & 3);
            s[e] = j <= last ? s[e] * c : -INFINITY;
            top = fmaxf(top, s[e]);
        }
        top = fmaxf(top, __shfl_xor(top, 32));
        const float base = top == -INFINITY ? 0.f : top;
        const float keep = exp2f(m - base);
        m = top;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = exp2f(s[e] - base);
            sum += s[e];
        }
        l = l * keep + sum;
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) {
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[b][e] *= keep;
#pragma unroll
            for (int u = 0; u < KEYS / M::STEP; ++u) M::mma(acc[b], M::read_cols(tile_v, PITCH, u * M::STEP, b * 32, lane), M::pack(s, u));
        }
    }
    l += __shfl_xor(l, 32);
    if (!there) return;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    T *o = (T *)a.o + (long)(sp.q0 + t) * a.ldo + (long)head * a.dim;
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int d = b * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
            if (d < a.dim) o[d] = (T)(acc[b][e] * inv);
        }
    if (a.lse && h == 0) a.lse[(long)head * a.q_tokens + sp.q0 + t] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
}

template <class T>
int launch(const Args &a, hipStream_t stream) {
    const dim3 grid((unsigned)a.tiles * a.kv_heads);
    if (a.dim <= 32) hipLaunchKernelGGL((attention_kernel<T, 32>), grid, dim3(256), 0, stream, a);
    else if (a.dim <= 64) hipLaunchKernelGGL((attention_kernel<T, 64>), grid, dim3(256), 0, stream, a);
    else if (a.dim <= 128) hipLaunchKernelGGL((attention_kernel<T, 128>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((attention_kernel<T, 256>), grid, dim3(256), 0, stream, a);
    D8_LAUNCH_CHECK();
    return 0;
}

}  // namespace

int check(const Args &a, int dtype, const char *name) {
    if (dtype != D8_FLOAT16 && dtype != D8_FLOAT32) return fail(D8_ERR_DTYPE, "%s: type %d is not support", name, dtype);
    D8_REQUIRE(a.sequences >= 0 && a.q_tokens >= 0 && a.k_tokens >= 0, "%s: %d sequences, %d queries, %d keys", name, a.sequences, a.q_tokens, a.k_tokens);
    D8_REQUIRE(a.kv_heads >= 1 && a.heads >= a.kv_heads && a.heads % a.kv_heads == 0, "%s: %d heads cannot share the keys of %d", name, a.heads, a.kv_heads);
    D8_REQUIRE(a.dim >= 1 && a.dim <= MOST_DIM, "%s: a head has 1 to %d elements, not %d", name, (int)MOST_DIM, a.dim);
    const long qrow = (long)a.heads * a.dim, krow = (long)a.kv_heads * a.dim;
    D8_REQUIRE(a.ldq >= qrow && a.ldo >= qrow && a.ldk >= krow && a.ldv >= krow, "%s: rows of %ld and %ld elements do not fit their leading dimensions", name, qrow, krow);
    D8_REQUIRE((long)a.q_tokens * a.heads < (1L << 30) && a.k_tokens < (1 << 30), "%s: too many queries or keys", name);
    D8_REQUIRE(a.scale == a.scale, "%s: the scale is no number", name);
    return 0;
}

// whether every row of these tensors starts at a multiple of 16 bytes
bool in_pieces(int dtype, int dim, std::initializer_list<const void *> p, std::initializer_list<long> ld) {
    const int v = 16 / (int)dtype_bytes(dtype);
    if (dim % v) return false;
    for (const void *x : p)
        if ((size_t)x & 15) return false;
    for (long x : ld)
        if (x % v) return false;
    return true;
}

}  // namespace attention
}  // namespace d8

using namespace d8;

extern "C" size_t d8_attention_scratch_bytes(int dtype, int which, int sequences, int q_tokens, int k_tokens, int heads, int kv_heads, int dim, int causal) {
    (void)causal, (void)sequences, (void)k_tokens, (void)kv_heads, (void)dim;
    if ((dtype != D8_FLOAT16 && dtype != D8_FLOAT32) || q_tokens < 0 || heads < 1) return 0;
    return which == 1 ? attention::grad_scratch_bytes(q_tokens, heads) : 0;
}

extern "C" int d8_attention(int dtype, const void *q, long ldq, const void *k, long ldk, const void *v, long ldv, void *o, long ldo, float *lse,
                            const int *q_starts, const int *k_starts, int sequences, int q_tokens, int k_tokens, int heads, int kv_heads, int dim,
                            float scale, int causal, void *scratch, size_t scratch_bytes, void *stream) {
    attention::Args a;
    memset(&a, 0, sizeof(a));
    a.q = q, a.k = k, a.v = v, a.o = o, a.lse = lse, a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldo = ldo;
    a.q_starts = q_starts, a.k_starts = k_starts, a.sequences = sequences, a.q_tokens = q_tokens, a.k_tokens = k_tokens;
    a.heads = heads, a.kv_heads = kv_heads, a.dim = dim, a.scale = scale, a.causal = causal != 0;
    if (int rc = attention::check(a, dtype, "attention")) return rc;
    if (!sequences || !q_tokens) return 0;
    D8_REQUIRE(q && o && q_starts && k_starts && (!k_tokens || (k && v)), "attention: null tensor");
    (void)scratch, (void)scratch_bytes;
    a.group = heads / kv_heads;
    a.vec = attention::in_pieces(dtype, dim, {q, k, v}, {ldq, ldk, ldv});
    const long tiles = ((long)q_tokens * a.group + attention::ROWS - 1) / attention::ROWS + sequences;
    D8_REQUIRE(tiles * kv_heads < (1L << 31), "attention: too many sequences");
    a.tiles = (int)tiles;
    return dtype == D8_FLOAT16 ? attention::launch<f16>(a, as_stream(stream)) : attention::launch<float>(a, as_stream(stream));
}
