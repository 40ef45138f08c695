// The way back through attention (attention.hip).  With p = exp(s - lse), recomputed from q, k and the forward pass's lse:
//
//   dv = p^T do,  dp = do v^T,  ds = p (dp - delta) with delta = rowsum(do o) = rowsum(p dp),  dq = scale ds k,  dk = scale ds^T q
//
// Three launches: delta of every row; dq, a workgroup for some rows that walks the keys; dk and dv, a workgroup for some keys that walks
// the rows that see them (those of all heads that share the keys, so that the sums over shared heads stay in its registers).  The
// scores are computed twice, seven products for the five that the formulas have, and in return no two workgroups add to one
// place: no atomics, the same bits every time.
//
// In half, p and ds are rounded to half for the products that follow.  p is scaled by 2^15 (it is at most 1) and ds by a power of two
// that a bound on it allows, so that small probabilities of long rows keep their bits: a probability of 10^-5 would otherwise be a
// subnormal half.  The bound is one of what meets in a sum: for dq |dp - delta| <= 2 |do_i| max |v_j| of the row's own and the keys that its
// tile sees, for dk max |do_i| max |v_j| + max |delta_i| of a workgroup's rows and keys.  Rows elsewhere do not matter, and rows that are
// no number leave the bound alone: their own results are no number, the others keep their bits.  The scales are taken out again in
// fp32, before sums of several workgroups meet.
#include "attention.h"

namespace d8 {
namespace attention {
namespace {

enum { TILE = 32 };
enum { ROW_GRAIN = 512 };    // rows of a chunk are a multiple of this
enum { DELTA_GROUPS = 512 }; // workgroups of the first launch
constexpr float P_SHIFT = 15.f;

template <class T>
constexpr bool scaled() { return sizeof(T) == 2; }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

// 0 where it is not finite
__device__ __forceinline__ float finite(float v) { return fabsf(v) <= 3.4e38f ? v : 0.f; }

// delta = sum of do o of each row; a group of lanes has a row, 16 bytes a lane.  In half also the norms of the rows of do and of v.
// Bound by bytes: 56 MB (6144 tokens, 16 + 4 heads of 128 halves) in 20 us; four rows' loads at once took 2 us off that
// and added as much to small calls.
template <class T>
__global__ __launch_bounds__(256) void attention_delta_kernel(Args a, int lanes) {
    typedef typename Type<T>::frag frag;
    constexpr int V = Type<T>::V;
    const int l = threadIdx.x & (lanes - 1);
    const long step = (long)gridDim.x * 256 / lanes, mine = ((long)blockIdx.x * 256 + threadIdx.x) / lanes;
    const long rows = (long)a.q_tokens * a.heads;
    for (long r = mine; r < rows; r += step) {
        const long t = r / a.heads;
        const int head = (int)(r - t * a.heads);
        const frag g = load_piece<T>((const T *)a.dout + t * a.lddo + (long)head * a.dim, l * V, a.dim, true, a.vec);
        const frag o = load_piece<T>((const T *)a.o + t * a.ldo + (long)head * a.dim, l * V, a.dim, true, a.vec);
        float dot = 0.f, sq = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) dot += (float)g[e] * (float)o[e], sq += (float)g[e] * (float)g[e];
        for (int d = 1; d < lanes; d <<= 1) {
            dot += __shfl_xor(dot, d);
            if (scaled<T>()) sq += __shfl_xor(sq, d);
        }
        if (l == 0) {
            a.delta[(long)head * a.q_tokens + t] = dot;
            if (scaled<T>()) a.norms[(long)head * a.q_tokens + t] = finite(sqrtf(sq));
        }
    }
    if (!scaled<T>()) return;
    const long krows = (long)a.k_tokens * a.kv_heads;
    for (long r = mine; r < krows; r += step) {
        const long t = r / a.kv_heads;
        const int head = (int)(r - t * a.kv_heads);
        const frag v = load_piece<T>((const T *)a.v + t * a.ldv + (long)head * a.dim, l * V, a.dim, true, a.vec);
        float sq = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) sq += (float)v[e] * (float)v[e];
        for (int d = 1; d < lanes; d <<= 1) sq += __shfl_xor(sq, d);
        if (l == 0) a.v_norms[(long)head * a.k_tokens + t] = finite(sqrtf(sq));
    }
}

// 2^-e with bound < 2^e (1 where there is nothing to bound); half: p 2^15 of at most 1 times what is bounded stays below 2^15
__device__ __forceinline__ float scale_for(float bound) { return bound > 0.f ? exp2f(-(float)(ilogbf(bound) + 1)) : 1.f; }

// the largest of each wave's values, for all of the workgroup (through LDS; every thread takes part)
template <int N>
__device__ __forceinline__ void group_max(float (&v)[N]) {
    __shared__ float most[N][4];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = wave_max(v[i]);
        if ((threadIdx.x & 63) == 0) most[i][threadIdx.x >> 6] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = fmaxf(fmaxf(most[i][0], most[i][1]), fmaxf(most[i][2], most[i][3]));
}

// half: the largest norm of the rows of v of keys 0 .. n - 1 of a sequence
template <class T>
__device__ __forceinline__ float largest_v(const Args &a, const Span &sp, int hk, int n) {
    if (!scaled<T>()) return 0.f;
    const float *from = a.v_norms + (long)hk * a.k_tokens + sp.k0;
    float v[1] = {0.f};
#pragma unroll 4
    for (int j = threadIdx.x; j < n; j += 256) v[0] = fmaxf(v[0], from[j]);
    group_max(v);
    return v[0];
}

// What a row's ds is scaled by in the sums of dq.
template <class T>
__device__ __forceinline__ float row_scale(float norm, float v) { return scaled<T>() ? scale_for(2.f * norm * v) : 1.f; }

// ... in the sums of dk of keys j0 .. j0 + n - 1 over all heads' rows of queries t0 .. t1 - 1 of a sequence
template <class T>
__device__ __forceinline__ float keys_scale(const Args &a, const Span &sp, int hk, int j0, int n, int t0, int t1) {
    if (!scaled<T>()) return 1.f;
    float m[3] = {0.f, 0.f, 0.f};  // norms of do, delta, norms of v
    const long first = (long)hk * a.group * a.q_tokens + sp.q0 + t0;
    const int tokens = max(t1 - t0, 1), all = (t1 - t0) * a.group;
#pragma unroll 4
    for (int i = threadIdx.x; i < all; i += 256) {
        const int g = (unsigned)i / (unsigned)tokens;
        const long at = first + (long)g * a.q_tokens + (i - g * tokens);
        m[0] = fmaxf(m[0], a.norms[at]), m[1] = fmaxf(m[1], fabsf(finite(a.delta[at])));
    }
    const int j = j0 + (int)threadIdx.x;
    if ((int)threadIdx.x < n && j < sp.nk) m[2] = a.v_norms[(long)hk * a.k_tokens + sp.k0 + j];
    group_max(m);
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, scale_for(m[0] * m[2] + m[1]))));
}

enum { KEYS = 128, ROWS = 128 };  // of a workgroup of the two kernels for tensors that cannot be moved in 16-byte pieces

// dk and dv
template <class T, int DP>
__global__ __launch_bounds__(256) void attention_grad_kv_any_kernel(Args a) {
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
    const int t_first = a.causal ? max(0, block * KEYS - back) : 0;  // the first query that sees a key of the block
    const float mult = keys_scale<T>(a, sp, hk, block * KEYS, KEYS, min(t_first, sp.nq), sp.nq), c = a.scale * LOG2E, shift = scaled<T>() ? P_SHIFT : 0.f;
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
    const long first = (long)t_first * group;
    for (long r0 = first / TILE * TILE; r0 < rows; r0 += TILE) {
        __syncthreads();
        for (int p = tid; p < TILE * PIECES; p += 256) {
            const int row = p / PIECES, d = (p - row * PIECES) * M::V;
            const int r = (int)r0 + row;
            const bool in = r < rows;
            const int t = in ? query_of(a, r) : 0, head = hk * group + (in ? r - t * group : 0);
            *(frag *)(tile_q + row * PITCH + d * (int)sizeof(T)) = load_piece<T>((const T *)a.q + (long)(sp.q0 + t) * a.ldq + (long)head * a.dim, d, a.dim, in, a.vec);
            *(frag *)(tile_g + row * PITCH + d * (int)sizeof(T)) = load_piece<T>((const T *)a.dout + (long)(sp.q0 + t) * a.lddo + (long)head * a.dim, d, a.dim, in, a.vec);
        }
        if (tid < TILE) {
            const int r = (int)r0 + tid;
            const bool in = r < rows;
            const int t = in ? query_of(a, r) : 0, head = hk * group + (in ? r - t * group : 0);
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
__global__ __launch_bounds__(256) void attention_grad_q_any_kernel(Args a) {
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
    const float c = a.scale * LOG2E, shift = scaled<T>() ? P_SHIFT : 0.f;
    const int r = tile * ROWS + wave * 32 + (lane & 31);
    const bool there = r < rows;
    const int t = there ? query_of(a, r) : 0, head = hk * group + (there ? r - t * group : 0);
    frag qf[UNITS], gf[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        qf[u] = load_piece<T>((const T *)a.q + (long)(sp.q0 + t) * a.ldq + (long)head * a.dim, u * M::STEP + h * M::V, a.dim, there, a.vec);
        gf[u] = load_piece<T>((const T *)a.dout + (long)(sp.q0 + t) * a.lddo + (long)head * a.dim, u * M::STEP + h * M::V, a.dim, there, a.vec);
    }
    const long at = (long)head * a.q_tokens + sp.q0 + t;
    const float lse = there ? a.lse[at] * LOG2E - shift : INFINITY, delta = there ? a.delta[at] : 0.f, norm = scaled<T>() && there ? a.norms[at] : 0.f;
    const int last = !there ? -1 : a.causal ? min(sp.nk - 1, t + back) : sp.nk - 1;
    const int t_end = query_of(a, min(rows, (tile + 1) * ROWS) - 1);
    const int end = a.causal ? min(sp.nk, t_end + back + 1) : sp.nk;
    const float mult = row_scale<T>(norm, largest_v<T>(a, sp, hk, end));
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

// a lane's column of sums (32 b + 8 (e / 4) + 4 h + e % 4) times `by`, over or onto four elements at a time
template <class T, int DP>
__device__ __forceinline__ void store_sums(T *to, const f32x16 (&x)[DP / 32], float by, int dim, int h, bool overwrite) {
    typedef T four __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int d = n * 32 + 2 * e + 4 * h;
            if (d >= dim) continue;
            four out;
            if (overwrite) {
#pragma unroll
                for (int i = 0; i < 4; ++i) out[i] = (T)(x[n][e + i] * by);
            } else {
                const four old = *(const four *)(to + d);
#pragma unroll
                for (int i = 0; i < 4; ++i) out[i] = (T)(x[n][e + i] * by + (float)old[i]);
            }
            *(four *)(to + d) = out;
        }
}

// The same two for tensors whose rows can be moved in 16-byte pieces: tiles straight into one of two stages of LDS, the next while this one is
// worked on.  A wave has 32 keys (rows) of its own, whose fragments and sums stay in registers.  SPLIT = 1: four waves, 128 keys
// (rows) a workgroup, each walks every tile; SPLIT = 2, where that would leave compute units idle: 64, two waves have the same
// 32 and take every other tile, and their sums are joined through LDS at the end.  Half, causal, sequences of 2010, 1461 and 2673, 16 + 4 heads of
// 128: dk and dv 191 to 214 us + 20 for the join (four products, 570 TFLOP/s at the least time: two waves of a SIMD with every register taken wait for
// LDS and barriers, at 2.36 GHz), dq 110 to 117 us (three, 740 TFLOP/s).  Single, 2048 tokens in four sequences, 8 heads of 64: 83 and 63 us (52 TFLOP/s).
template <class T, int DP, int SPLIT>
struct Shape {
    static constexpr int PB = row_bytes<T, DP>(), OWN = 128 / SPLIT, BLOCKS = PB <= 256 || SPLIT == 2 ? 2 : 1;
    static constexpr int KB = 32 * BLOCKS, TILE_BYTES = KB * PB, LOADS = TILE_BYTES / 1024 / 4;
    static constexpr int OCCUPANCY = DP * (int)sizeof(T) <= 256 ? 2 : 1;     // waves of a SIMD, dq
    // ... dk and dv, whose sums and operands alone are 192 registers at 128 halves (at 64, three registers more than
    // let a third wave in: 475 -> 510 us for the same call)
    static constexpr int OCCUPANCY_KV = DP * (int)sizeof(T) <= 128 ? 3 : DP * (int)sizeof(T) <= 256 ? 2 : 1;
    // dk and dv at 128 halves, two waves of a SIMD: the registers are a few fragments short, and the compiler's own way out would be scratch memory,
    // whose answers wait behind the tiles on their way (waits are in order); so some fragments of the values stay in LDS, where
    // the two waves of SPLIT = 2 share them (one more there than would fit twice: 388 -> 379 us for the whole gradient above).  SPLIT = 1, at 64
    // halves too, is still three registers short: 12 bytes of scratch memory a thread (a fragment more in LDS, which 64 halves have room for, leaves
    // that as it is: 741 -> 748 us for 2 x 4096 tokens of 32 + 8 heads).  Heads above 128 in single are 221 (dk, dv) and 386 (dq) registers
    // short, attention.hip's kernels 109 and 143: they are right, and slow (no shape for them was looked for).
    static constexpr int SPARE = DP == 128 && sizeof(T) == 2 ? (SPLIT == 2 ? 4 : 3) : 0;
    static_assert(LOADS >= 1 && 4 * TILE_BYTES <= 160 * 1024, "a tile is at least a load of every wave, and two stages fit");
};

// The rows that dk and dv walk are ordered so that those of one load are neighbours in memory: CT tokens (the rows of a load) of one head, then
// the same tokens of the group's next head.  Row r is token Q CT + r % CT of head g with r / CT = Q group + g.  A load then has one
// descriptor and an offset that a lane keeps, instead of a division and two products for each row.
template <class T, int PB>
struct ChunkLoader {
    static constexpr int CT = TileLoader<T, PB>::ROWS;
    // LOADS loads from load `first` of the tile that starts at row r0 on; `x` is the group's first head of the sequence's first query.  What
    // lies beyond the last query is beyond the descriptor.
    template <int LOADS, int KB>
    static __device__ __forceinline__ void load(const Args &a, const TileLoader<T, PB> &l, const T *x, long ld, int nq, int r0, int first, unsigned tile) {
        const int t0 = query_of(a, r0 / CT) * CT, chunk = r0 / CT + first;
        int Q = query_of(a, chunk), g = chunk - Q * a.group;
        const unsigned long p = (unsigned long)(x + (long)t0 * ld);
        const unsigned row = (unsigned)(ld * sizeof(T)), head = (unsigned)a.dim * (unsigned)sizeof(T);
        const int left = min(nq - t0, KB + CT);
        const desc_t d = {(unsigned)__builtin_amdgcn_readfirstlane((int)p), (unsigned)__builtin_amdgcn_readfirstlane((int)(p >> 32)) & 0xffffu,
                          (unsigned)__builtin_amdgcn_readfirstlane(left > 0 ? (int)((left - 1) * row + a.group * head) : 0), 0x00020000u};
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int piece = l.lane_pos ^ swizzle<PB>((first + i) * CT + l.lane_row);
            const unsigned at = (unsigned)(Q * CT - t0) * row + (unsigned)g * head;
            load_to_lds(d, piece < l.pieces ? l.voff + piece * 16 + at : 0x80000000u, __builtin_amdgcn_readfirstlane(tile + (first + i) * 1024));
            const bool wrap = g + 1 == a.group;
            g = wrap ? 0 : g + 1, Q += wrap ? 1 : 0;
        }
    }
    static __device__ __forceinline__ int token(const Args &a, int r, int &g) {
        const int chunk = r / CT, Q = query_of(a, chunk);
        g = chunk - Q * a.group;
        return Q * CT + r % CT;
    }
    static __device__ __forceinline__ int rows(const Args &a, int nq) { return (nq + CT - 1) / CT * CT * a.group; }
};

// The rows that a workgroup for some keys walks, cut into chunks of one length for the whole call so that no workgroup has much more to do than
// another (causal, the first keys of a long sequence are seen by all its rows, the last ones by few).  Found on the device from the
// lengths: blocks of keys times the rows that see them, over the pieces wanted.  The sums of a block's chunks meet through scratch in a second launch,
// in the order of the chunks.
template <class T, int DP, int SPLIT>
struct RowCut {
    typedef Shape<T, DP, SPLIT> S;
    typedef ChunkLoader<T, S::PB> Rows;
    int chunk;  // rows
    static __device__ __forceinline__ int blocks(const Span &s) { return (s.nk + S::OWN - 1) / S::OWN; }
    __device__ __forceinline__ int chunks(const Args &a, const Span &s) const { return max(1, (Rows::rows(a, s.nq) + chunk - 1) / chunk); }
    __device__ __forceinline__ void init(const Args &a) {
        chunk = 1 << 30;
        if (!a.pieces) return;
        float all = 0.f, seen = 0.f, own = 0.f;
        for (int first = 0, q_top = 0, k_top = 0; first < a.sequences; first += 64) {
            const Span sp = spans_from(a, first, q_top, k_top);
            const float n = (float)min(sp.nq, sp.nk), pairs = 0.5f * n * n + (float)max(0, sp.nk - sp.nq) * (float)sp.nq;
            own += (float)blocks(sp), all += (float)blocks(sp) * (float)Rows::rows(a, sp.nq), seen += pairs * (float)a.group / S::OWN;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) own += __shfl_xor(own, d), all += __shfl_xor(all, d), seen += __shfl_xor(seen, d);
        // What is seen in a causal call, counted as half of all at least; half a chunk a block is lost to rounding.  Rather too long: there are
        // never more chunks than room, which is for twice as many as are wanted in a causal call.
        const float work = a.causal ? fmaxf(seen, 0.5f * all) : all, wanted = fmaxf((float)a.pieces - 0.5f * own, 0.5f * (float)a.pieces);
        const float grains = ceilf(work * 1.0001f / wanted / (float)ROW_GRAIN);
        chunk = __builtin_amdgcn_readfirstlane(max(1, (int)fminf(grains, (float)((1 << 29) / ROW_GRAIN))) * ROW_GRAIN);
    }
};

template <class T, int DP, int SPLIT>
__global__ __launch_bounds__(256, (Shape<T, DP, SPLIT>::OCCUPANCY_KV)) void attention_grad_kv_kernel(Args a) {
    typedef Type<T> M;
    typedef typename M::frag frag;
    typedef Shape<T, DP, SPLIT> S;
    constexpr int PB = S::PB, UNITS = DP / M::STEP, N = DP / 32;
    __shared__ __attribute__((aligned(1024))) char lds[4 * S::TILE_BYTES];
    __shared__ __attribute__((aligned(16))) float row_lse[2][S::KB], row_delta[2][S::KB];
    __shared__ __attribute__((aligned(16))) frag spare[S::SPARE ? S::SPARE : 1][256 / SPLIT];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int hk = blockIdx.x % a.kv_heads;
    int unit = blockIdx.x / a.kv_heads;
    typedef ChunkLoader<T, PB> Rows;
    RowCut<T, DP, SPLIT> cut;
    cut.init(a);
    Span sp = {0, 0, 0, 0};
    int seq = 0, item = 0;
    const bool there_is = locate(a, unit, sp, seq, item, [&](const Span &s) { return cut.blocks(s) * cut.chunks(a, s); });
    const int chunks = there_is ? cut.chunks(a, sp) : 1, block = item / chunks, nth = item - block * chunks;
    // (each block begins with another chunk: workgroups go round the XCDs, and with a multiple of 8 chunks one XCD would have all the last ones, to
    // which a causal call gives most work: half, one sequence of 8192, 8 + 1 heads of 128, the whole gradient 925 -> 871 us; 725 with RowCut's count
    // of what is seen)
    const int turn = nth + block % chunks, part = turn < chunks ? turn : turn - chunks;
    unit += part - nth;
    const int group = a.group, rows = Rows::rows(a, sp.nq), back = sp.nk - sp.nq;
    // the first row that sees a key of the block (its query is the block's first key less nk - nq), and the chunk that it is in
    const int begin = a.causal ? (int)min((long)(max(0, block * S::OWN - back) / Rows::CT * Rows::CT) * group / S::KB * S::KB, (long)rows) : 0;
    const int first_part = min(begin / cut.chunk, chunks - 1), parts = chunks - first_part;
    // for the second launch: how many chunks the block that begins here has, and which keys
    if (a.pieces && hk == 0 && tid == 0)
        a.joins[unit] = make_int4(there_is && part == first_part && parts > 1 ? parts : 0, sp.k0 + block * S::OWN, min(S::OWN, sp.nk - block * S::OWN), 0);
    if (!there_is || part < first_part) return;
    const int r_begin = max(begin, part * cut.chunk), r_end = min((long)rows, (part + 1L) * cut.chunk);
    // (of the rows from the first query of r_begin's load to the last one of the load before r_end)
    const int t_begin = min(query_of(a, r_begin / Rows::CT) * Rows::CT, sp.nq), t_end = r_begin < r_end ? min(sp.nq, (query_of(a, (r_end - 1) / Rows::CT) + 1) * Rows::CT) : t_begin;
    const float mult = keys_scale<T>(a, sp, hk, block * S::OWN, S::OWN, t_begin, t_end), c = a.scale * LOG2E, shift = scaled<T>() ? P_SHIFT : 0.f;
    const int j0 = block * S::OWN + wave % (4 / SPLIT) * 32;  // the wave's first key
    frag kf[UNITS], vf[UNITS - S::SPARE];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const int j = j0 + (lane & 31);
        const bool there = j < sp.nk;
        const long key = sp.k0 + (there ? j : 0);
        kf[u] = load_piece<T>((const T *)a.k + key * a.ldk + (long)hk * a.dim, u * M::STEP + h * M::V, a.dim, there, 1);
        const frag v = load_piece<T>((const T *)a.v + key * a.ldv + (long)hk * a.dim, u * M::STEP + h * M::V, a.dim, there, 1);
        if (u < UNITS - S::SPARE) vf[u] = v;
        else spare[u - (UNITS - S::SPARE)][tid % (256 / SPLIT)] = v;
    }
    f32x16 dk[N], dv[N];
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[b][e] = dv[b][e] = 0.f;
    const unsigned lds0 = lds_address(lds);
    const T *q = (const T *)a.q + (long)sp.q0 * a.ldq + (long)hk * group * a.dim, *g = (const T *)a.dout + (long)sp.q0 * a.lddo + (long)hk * group * a.dim;
    float next_lse = 0.f, next_delta = 0.f;  // of row tid of the next tile
    bool next_in = false;
    auto fetch = [&](int r0, int stage) {
        int fl = lane;
        asm volatile("" : "+v"(fl));  // (what follows from the lane is formed anew each time: registers are what this kernel is short of)
        TileLoader<T, PB> lq, lg;
        lq.init(a.ldq, a.dim, fl), lg.init(a.lddo, a.dim, fl);
        const int tid = wave * 64 + fl;
        Rows::template load<S::LOADS, S::KB>(a, lq, q, a.ldq, sp.nq, r0, wave * S::LOADS, lds0 + stage * 2 * S::TILE_BYTES);
        Rows::template load<S::LOADS, S::KB>(a, lg, g, a.lddo, sp.nq, r0, wave * S::LOADS, lds0 + stage * 2 * S::TILE_BYTES + S::TILE_BYTES);
        // (every lane asks, and nothing is done with the answers here: that would wait for them, and for the tiles asked for before them)
        int head;
        const int t = Rows::token(a, r0 + min(tid, S::KB - 1), head);
        next_in = t < sp.nq;
        const long at = (long)(hk * group + head) * a.q_tokens + sp.q0 + (next_in ? t : 0);
        next_lse = a.lse[at], next_delta = a.delta[at];
    };
    if (r_begin < r_end) fetch(r_begin, 0);
    for (int r0 = r_begin, stage = 0; r0 < r_end; r0 += S::KB, stage ^= 1) {
        if (wave * 64 < S::KB) {
            int wl = lane;
            asm volatile("" : "+v"(wl));
            if (wave * 64 + wl < S::KB) {  // (rows that are not there: probability zero)
                row_lse[stage][wave * 64 + wl] = next_in ? next_lse * LOG2E - shift : INFINITY;
                row_delta[stage][wave * 64 + wl] = next_in ? next_delta * mult : 0.f;
            }
        }
        ATTN_VMCNT(0);
        lds_reads_done();
        __syncthreads();
        if (r0 + S::KB < r_end) fetch(r0 + S::KB, stage ^ 1);
        const char *tq = lds + stage * 2 * S::TILE_BYTES, *tg = tq + S::TILE_BYTES;
#pragma unroll 1
        for (int i = 0; i < S::BLOCKS / SPLIT; ++i) {
            const int b = SPLIT == 1 ? i : wave / (4 / SPLIT), rb = r0 + b * 32;
            // (a block of rows that see none of the wave's keys is masked, not left out: a way round the products makes the compiler move the sums
            // to and fro, and few are such)
            int l = lane;
            asm volatile("" : "+v"(l));  // fragments' addresses are formed here, not kept in registers across the loop
            f32x16 s, w;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = w[e] = 0.f;
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                M::mma(s, rows_frag<T, PB>(tq, b * 32, u, l), kf[u]);
                M::mma(w, rows_frag<T, PB>(tg, b * 32, u, l), u < UNITS - S::SPARE ? vf[u] : spare[u - (UNITS - S::SPARE)][wave % (4 / SPLIT) * 64 + l]);
            }
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const f32x4 l4 = *(const f32x4 *)&row_lse[stage][b * 32 + 2 * e + 4 * (l >> 5)], d4 = *(const f32x4 *)&row_delta[stage][b * 32 + 2 * e + 4 * (l >> 5)];
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) {
                    s[e + i4] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e + i4], c, -l4[i4]));
                    w[e + i4] = __builtin_fmaf(w[e + i4], mult, -d4[i4]);
                }
            }
            if (a.causal && j0 + 31 > query_of(a, rb / Rows::CT) * Rows::CT + back) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    int head;
                    const bool seen = j0 + (l & 31) <= Rows::token(a, rb + 8 * (e >> 2) + 4 * (l >> 5) + (e & 3), head) + back;
                    s[e] = seen ? s[e] : 0.f, w[e] = seen ? w[e] : 0.f;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] *= s[e];
#pragma unroll
            for (int u = 0; u < 32 / M::STEP; ++u) {
                const frag p = M::pack(s, u), d = M::pack(w, u);
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    M::mma(dv[n], cols_frag<T, PB>(tg, b * 32 + u * M::STEP, n * 32, l), p);
                    M::mma(dk[n], cols_frag<T, PB>(tq, b * 32 + u * M::STEP, n * 32, l), d);
                }
            }
        }
    }
    int el = lane;
    asm volatile("" : "+v"(el));
    if constexpr (SPLIT == 2) {
        __syncthreads();
        float *to = (float *)lds + (wave & 1) * 2 * N * 16 * 64 + el;
        if (wave >= 2) {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) to[(n * 16 + e) * 64] = dk[n][e], to[((N + n) * 16 + e) * 64] = dv[n][e];
        }
        __syncthreads();
        if (wave >= 2) return;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) dk[n][e] += to[(n * 16 + e) * 64], dv[n][e] += to[((N + n) * 16 + e) * 64];
    }
    const float unshift = exp2f(-shift), by = a.scale * unshift / mult;
    if (parts > 1) {  // as the registers hold them: the second launch's lanes hold the same elements
        float *to = a.part + (((long)unit * a.kv_heads + hk) * (S::OWN / 32) + wave % (4 / SPLIT)) * 2 * N * 16 * 64 + el;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) to[(n * 16 + e) * 64] = dk[n][e] * by, to[((N + n) * 16 + e) * 64] = dv[n][e] * unshift;
        return;
    }
    const int j = j0 + (el & 31);
    if (j >= sp.nk) return;
    const long key = sp.k0 + j;
    T *pk = (T *)a.dk + key * a.lddk + (long)hk * a.dim, *pv = (T *)a.dv + key * a.lddv + (long)hk * a.dim;
    store_sums<T, DP>(pk, dk, by, a.dim, el >> 5, a.overwrite & 2);
    store_sums<T, DP>(pv, dv, unshift, a.dim, el >> 5, a.overwrite & 4);
}

template <class T, int DP, int SPLIT>
__global__ __launch_bounds__(256, (Shape<T, DP, SPLIT>::OCCUPANCY)) void attention_grad_q_kernel(Args a) {
    typedef Type<T> M;
    typedef typename M::frag frag;
    typedef Shape<T, DP, SPLIT> S;
    constexpr int PB = S::PB, UNITS = DP / M::STEP, N = DP / 32;
    __shared__ __attribute__((aligned(1024))) char lds[4 * S::TILE_BYTES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int hk = blockIdx.x % a.kv_heads;
    Span sp;
    int seq, tile;
    auto tiles_of = [&](const Span &s) { return (int)(((long)s.nq * a.group + S::OWN - 1) / S::OWN); };
    if (!locate(a, blockIdx.x / a.kv_heads, sp, seq, tile, tiles_of)) return;
    const int group = a.group, rows = sp.nq * group, back = sp.nk - sp.nq;
    tile = tiles_of(sp) - 1 - tile;  // the rows that see most keys first
    const float c = a.scale * LOG2E, shift = scaled<T>() ? P_SHIFT : 0.f;
    const int r = tile * S::OWN + wave % (4 / SPLIT) * 32 + (lane & 31);
    const bool there = r < rows;
    const int t = query_of(a, there ? r : rows - 1), head = hk * group + (there ? r - t * group : 0);
    frag qf[UNITS], gf[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        qf[u] = load_piece<T>((const T *)a.q + (long)(sp.q0 + t) * a.ldq + (long)head * a.dim, u * M::STEP + h * M::V, a.dim, there, 1);
        gf[u] = load_piece<T>((const T *)a.dout + (long)(sp.q0 + t) * a.lddo + (long)head * a.dim, u * M::STEP + h * M::V, a.dim, there, 1);
    }
    const long at = (long)head * a.q_tokens + sp.q0 + t;
    const float lse = there ? a.lse[at] * LOG2E - shift : INFINITY, norm = scaled<T>() && there ? a.norms[at] : 0.f;
    float delta = there ? a.delta[at] : 0.f;
    const int last = a.causal ? min(sp.nk - 1, t + back) : sp.nk - 1;
    const int end = a.causal ? min(sp.nk, query_of(a, min(rows, (tile + 1) * S::OWN) - 1) + back + 1) : sp.nk;
    const int wave_all = __builtin_amdgcn_readfirstlane(__shfl(last, 0)), wave_end = __builtin_amdgcn_readfirstlane(__shfl(last, 31)) + 1;
    const float mult = row_scale<T>(norm, largest_v<T>(a, sp, hk, end));
    delta *= mult;
    f32x16 dq[N];
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) dq[b][e] = 0.f;
    const T *k = (const T *)a.k + (long)sp.k0 * a.ldk + (long)hk * a.dim, *v = (const T *)a.v + (long)sp.k0 * a.ldv + (long)hk * a.dim;
    TileLoader<T, PB> lk, lv;
    lk.init(a.ldk, a.dim, lane), lv.init(a.ldv, a.dim, lane);
    const unsigned lds0 = lds_address(lds);
    auto fetch = [&](int j0, int stage) {
        const desc_t dk = lk.desc(k + (long)j0 * a.ldk, min(S::KB, sp.nk - j0), a.ldk, a.dim), dv = lv.desc(v + (long)j0 * a.ldv, min(S::KB, sp.nk - j0), a.ldv, a.dim);
#pragma unroll
        for (int i = 0; i < S::LOADS; ++i) lk.load(dk, wave * S::LOADS + i, lds0 + stage * 2 * S::TILE_BYTES);
#pragma unroll
        for (int i = 0; i < S::LOADS; ++i) lv.load(dv, wave * S::LOADS + i, lds0 + stage * 2 * S::TILE_BYTES + S::TILE_BYTES);
    };
    if (end > 0) fetch(0, 0);
    for (int j0 = 0, stage = 0; j0 < end; j0 += S::KB, stage ^= 1) {
        ATTN_VMCNT(0);
        lds_reads_done();
        __syncthreads();
        if (j0 + S::KB < end) fetch(j0 + S::KB, stage ^ 1);
        const char *tk = lds + stage * 2 * S::TILE_BYTES, *tv = tk + S::TILE_BYTES;
#pragma unroll 1
        for (int i = 0; i < S::BLOCKS / SPLIT; ++i) {
            const int b = SPLIT == 1 ? i : wave / (4 / SPLIT), jb = j0 + b * 32;
            if (jb >= wave_end) continue;
            f32x16 s, w;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = w[e] = 0.f;
#pragma unroll
            for (int u = 0; u < UNITS; ++u) M::mma(s, rows_frag<T, PB>(tk, b * 32, u, lane), qf[u]);
#pragma unroll
            for (int u = 0; u < UNITS; ++u) M::mma(w, rows_frag<T, PB>(tv, b * 32, u, lane), gf[u]);
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -lse));
            if (jb + 31 > wave_all) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const bool seen = jb + 8 * (e >> 2) + 4 * h + (e & 3) <= last;
                    s[e] = seen ? s[e] : 0.f, w[e] = seen ? w[e] : 0.f;
                }
            }
            if (end <= 32) {
                // rows of few keys: delta from the probabilities themselves; do o has the rounding of o in it, which there weighs as much as
                // the rounding of ds (up to 64 keys, by a pass before: 3.1 instead of 3.5 10^-4 of dq at 5 sequences of 26 in half, but then
                // the loop's fragments no longer stay in registers, and the gradient of long sequences takes 640 us for 370)
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 16; ++e) sum += s[e] * w[e];
                sum += __shfl_xor(sum, 32);
                sum *= exp2f(-shift);
                if (there && h == 0) a.delta[at] = sum;
                delta = sum * mult;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = s[e] * __builtin_fmaf(w[e], mult, -delta);
#pragma unroll
            for (int u = 0; u < 32 / M::STEP; ++u) {
                const frag d = M::pack(w, u);
#pragma unroll
                for (int n = 0; n < N; ++n) M::mma(dq[n], cols_frag<T, PB>(tk, b * 32 + u * M::STEP, n * 32, lane), d);
            }
        }
    }
    if constexpr (SPLIT == 2) {
        __syncthreads();
        float *to = (float *)lds + (wave & 1) * N * 16 * 64 + lane;
        if (wave >= 2) {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) to[(n * 16 + e) * 64] = dq[n][e];
        }
        __syncthreads();
        if (wave >= 2) return;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) dq[n][e] += to[(n * 16 + e) * 64];
    }
    if (!there) return;
    store_sums<T, DP>((T *)a.dq + (long)(sp.q0 + t) * a.lddq + (long)head * a.dim, dq, a.scale * exp2f(-shift) / mult, a.dim, h, a.overwrite & 1);
}

// the chunks of a block of keys joined; a wave has dk or dv of 32 keys.  Bound by the partial sums' bytes.
template <class T, int DP, int SPLIT>
__global__ __launch_bounds__(256) void attention_grad_join_kernel(Args a) {
    typedef Shape<T, DP, SPLIT> S;
    constexpr int N = DP / 32;
    const int lane = threadIdx.x & 63, hk = blockIdx.x % a.kv_heads, unit = blockIdx.x / a.kv_heads;
    const int4 join = a.joins[unit];
    if (!join.x) return;
    for (int i = threadIdx.x >> 6; i < S::OWN / 32 * 2; i += 4) {
        const int keys = i >> 1, which = i & 1;
        const float *from = a.part + (((long)unit * a.kv_heads + hk) * (S::OWN / 32) + keys) * 2 * N * 16 * 64 + which * N * 16 * 64 + lane;
        const long step = (long)a.kv_heads * (S::OWN / 32) * 2 * N * 16 * 64;
        f32x16 x[N];
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) x[n][e] = from[(n * 16 + e) * 64];
        for (int p = 1; p < join.x; ++p)
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) x[n][e] += from[p * step + (n * 16 + e) * 64];
        const int j = keys * 32 + (lane & 31);
        if (j >= join.z) continue;
        const long key = join.y + j;
        if (which == 0) store_sums<T, DP>((T *)a.dk + key * a.lddk + (long)hk * a.dim, x, 1.f, a.dim, lane >> 5, a.overwrite & 2);
        else store_sums<T, DP>((T *)a.dv + key * a.lddv + (long)hk * a.dim, x, 1.f, a.dim, lane >> 5, a.overwrite & 4);
    }
}

// SPLIT for so many keys (rows), of which a workgroup has 128 or 64
int split_for(long own, int kv_heads) { return (own + 127) / 128 * kv_heads < 2 * cu_count() ? 2 : 1; }

template <class T, int DP, int SPLIT>
int launch_kv(const Args &a, hipStream_t stream) {
    hipLaunchKernelGGL((attention_grad_kv_kernel<T, DP, SPLIT>), dim3((unsigned)a.units * a.kv_heads), dim3(256), 0, stream, a);
    D8_LAUNCH_CHECK();
    if (!a.pieces) return 0;
    hipLaunchKernelGGL((attention_grad_join_kernel<T, DP, SPLIT>), dim3((unsigned)a.units * a.kv_heads), dim3(256), 0, stream, a);
    D8_LAUNCH_CHECK();
    return 0;
}
template <class T, int DP, int SPLIT>
int launch_q(const Args &a, hipStream_t stream) {
    const long tiles = ((long)a.q_tokens * a.group + 128 / SPLIT - 1) / (128 / SPLIT) + a.sequences;
    hipLaunchKernelGGL((attention_grad_q_kernel<T, DP, SPLIT>), dim3((unsigned)tiles * a.kv_heads), dim3(256), 0, stream, a);
    D8_LAUNCH_CHECK();
    return 0;
}

template <class T, int DP>
int launch_dim(const Args &a, bool fast, hipStream_t stream) {
    constexpr bool CAN_SPLIT = row_bytes<T, DP>() <= 512;
    if (a.q_tokens) {  // dq first: it may set delta anew
        const int split = split_for((long)a.q_tokens * a.group, a.kv_heads);
        if (!fast) {
            const long tiles = ((long)a.q_tokens * a.group + ROWS - 1) / ROWS + a.sequences;
            hipLaunchKernelGGL((attention_grad_q_any_kernel<T, DP>), dim3((unsigned)tiles * a.kv_heads), dim3(256), 0, stream, a);
            D8_LAUNCH_CHECK();
        } else if (int rc = CAN_SPLIT && split == 2 ? launch_q<T, DP, CAN_SPLIT ? 2 : 1>(a, stream) : launch_q<T, DP, 1>(a, stream)) {
            return rc;
        }
    }
    if (!a.k_tokens) return 0;
    if (!fast) {
        const long blocks = ((long)a.k_tokens + KEYS - 1) / KEYS + a.sequences;
        hipLaunchKernelGGL((attention_grad_kv_any_kernel<T, DP>), dim3((unsigned)blocks * a.kv_heads), dim3(256), 0, stream, a);
        D8_LAUNCH_CHECK();
        return 0;
    }
    return CAN_SPLIT && a.split_kv == 2 ? launch_kv<T, DP, CAN_SPLIT ? 2 : 1>(a, stream) : launch_kv<T, DP, 1>(a, stream);
}

template <class T>
int launch(const Args &a, bool fast, hipStream_t stream) {
    int lanes = 1;
    while (lanes * Type<T>::V < a.dim) lanes *= 2;
    hipLaunchKernelGGL(attention_delta_kernel<T>, dim3(DELTA_GROUPS), dim3(256), 0, stream, a, lanes);
    D8_LAUNCH_CHECK();
    if (a.dim <= 32) return launch_dim<T, 32>(a, fast, stream);
    if (a.dim <= 64) return launch_dim<T, 64>(a, fast, stream);
    if (a.dim <= 96) return launch_dim<T, 96>(a, fast, stream);
    if (a.dim <= 128) return launch_dim<T, 128>(a, fast, stream);
    return launch_dim<T, 256>(a, fast, stream);
}

}  // namespace

// How dk and dv are cut: keys of a workgroup, pieces that the rows are cut into (0: not at all), pieces of work there is room for.  Four
// workgroups a compute unit, two rounds of what runs at once, are wanted.
struct GradPlan {
    int split, pieces, units;
    size_t lists, parts;  // bytes
};
static GradPlan grad_plan(int dtype, int sequences, int q_tokens, int k_tokens, int heads, int kv_heads, int dim, bool causal) {
    GradPlan p;
    const int padded = dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : 256;
    p.split = dtype == D8_FLOAT32 && padded == 256 ? 1 : split_for(k_tokens, kv_heads);
    const int own = 128 / p.split;
    const long blocks = ((long)k_tokens + own - 1) / own + sequences, rows = (long)q_tokens * (heads / kv_heads);
    const long want = (4L * cu_count() + kv_heads - 1) / kv_heads, most = (blocks * rows + ROW_GRAIN - 1) / ROW_GRAIN;
    p.pieces = (int)(blocks >= 2 * want ? 0 : want < most ? want : most);
    if (rows <= ROW_GRAIN) p.pieces = 0;
    p.units = (int)(blocks + (causal ? 2 : 1) * p.pieces);
    p.lists = p.pieces ? ((size_t)p.units * sizeof(int4) + 255) & ~(size_t)255 : 0;
    p.parts = p.pieces ? (size_t)p.units * kv_heads * own * 2 * padded * sizeof(float) : 0;
    return p;
}

// delta and norms
static size_t row_bytes_of(int dtype, int q_tokens, int k_tokens, int heads, int kv_heads) {
    const size_t rows = (size_t)q_tokens * heads, floats = dtype == D8_FLOAT16 ? 2 * rows + (size_t)k_tokens * kv_heads : rows;
    return (sizeof(float) * floats + 255) & ~(size_t)255;
}

size_t grad_scratch_bytes(int dtype, int sequences, int q_tokens, int k_tokens, int heads, int kv_heads, int dim, bool causal) {
    const GradPlan p = grad_plan(dtype, sequences, q_tokens, k_tokens, heads, kv_heads, dim, causal != 0);
    return row_bytes_of(dtype, q_tokens, k_tokens, heads, kv_heads) + p.lists + p.parts;
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
    const attention::GradPlan plan = attention::grad_plan(dtype, sequences, q_tokens, k_tokens, heads, kv_heads, dim, causal != 0);
    const size_t need = attention::grad_scratch_bytes(dtype, sequences, q_tokens, k_tokens, heads, kv_heads, dim, causal != 0);
    D8_REQUIRE(scratch && scratch_bytes >= need && ((size_t)scratch & 15) == 0, "attention_grad: 16-byte aligned scratch of %zu bytes is needed, not %zu", need, scratch_bytes);
    a.delta = (float *)scratch, a.norms = a.delta + (size_t)q_tokens * heads, a.v_norms = a.norms + (size_t)q_tokens * heads;
    a.joins = (int4 *)((char *)scratch + attention::row_bytes_of(dtype, q_tokens, k_tokens, heads, kv_heads)), a.part = (float *)((char *)a.joins + plan.lists);
    a.pieces = plan.pieces, a.units = plan.units, a.split_kv = plan.split;
    attention::set_group(a);
    a.vec = attention::in_pieces(dtype, dim, {q, k, v, o, dout}, {ldq, ldk, ldv, ldo, lddo});
    // (a tile's rows are addressed by 31 bits)
    const long most = 1 << 21;
    const bool fast = a.vec && attention::in_pieces(dtype, dim, {dq, dk, dv}, {lddq, lddk, lddv}) && ldq < most && ldk < most && ldv < most && lddo < most;
    D8_REQUIRE((((long)q_tokens * a.group + k_tokens) / 64 + 2 * (long)sequences + 2 * plan.pieces + 2) * kv_heads < (1L << 31), "attention_grad: too many sequences");
    return dtype == D8_FLOAT16 ? attention::launch<f16>(a, fast, as_stream(stream)) : attention::launch<float>(a, fast, as_stream(stream));
}
