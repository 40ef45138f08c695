// Attention over packed sequences of different lengths, heads sharing keys and values, forward.
//
//   s = scale q k^T (query t of a sequence with nq queries and nk keys sees keys j <= t + nk - nq, or all),  o = softmax(s) v,
//   lse = log(sum exp s);  a row that sees nothing: o = 0, lse = -inf
//
// One pass over the keys with the running maximum and sum of the softmax (fp32).  A workgroup has 128 rows, each of its four waves
// 32 of them; the scores are computed transposed (keys x rows), so that a row's scores lie in one lane (and its partner 32 lanes on),
// maximum and sum are lane arithmetic, and the probabilities are the right operand of the product with the values where they are.
// In half the probabilities, at most 1 relative to the running maximum (up to 2^8 where it lags), are rounded to half for that product,
// the type that the matrix instruction takes at full rate: as much error again as the rounding of o where values have random signs, 2.6 (prompts)
// to 2.9 10^-4 (single queries over thousands of keys) for 2.1.  Maxima, sums and o are fp32, the sum that of the unrounded ones.
#include "attention.h"

namespace d8 {
namespace attention {
namespace {

enum { ROWS = 128, KEYS = 32 };

template <class T, int DP>
__global__ __launch_bounds__(256) void attention_any_kernel(Args a) {
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
    const int t = query_of(a, r), head = hk * group + r - t * group;
    const bool there = r < rows;
    const T *q = (const T *)a.q + (long)(sp.q0 + (there ? t : 0)) * a.ldq + (long)head * a.dim;
    frag qf[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) qf[u] = load_piece<T>(q, u * M::STEP + h * M::V, a.dim, there, a.vec);
    const int back = sp.nk - sp.nq;
    const int last = a.causal ? min(sp.nk - 1, t + back) : sp.nk - 1;  // last key that the lane's row sees
    const int t_end = query_of(a, min(rows, (tile + 1) * ROWS) - 1);
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

// The lane's row of q as fragments, negated where the scale is negative (the softmax below takes |scale|).
template <class T, int DP>
__device__ __forceinline__ void load_query(const Args &a, const T *q, bool there, int h, typename Type<T>::frag (&qf)[DP / Type<T>::STEP]) {
#pragma unroll
    for (int u = 0; u < DP / Type<T>::STEP; ++u) {
        qf[u] = load_piece<T>(q, u * Type<T>::STEP + h * Type<T>::V, a.dim, there, 1);
        if (a.scale < 0.f) qf[u] = -qf[u];
    }
}
// (a scale of zero as one so small that no score is seen: infinite hidden scores times zero would be no number)
__device__ __forceinline__ float exponent_scale(const Args &a) { return fmaxf(fabsf(a.scale) * LOG2E, 1e-30f); }

// Large outputs.  128 rows a workgroup, keys in tiles of 64 (32 where a row takes more than 256 bytes) that go from memory straight into one of
// two stages of LDS, the next tile's while this one is worked on; one barrier a tile.  Two workgroups a compute unit, so that
// one's products run under the other's exponentials.  Half, causal, sequences of 7290, 7240 and 1854, 16 + 4 heads of 128: 480 us at the least,
// 530 in the mean of 40 calls in a row, 930 and 840 TFLOP/s (a large product 1320).  Bound by power: 7.3 M cycles at 1.89 GHz, where a kernel that waits
// for memory runs at 2.5; fragments read four products ahead take 5 % of the cycles away and the clock falls by as much.
template <class T, int DP>
__global__ __launch_bounds__(256, (DP * (int)sizeof(T) <= 256 ? 2 : 1)) void attention_rows_kernel(Args a) {
    typedef Type<T> M;
    typedef typename M::frag frag;
    constexpr int PB = row_bytes<T, DP>(), KB = PB <= 256 ? 64 : 32, NB = KB / 32, TILE = KB * PB, LOADS = TILE / 1024 / 4;
    static_assert(LOADS >= 1, "every wave has a share of a tile");
    __shared__ __attribute__((aligned(1024))) char lds[4 * TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int hk = blockIdx.x % a.kv_heads;
    Span sp;
    int seq, tile;
    auto tiles_of = [&](const Span &s) { return (int)(((long)s.nq * a.group + ROWS - 1) / ROWS); };
    if (!locate(a, blockIdx.x / a.kv_heads, sp, seq, tile, tiles_of)) return;
    const int group = a.group, rows = sp.nq * group;
    tile = tiles_of(sp) - 1 - tile;  // the rows that see most keys first
    const int r = tile * ROWS + wave * 32 + (lane & 31);
    const bool there = r < rows;
    const int t = query_of(a, there ? r : rows - 1), head = hk * group + (there ? r - t * group : 0);
    frag qf[DP / M::STEP];
    load_query<T, DP>(a, (const T *)a.q + (long)(sp.q0 + t) * a.ldq + (long)head * a.dim, there, h, qf);
    const int back = sp.nk - sp.nq;
    const int last = a.causal ? min(sp.nk - 1, t + back) : sp.nk - 1;  // last key that the lane's row sees
    const int end = a.causal ? min(sp.nk, query_of(a, min(rows, (tile + 1) * ROWS) - 1) + back + 1) : sp.nk;
    // what all rows of the wave see, and the end of what one of them sees
    const int wave_all = __builtin_amdgcn_readfirstlane(__shfl(last, 0)), wave_end = __builtin_amdgcn_readfirstlane(__shfl(last, 31)) + 1;
    const float c = exponent_scale(a);
    f32x16 acc[DP / 32];
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[b][e] = 0.f;
    Softmax soft;
    soft.init();
    const T *k = (const T *)a.k + (long)sp.k0 * a.ldk + (long)hk * a.dim, *v = (const T *)a.v + (long)sp.k0 * a.ldv + (long)hk * a.dim;
    TileLoader<T, PB> lk, lv;
    lk.init(a.ldk, a.dim, lane), lv.init(a.ldv, a.dim, lane);
    const unsigned lds0 = lds_address(lds);
    auto fetch = [&](int j0, int stage) {
        const desc_t dk = lk.desc(k + (long)j0 * a.ldk, min(KB, sp.nk - j0), a.ldk, a.dim), dv = lv.desc(v + (long)j0 * a.ldv, min(KB, sp.nk - j0), a.ldv, a.dim);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) lk.load(dk, wave * LOADS + i, lds0 + stage * 2 * TILE);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) lv.load(dv, wave * LOADS + i, lds0 + stage * 2 * TILE + TILE);
    };
    if (end > 0) fetch(0, 0);
    for (int j0 = 0, stage = 0; j0 < end; j0 += KB, stage ^= 1) {
        // this tile has landed, and every wave is through with the other stage
        ATTN_VMCNT(0);
        lds_reads_done();
        __syncthreads();
        if (j0 + KB < end) fetch(j0 + KB, stage ^ 1);
        if (j0 >= wave_end) continue;
        const char *tk = lds + stage * 2 * TILE, *tv = tk + TILE;
        f32x16 s[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[b][e] = 0.f;
#pragma unroll
        for (int u = 0; u < DP / M::STEP; ++u)
#pragma unroll
            for (int b = 0; b < NB; ++b) M::mma(s[b], rows_frag<T, PB>(tk, b * 32, u, lane), qf[u]);
        if (j0 + KB - 1 > wave_all) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[b][e] = j0 + b * 32 + 8 * (e >> 2) + 4 * h + (e & 3) <= last ? s[b][e] : -INFINITY;
        }
        float keep;
        if (soft.step<NB>(s, c, keep)) {
#pragma unroll
            for (int b = 0; b < DP / 32; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[b][e] *= keep;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int u = 0; u < 32 / M::STEP; ++u) {
                const frag p = M::pack(s[b], u);
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) M::mma(acc[d], cols_frag<T, PB>(tv, b * 32 + u * M::STEP, d * 32, lane), p);
            }
    }
    const float sum = soft.sum + __shfl_xor(soft.sum, 32);
    if (!there) return;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T *o = (T *)a.o + (long)(sp.q0 + t) * a.ldo + (long)head * a.dim;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int at = d * 32 + 2 * e + 4 * h;
            T out[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = (T)(acc[d][e + i] * inv);
            if (at < a.dim) __builtin_memcpy(__builtin_assume_aligned(o + at, 4 * sizeof(T)), out, 4 * sizeof(T));
        }
    if (a.lse && h == 0) a.lse[(long)head * a.q_tokens + sp.q0 + t] = sum == 0.f ? -INFINITY : (soft.base + log2f(sum)) * LN2;
}

// Few rows: 32 a workgroup, whose waves have the same rows and take every WAVES-th tile of 32 keys, each with its own LDS and no
// barrier: the keys and values of a tile are asked for again as soon as the last read of their place has been answered.  The keys of
// a sequence are cut into chunks of one length for the whole call, found from the lengths on the device, so that the
// pieces of work are alike whatever the lengths; a row's chunks are joined by a second launch (their unnormalised outputs with
// their maxima and sums).  One query a sequence: bound by the keys' and values' bytes, 537 MB (16 sequences, 131072 keys, 8 heads of 128 halves) in
// 105 us = 5.1 TB/s and 6 for the join.  Short prompts: by what a workgroup waits for at its start and end; in single a compute unit
// holds one workgroup with heads of more than 64 (sequences of 336 to 604, 6 + 2 heads of 80: 50 us for 8 of products).
struct Cut {
    int chunk;  // keys
    __device__ __forceinline__ int tiles(const Args &a, const Span &s) const { return (s.nq * a.group + 31) / 32; }
    __device__ __forceinline__ int chunks(const Span &s) const { return max(1, (s.nk + chunk - 1) / chunk); }
    // tiles times keys over the pieces wanted, rounded up to whole grains.  In fp32, a little too long rather than too short: there are then never
    // more chunks than pieces and tiles.  Every wave of the call computes the same bits.
    __device__ __forceinline__ void init(const Args &a, int grain) {
        chunk = 1 << 30;
        if (!a.pieces) return;
        float work = 0.f;
        for (int first = 0, q_top = 0, k_top = 0; first < a.sequences; first += 64) {
            const Span sp = spans_from(a, first, q_top, k_top);
            work += (float)tiles(a, sp) * (float)sp.nk;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) work += __shfl_xor(work, d);
        const float grains = ceilf(work * 1.0001f / (float)a.pieces / (float)grain);
        chunk = __builtin_amdgcn_readfirstlane(max(1, (int)fminf(grains, (float)((1 << 29) / grain))) * grain);
    }
    // keys that some row of the tile sees
    __device__ __forceinline__ int end(const Args &a, const Span &s, int tile) const {
        const int rows = s.nq * a.group;
        return a.causal ? max(0, min(s.nk, query_of(a, min(rows, (tile + 1) * 32) - 1) + s.nk - s.nq + 1)) : s.nk;
    }
};
enum { CHUNK_GRAIN = 256 };

template <class T, int DP, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void attention_keys_kernel(Args a) {
    typedef Type<T> M;
    typedef typename M::frag frag;
    constexpr int PB = row_bytes<T, DP>(), TILE = 32 * PB, LOADS = TILE / 1024, OUT = DP + 4;
    constexpr int STAGES = WAVES * 2 * TILE, JOIN = WAVES * 32 * OUT * 4;
    __shared__ __attribute__((aligned(1024))) char lds[STAGES > JOIN ? STAGES : JOIN];
    __shared__ float wave_base[WAVES][32], wave_sum[WAVES][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int hk = blockIdx.x % a.kv_heads, unit = blockIdx.x / a.kv_heads;
    Cut cut;
    cut.init(a, CHUNK_GRAIN);
    Span sp = {0, 0, 0, 0};
    int seq = 0, item = 0;
    const bool there_is = locate(a, unit, sp, seq, item, [&](const Span &s) { return cut.tiles(a, s) * cut.chunks(s); });
    // (the rows that see most keys first, so that the last to start have little to do: single, 5 prompts of 500, heads of 80, 60 -> 55 us)
    const int chunks = there_is ? cut.chunks(sp) : 1, nth = item / chunks, tile = cut.tiles(a, sp) - 1 - nth, begin = (item - nth * chunks) * cut.chunk;
    const int group = a.group, rows = sp.nq * group, all = there_is ? cut.end(a, sp, tile) : 0, end = min(all, begin + cut.chunk);
    const bool whole = all <= cut.chunk;
    // for the second launch: how many chunks the tile that begins here has, and which rows
    if (a.pieces && hk == 0 && tid == 0) a.joins[unit] = make_int4(there_is && !whole && begin == 0 ? (all + cut.chunk - 1) / cut.chunk : 0, sp.q0, tile, rows);
    if (!there_is || (begin > 0 && begin >= all)) return;  // (the first chunk is there even if its rows see nothing)
    const int r = tile * 32 + (lane & 31);
    const bool there = r < rows;
    const int t = query_of(a, there ? r : rows - 1), head = hk * group + (there ? r - t * group : 0);
    frag qf[DP / M::STEP];
    load_query<T, DP>(a, (const T *)a.q + (long)(sp.q0 + t) * a.ldq + (long)head * a.dim, there, h, qf);
    const int last = a.causal ? min(sp.nk - 1, t + sp.nk - sp.nq) : sp.nk - 1;
    const int wave_all = __builtin_amdgcn_readfirstlane(__shfl(last, 0));
    const float c = exponent_scale(a);
    f32x16 acc[DP / 32];
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[b][e] = 0.f;
    Softmax soft;
    soft.init();
    const T *k = (const T *)a.k + (long)sp.k0 * a.ldk + (long)hk * a.dim, *v = (const T *)a.v + (long)sp.k0 * a.ldv + (long)hk * a.dim;
    TileLoader<T, PB> lk, lv;
    lk.init(a.ldk, a.dim, lane), lv.init(a.ldv, a.dim, lane);
    const char *tk = lds + wave * 2 * TILE, *tv = tk + TILE;
    const unsigned at_k = lds_address(lds) + wave * 2 * TILE, at_v = at_k + TILE;
    auto fetch = [&](const TileLoader<T, PB> &l, const T *x, long ld, int j, unsigned at) {
        const desc_t d = l.desc(x + (long)j * ld, min(32, sp.nk - j), ld, a.dim);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) l.load(d, i, at);
    };
    int j = begin + wave * 32;
    if (j < end) fetch(lk, k, a.ldk, j, at_k), fetch(lv, v, a.ldv, j, at_v);
    for (; j < end; j += WAVES * 32) {
        const bool more = j + WAVES * 32 < end;
        ATTN_VMCNT(LOADS);  // the keys have landed, the values may be on their way
        asm volatile("" ::: "memory");
        f32x16 s[1];
#pragma unroll
        for (int e = 0; e < 16; ++e) s[0][e] = 0.f;
#pragma unroll
        for (int u = 0; u < DP / M::STEP; ++u) M::mma(s[0], rows_frag<T, PB>(tk, 0, u, lane), qf[u]);
        lds_reads_done();
        if (more) fetch(lk, k, a.ldk, j + WAVES * 32, at_k);
        if (j + 31 > wave_all) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[0][e] = j + 8 * (e >> 2) + 4 * h + (e & 3) <= last ? s[0][e] : -INFINITY;
        }
        float keep;
        if (soft.step<1>(s, c, keep)) {
#pragma unroll
            for (int b = 0; b < DP / 32; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[b][e] *= keep;
        }
        if (more) ATTN_VMCNT(LOADS);
        else ATTN_VMCNT(0);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int u = 0; u < 32 / M::STEP; ++u) {
            const frag p = M::pack(s[0], u);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) M::mma(acc[d], cols_frag<T, PB>(tv, u * M::STEP, d * 32, lane), p);
        }
        lds_reads_done();
        if (more) fetch(lv, v, a.ldv, j + WAVES * 32, at_v);
    }
    // the waves' results joined through LDS, a row's elements next to each other
    __syncthreads();
    float *mine = (float *)lds + (wave * 32 + (lane & 31)) * OUT;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4) *(f32x4 *)(mine + d * 32 + 2 * e + 4 * h) = f32x4{acc[d][e], acc[d][e + 1], acc[d][e + 2], acc[d][e + 3]};
    const float sum = soft.sum + __shfl_xor(soft.sum, 32);
    if (h == 0) wave_base[wave][lane] = soft.base, wave_sum[wave][lane] = sum;
    __syncthreads();
    const int n = min(32, rows - tile * 32);
    for (int row = wave; row < n; row += WAVES) {
        float base = wave_base[0][row], total = 0.f, by[WAVES];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) base = fmaxf(base, wave_base[w][row]);
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            by[w] = wave_base[w][row] == base ? (base == -INFINITY ? 0.f : 1.f) : __builtin_amdgcn_exp2f(wave_base[w][row] - base);
            total += wave_sum[w][row] * by[w];
        }
        const int rt = query_of(a, tile * 32 + row), rh = hk * group + tile * 32 + row - rt * group;
        const float inv = !whole ? 1.f : total == 0.f ? 0.f : 1.f / total;
        const long slot = ((long)unit * a.kv_heads + hk) * 32 + row;
        for (int d = lane; d < a.dim; d += 64) {
            float x = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) x += ((const float *)lds)[(w * 32 + row) * OUT + d] * by[w];
            if (whole) ((T *)a.o)[(long)(sp.q0 + rt) * a.ldo + (long)rh * a.dim + d] = (T)(x * inv);
            else a.part[slot * a.dim + d] = x;
        }
        if (lane == 0) {
            if (!whole) a.part_ml[slot * 2] = base, a.part_ml[slot * 2 + 1] = total;
            else if (a.lse) a.lse[(long)rh * a.q_tokens + sp.q0 + rt] = total == 0.f ? -INFINITY : (base + log2f(total)) * LN2;
        }
    }
}

// the chunks of a tile's rows joined: a wave for each row (4 to 7 us, most of it one wait after another: list, maxima, sums)
template <class T>
__global__ __launch_bounds__(256) void attention_join_kernel(Args a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hk = blockIdx.x % a.kv_heads, unit = blockIdx.x / a.kv_heads;
    const int4 join = a.joins[unit];
    const int parts = join.x, q0 = join.y, tile = join.z, n = min(32, join.w - tile * 32);
    if (!parts) return;
    const long first = ((long)unit * a.kv_heads + hk) * 32, step = (long)a.kv_heads * 32;
    for (int row = blockIdx.y * 4 + wave; row < n; row += gridDim.y * 4) {
        const long slot = first + row;
        // lane i has the maximum and the sum of chunk i, of every 64th one
        float base = -INFINITY;
        for (int i = lane; i < parts; i += 64) base = fmaxf(base, a.part_ml[(slot + i * step) * 2]);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) base = fmaxf(base, __shfl_xor(base, d));
        const float at = base == -INFINITY ? 0.f : base;
        float total = 0.f;
        for (int i = lane; i < parts; i += 64) total += a.part_ml[(slot + i * step) * 2 + 1] * __builtin_amdgcn_exp2f(a.part_ml[(slot + i * step) * 2] - at);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d);
        const int rt = query_of(a, tile * 32 + row), rh = hk * a.group + tile * 32 + row - rt * a.group;
        const float inv = total == 0.f ? 0.f : 1.f / total;
        for (int d = lane; d < a.dim; d += 64) {
            float x = 0.f;
#pragma unroll 4
            for (int i = 0; i < parts; ++i) x += a.part[(slot + i * step) * a.dim + d] * __builtin_amdgcn_exp2f(a.part_ml[(slot + i * step) * 2] - at);
            ((T *)a.o)[(long)(q0 + rt) * a.ldo + (long)rh * a.dim + d] = (T)(x * inv);
        }
        if (lane == 0 && a.lse) a.lse[(long)rh * a.q_tokens + q0 + rt] = total == 0.f ? -INFINITY : (base + log2f(total)) * LN2;
    }
}

// How a forward call runs.
enum Way { ANY, BY_ROWS, BY_KEYS };
struct Plan {
    Way way;
    int tiles, pieces, units;
};

constexpr int keys_waves(int row_bytes) { return row_bytes > 512 ? 2 : 4; }

// Workgroups of attention_keys_kernel that a compute unit holds at once: what its LDS has room for, four at most.  As many pieces as that are
// wanted: twice as many cost a round of first loads and joins more (half, 16 sequences of 8192 keys, one query each, 32 + 8 heads of 128: 118
// us with four pieces a compute unit where two fit, 112 with two; single, heads of 80 over 5 prompts of 500: 76 with four where one fits, 60
// with one), half as many leave none to compute while another one loads (145 us in the first).
int at_once(int dtype, int dim) {
    const int padded = dim <= 96 ? (dim + 31) / 32 * 32 : dim <= 128 ? 128 : 256;
    int bytes = 64;
    while (bytes < padded * (int)dtype_bytes(dtype)) bytes *= 2;
    const int n = 160 * 1024 / (keys_waves(bytes) * 2 * 32 * bytes);
    return n > 4 ? 4 : n;
}

// Tensors that cannot be moved in 16-byte pieces: ANY.  128 rows a workgroup where that gives the chip two rounds of workgroups and
// sequences are not shorter than half of it; else 32, and their keys in pieces while there are fewer workgroups than compute units need.
Plan plan_of(int dtype, int dim, bool vec, int sequences, int q_tokens, int k_tokens, int heads, int kv_heads) {
    Plan p;
    const long rows = (long)q_tokens * (heads / kv_heads), cus = cu_count();
    const long some = sequences < q_tokens ? sequences : q_tokens;
    const long big = (rows + ROWS - 1) / ROWS, small = (rows + 31) / 32;
    p.pieces = p.units = 0;
    p.way = !vec ? ANY : big * kv_heads >= 2 * cus && rows >= some * (ROWS / 2) ? BY_ROWS : BY_KEYS;
    p.tiles = (int)((p.way == BY_KEYS ? small : big) + sequences);
    if (p.way == BY_KEYS) {
        const long groups = (small > some ? small : some) * kv_heads;
        if (groups < 2 * cus && k_tokens > CHUNK_GRAIN) p.pieces = (int)((at_once(dtype, dim) * cus + kv_heads - 1) / kv_heads);
        p.units = p.tiles + p.pieces;
    }
    return p;
}

template <class T, int DP>
int launch_dim(const Args &a, const Plan &p, hipStream_t stream) {
    constexpr int WAVES = keys_waves(row_bytes<T, DP>());
    if (p.way == ANY) hipLaunchKernelGGL((attention_any_kernel<T, DP>), dim3((unsigned)p.tiles * a.kv_heads), dim3(256), 0, stream, a);
    else if (p.way == BY_ROWS) hipLaunchKernelGGL((attention_rows_kernel<T, DP>), dim3((unsigned)p.tiles * a.kv_heads), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((attention_keys_kernel<T, DP, WAVES>), dim3((unsigned)p.units * a.kv_heads), dim3(WAVES * 64), 0, stream, a);
    D8_LAUNCH_CHECK();
    return 0;
}

template <class T>
int launch(const Args &a, const Plan &p, hipStream_t stream) {
    int rc;
    if (a.dim <= 32) rc = launch_dim<T, 32>(a, p, stream);
    else if (a.dim <= 64) rc = launch_dim<T, 64>(a, p, stream);
    else if (a.dim <= 96) rc = launch_dim<T, 96>(a, p, stream);
    else if (a.dim <= 128) rc = launch_dim<T, 128>(a, p, stream);
    else rc = launch_dim<T, 256>(a, p, stream);
    if (rc || !p.pieces) return rc;
    // (a tile has up to 32 rows; where no sequence has more than one query, the heads of a group)
    const int most = a.sequences >= a.q_tokens && a.group < 32 ? a.group : 32;
    hipLaunchKernelGGL(attention_join_kernel<T>, dim3((unsigned)p.units * a.kv_heads, (most + 3) / 4), dim3(256), 0, stream, a);
    D8_LAUNCH_CHECK();
    return 0;
}

size_t part_rows(const Plan &p, int kv_heads) { return p.pieces ? (size_t)p.units * kv_heads * 32 : 0; }
size_t part_bytes(const Plan &p, int kv_heads, int dim) {
    return part_rows(p, kv_heads) * (size_t)(dim + 2) * sizeof(float) + (p.pieces ? (size_t)p.units * sizeof(int4) : 0);
}

}  // namespace

int check(const Args &a, int dtype, const char *name) {
    if (dtype != D8_FLOAT16 && dtype != D8_FLOAT32) return fail(D8_ERR_DTYPE, "%s: type %d is not support", name, dtype);
    D8_REQUIRE(a.sequences >= 0 && a.q_tokens >= 0 && a.k_tokens >= 0, "%s: %d sequences, %d queries, %d keys", name, a.sequences, a.q_tokens, a.k_tokens);
    D8_REQUIRE(a.kv_heads >= 1 && a.heads >= a.kv_heads && a.heads % a.kv_heads == 0, "%s: %d heads cannot share the keys of %d", name, a.heads, a.kv_heads);
    D8_REQUIRE(a.dim >= 1 && a.dim <= MOST_DIM, "%s: a head has 1 to %d elements, not %d", name, (int)MOST_DIM, a.dim);
    const long qrow = (long)a.heads * a.dim, krow = (long)a.kv_heads * a.dim;
    D8_REQUIRE(a.ldq >= qrow && a.ldo >= qrow && a.ldk >= krow && a.ldv >= krow, "%s: rows of %ld and %ld elements do not fit their leading dimensions", name, qrow, krow);
    D8_REQUIRE((long)a.q_tokens * a.heads < (1L << 30) && a.k_tokens < (1 << 30) && a.sequences < (1 << 30), "%s: too many queries, keys or sequences", name);
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
    (void)causal;
    if ((dtype != D8_FLOAT16 && dtype != D8_FLOAT32) || sequences < 0 || q_tokens < 0 || k_tokens < 0 || kv_heads < 1 || heads < kv_heads || dim < 1) return 0;
    if (which == 1) return attention::grad_scratch_bytes(dtype, sequences, q_tokens, k_tokens, heads, kv_heads, dim, causal != 0);
    const attention::Plan p = attention::plan_of(dtype, dim, true, sequences, q_tokens, k_tokens, heads, kv_heads);
    return attention::part_bytes(p, kv_heads, dim);
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
    attention::set_group(a);
    a.vec = attention::in_pieces(dtype, dim, {q, k, v}, {ldq, ldk, ldv});
    // (a tile's rows are addressed by 32 bits)
    const bool fast = a.vec && attention::in_pieces(dtype, dim, {o}, {ldo}) && ldk < (1 << 23) && ldv < (1 << 23);
    const attention::Plan p = attention::plan_of(dtype, dim, fast, sequences, q_tokens, k_tokens, heads, kv_heads);
    const size_t part = attention::part_rows(p, kv_heads), need = attention::part_bytes(p, kv_heads, dim);
    D8_REQUIRE(!need || (scratch && scratch_bytes >= need && ((size_t)scratch & 15) == 0), "attention: 16-byte aligned scratch of %zu bytes is needed, not %zu", need, scratch_bytes);
    D8_REQUIRE((long)(p.tiles + p.pieces) * kv_heads < (1L << 31), "attention: too many sequences");
    a.tiles = p.tiles, a.units = p.units, a.pieces = p.pieces;
    a.joins = (int4 *)scratch, a.part = (float *)(a.joins + (p.pieces ? p.units : 0)), a.part_ml = a.part + part * dim;
    return dtype == D8_FLOAT16 ? attention::launch<f16>(a, p, as_stream(stream)) : attention::launch<float>(a, p, as_stream(stream));
}
