// Attention over a cache in 8-bit pages (cache.h).
//
//   o = softmax(scale q k^T) v,  k = codes * k_scale,  v = codes * v_scale;  the pages' scales go into the scores and the sums, not into the codes:
//   s = (q . codes) (k_scale scale),  o = sum over pages of v_scale (p . codes)
//
// Rows.  The queries of all heads that share keys are one matrix, row r of a sequence query r / group of the kv head's head r % group.
//
// Products.  Both are formed transposed (keys x rows, elements x rows) with 16 x 16 accumulators: lane l has row l % 16, and with it its
// maximum, sum and limit; the probabilities are the next product's right operand where they are.  A lane (r = l % 16, g = l / 16) of tile t of a
// page's keys holds 16 bytes of key 16 (r / 4) + 4 t + r % 4, so that after the product lane group g has keys 16 g .. 16 g + 15 in order: the 16 bytes of
// values [element][token] that a lane reads are then the matching left operand.  So codes go from memory to registers in 16-byte pieces, and are
// converted there: half in pairs, by putting the byte (its sign bit flipped) below the bits of 1024 and taking off 1024 + 128.
//
// KEYS, for few rows: a workgroup has 16 rows, its four waves share out the pages, each by itself and a page ahead, and join through LDS.
// ROWS, for more, and heads of 128 elements at most: eight waves have 16 rows each and go through the pages together; a page's codes
// are converted once and go through LDS as operands, in two buffers.  (512 queries of 4 sequences and 32 heads over 32768 keys of 8: 320 us with every wave converting
// for itself, 123 so.)
//
// All tiles' pages, one after the other, are cut into as many equal runs as workgroups run at once, whatever sequences have how many: a workgroup
// goes through its run and leaves, for a tile that it has not all of, sums in scratch, which a second launch joins.  Cuts are found from the
// lengths on the device, so a call can be captured and replayed as sequences grow.
//
// KEYS is bound by memory (a page and head is 16 KB at 128 elements): 16 queries over 131072 keys of 8 heads of 128, 269 MB, take 60.6 us, 4.4 TB/s, where
// a large copy moves 5.2; single precision 65 us.  ROWS by no unit alone: 1 x 2048 queries of 32 heads over
// 8192 keys take 347 us, 700 TFLOP/s, where a large product of the library makes 1200; counters of the 512 queries above have the vector units, matrix
// instructions' issue among it, busy for 63 % of the time, the matrix units for 30 %, LDS for 38 %.  What takes vector instructions away helps, as long as no
// register more is needed.  (Two sets of rows a wave, which halve what LDS reads and leave two waves a SIMD: 155 us in place of 133; half the waves a phase behind
// the others, no gain; accumulators in units of the pages' scales: 139 for 126.)  Short calls are bound by latency: a wave's
// way from the first length to its last store is 10 us, and the join 4.
//
// Maxima, sums and accumulators are fp32.  Probabilities are halves in the second product (single: two), 2^LIFT times what they are: one of 2^-28 of the row's
// largest so far still has all of a half's bits, and below that they are off by 2^-39 of it, which a million keys make 2^-19.  (As they are, those below 2^-25 would
// be lost from the result and kept in the sum: a first key that takes nearly all the weight, and 131072 others that have 2^-25 each, 0.4 % of the values' size.)
#include "cache.h"
#include "lanes.h"

namespace d8 {
namespace cache {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LIFT = 14.f, LOWER = 1.f / 16384.f;  // (log2 of what probabilities are multiplied by: the largest, 1, stays in half's range; and back)
enum { KEYS_WAVES = 4, KEYS_ROWS = 16, ROWS_WAVES = 8, MANY_ROWS = 128 };

struct Join;

struct AttArgs {
    Pages c;
    const void *q;
    void *o;
    float *lse;   // [heads][tokens]
    float *part;  // [slots][kv_heads][rows of a tile][part_ld], then maximum and sum [slots][kv_heads][rows of a tile][2]
    float *part_ml;
    Join *joins;  // [units]
    long units;
    long ldq, ldo;
    int heads, group, causal, vec;
    int part_ld;  // elements of a row of partial sums: whole pieces of four
    int runs;  // workgroups of a kv head
    float scale;
};

// One sequence: its queries' rows, how many tokens it has (`len`, which places the queries) and keys (those that the table has room for).
struct Seq {
    int q0, n;
    long len;
    int keys;
    long tiles, pages;  // tiles of rows, pages that each goes through (1 where there is none: a result of nothing is written too)
    __device__ __forceinline__ long cost() const { return tiles * pages; }
    template <int R>
    __device__ __forceinline__ void set(const AttArgs &a, int first, int rows, int length) {
        q0 = first, n = rows, len = max(length, 0);
        keys = (int)min(len, (long)a.c.table_pages * PAGE);
        tiles = n ? ((long)n * a.group + R - 1) / R : 0, pages = keys ? (keys + PAGE - 1) / PAGE : 1;
    }
};

// the lane's sequence of the 64 from `first` on; top: the largest start so far (starts as in cache.hip)
template <int R>
__device__ __forceinline__ Seq seqs_from(const AttArgs &a, int first, int &top) {
    const Pages &c = a.c;
    const int lane = threadIdx.x & 63, at = min(first + lane, c.sequences), next = min(first + lane + 1, c.sequences);
    int q0 = min(max(c.starts[at], 0), c.tokens), q1 = min(max(c.starts[next], 0), c.tokens);
    if (__ballot(q0 < top || q1 < q0)) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int q = __shfl_up(q0, d);
            q0 = lane >= d ? max(q0, q) : q0;
        }
        q0 = max(q0, top), q1 = max(q1, q0);
    }
    top = __builtin_amdgcn_readlane(q1, 63);
    Seq s;
    s.set<R>(a, q0, q1 - q0, at < c.sequences ? c.lengths[at] : 0);
    return s;
}

__device__ __forceinline__ int from_lane(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }  // (`lane` as all lanes have it)
__device__ __forceinline__ long from_lane(long x, int lane) {
    return (long)((unsigned long)(unsigned)from_lane((int)(x >> 32), lane) << 32 | (unsigned)from_lane((int)x, lane));
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// What a workgroup knows of all sequences: the lane's of the first 64 with the tiles and costs up to it, and the sums over all.
template <int R>
struct Scan {
    Seq own;
    long tiles_upto, cost_upto, tiles, cost;
    int top;  // largest start of those 64
    __device__ __forceinline__ void begin(const AttArgs &a) {
        top = 0;
        own = seqs_from<R>(a, 0, top);
        tiles_upto = own.tiles, cost_upto = own.cost();
        if (a.c.sequences > 1) tiles_upto = sum_upto_lane(tiles_upto), cost_upto = sum_upto_lane(cost_upto);
        const int last = min(a.c.sequences, 64) - 1;
        tiles = from_lane(tiles_upto, last), cost = from_lane(cost_upto, last);
        int at = top;
        for (int first = 64; first < a.c.sequences; first += 64) {
            const Seq s = seqs_from<R>(a, first, at);
            tiles += from_lane(sum_upto_lane(s.tiles), 63), cost += from_lane(sum_upto_lane(s.cost()), 63);
        }
    }
    // the sequence of page `at` of the list: the list's pages and tiles before it
    __device__ __forceinline__ bool locate(const AttArgs &a, long at, Seq &seq, int &s, long &cost_base, long &tile_base) const {
        Seq x = own;
        long t = tiles_upto, c = cost_upto, tiles_before = 0, cost_before = 0;
        int start = top;
        for (int first = 0; first < a.c.sequences; first += 64) {
            if (first) {
                x = seqs_from<R>(a, first, start);
                t = sum_upto_lane(x.tiles), c = sum_upto_lane(x.cost());
            }
            const unsigned long long past = __ballot(first + (int)(threadIdx.x & 63) < a.c.sequences && cost_before + c > at);
            if (past) {
                const int l = __ffsll((long long)past) - 1;
                s = uniform(first + l);
                cost_base = cost_before + from_lane(c - x.cost(), l), tile_base = tiles_before + from_lane(t - x.tiles, l);
                seq.q0 = from_lane(x.q0, l), seq.n = from_lane(x.n, l), seq.len = from_lane(x.len, l), seq.keys = from_lane(x.keys, l);
                seq.tiles = from_lane(x.tiles, l), seq.pages = from_lane(x.pages, l);
                return true;
            }
            const int last = min(a.c.sequences - first, 64) - 1;
            cost_before += from_lane(c, last), tiles_before += from_lane(t, last);
        }
        return false;
    }
};

// The next sequence that has queries, after `seq`, number s; false beyond the last.
template <int R>
__device__ __forceinline__ bool advance(const AttArgs &a, Seq &seq, int &s) {
    int end = seq.q0 + seq.n;
    while (++s < a.c.sequences) {
        const int first = end;
        end = uniform(max(first, min(a.c.starts[s + 1], a.c.tokens)));
        if (end == first) continue;
        seq.set<R>(a, first, end - first, uniform(a.c.lengths[s]));
        return true;
    }
    return false;
}

// What the second launch joins of a tile: how many runs have a part of it (0: nothing to join), the first of them, the sequence's first query, and
// the tile's first row and those from it on.
struct Join {
    int parts, run, q0, row0, rows, pad[3];
};

// How long the runs of a call are: equal, but not so short that a tile's many pieces cost more to join than is gained: KEYS stays at a tile, or a page a
// wave, ROWS at a quarter of a tile, or four pages.  (One token over 8000 keys of 8 heads: 17 us so, 22 with runs of a page; 256 queries of 8 heads over
// 4096 keys in single, 38 and 50.  Runs longer than a tile go through short sequences one after the other: 16 of 100 keys took 24 us with four pages, 17 so.)
template <int R>
__device__ __forceinline__ long run_of(long total, long tiles, int runs) {
    const long even = (total + runs - 1) / runs, mean = (total + tiles - 1) / max(tiles, 1L);
    return max(even, min(R == KEYS_ROWS ? mean : mean / 4, 4L));
}

// ---- operands -------------------------------------------------------------------------------------------------------
// 16 codes as halves, exactly
__device__ __forceinline__ void to_halves(const i32x4 &codes, f16x8 (&out)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        f16x2 p[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const unsigned w = (unsigned)codes[2 * i + e] ^ 0x80808080u;
            const f16x2 off = {(f16)1152.f, (f16)1152.f};
            p[2 * e] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - off;
            p[2 * e + 1] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - off;
        }
        out[i] = __builtin_shufflevector(__builtin_shufflevector(p[0], p[1], 0, 1, 2, 3), __builtin_shufflevector(p[2], p[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// sixteen numbers as halves, two a conversion, to nearest
__device__ __forceinline__ void round_halves(const float (&x)[16], f16x8 (&out)[2]) {
    f16x2 p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __builtin_convertvector((f32x2){x[2 * i], x[2 * i + 1]}, f16x2);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        out[i] = __builtin_shufflevector(__builtin_shufflevector(p[4 * i], p[4 * i + 1], 0, 1, 2, 3), __builtin_shufflevector(p[4 * i + 2], p[4 * i + 3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

// What meets the codes in a product: a query's elements, or a page's probabilities.  Codes are halves exactly, so single precision runs on the same
// instructions, its numbers as sums of halves, each what the ones before leave: queries of three (33 bits, all of them), probabilities of two (22 bits: off by
// 2^-22 each at most, which the sum over keys averages).  Single precision's own matrix instructions take eight times as long as half's for a product: 16
// queries over 131072 keys, 32 + 8 heads of 128, in 161 us.
template <class T>
struct Precision;
template <>
struct Precision<f16> {
    static constexpr int QUERY = 1, WEIGHT = 1;
};
// So that what is left stays in half's range too, a row of queries is brought to 2^13 .. 2^14 by a power of two, as probabilities are by LIFT.
template <>
struct Precision<float> {
    static constexpr int QUERY = 3, WEIGHT = 2;
};

template <int PARTS>
__device__ __forceinline__ void split(float (&x)[16], f16x8 (&out)[PARTS][2]) {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        round_halves(x, out[p]);
        if (p + 1 < PARTS)
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] -= (float)out[p][i >> 3][i & 7];
    }
}

__device__ __forceinline__ f32x4 mma(const f16x8 &a, const f16x8 &b, const f32x4 &c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// the larger, and the sum, of the four lanes that have a row (l, l + 16, l + 32, l + 48)
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u32x2 half_rows(float x) { return __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false)); }
__device__ __forceinline__ u32x2 halves(float x) { return __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false)); }
// (asm: fmaxf quiets each operand first that the compiler cannot tell to be a quiet NaN or none)
__device__ __forceinline__ float larger(float a, float b) {
    float c;
    asm("v_max_f32 %0, %1, %2" : "=v"(c) : "v"(a), "v"(b));
    return c;
}
__device__ __forceinline__ float row_max(float x) {
    u32x2 y = half_rows(x);
    y = halves(larger(__uint_as_float(y[0]), __uint_as_float(y[1])));
    return larger(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
__device__ __forceinline__ float row_sum(float x) {
    u32x2 y = half_rows(x);
    y = halves(__uint_as_float(y[0]) + __uint_as_float(y[1]));
    return __uint_as_float(y[0]) + __uint_as_float(y[1]);
}

// ---- one wave, 16 rows ----------------------------------------------------------------------------------------------
// NC: chunks of 64 elements of a head.
// The lane, and a number that all lanes have, to the compiler others at every tile: what depends on them (addresses, comparisons with a head's elements,
// reciprocals of divisors) would be kept for the whole launch in registers that the products need: 16 queries over 131072 keys in single, 75 us with and 66 without.
__device__ __forceinline__ int fresh_lane() {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}
template <class N>
__device__ __forceinline__ N fresh(N x) {
    asm volatile("" : "+s"(x));
    return x;
}

template <class T, int NC>
struct Wave {
    typedef Precision<T> P;
    f16x8 q[NC][P::QUERY][2];
    float q_scale;  // of the lane's row (single precision)
    f32x4 o[NC * 4];
    float m, sum;  // of scores times log2 e; the lane's part of the sum, 2^LIFT times it
    int limit;     // keys that the lane's row sees

    const T *from;  // the lane's row of queries, or another's where it has none
    bool there;

    // rows row0 .. of the sequence (those beyond `rows` are zero and see nothing)
    __device__ __forceinline__ void begin(const AttArgs &a, const Seq &s, int head, long row0, long rows) {
        const long row = row0 + (fresh_lane() & 15);
        there = row < rows;
        const int group = fresh(a.group), t = there ? (int)row / group : 0, h = there ? (int)row - t * group : 0;
        const long sees = a.causal ? t + s.len - s.n + 1 : s.len;
        limit = there ? (int)min(max(sees, 0L), (long)s.keys) : 0;
        from = (const T *)a.q + (s.q0 + (long)t) * a.ldq + ((long)head * group + h) * a.c.dim;
        m = -INFINITY, sum = 0.f;
#pragma unroll
        for (int i = 0; i < NC * 4; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    __device__ __forceinline__ void load_queries(const AttArgs &a) {
        const int g = fresh_lane() >> 4;
        const int dim = fresh(a.c.dim);
        float x[NC][16], largest = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = c * 64 + g * 16;
            if (a.vec) {  // (dim is whole pieces; where there are none, the first is loaded for nothing)
                constexpr int V = 16 / sizeof(T);
                typedef T piece __attribute__((ext_vector_type(V)));
#pragma unroll
                for (int i = 0; i < 16; i += V) {
                    const bool some = there && d + i < dim;
                    const piece p = *(const piece *)(from + (some ? d + i : 0));
#pragma unroll
                    for (int e = 0; e < V; ++e) x[c][i + e] = some ? (float)p[e] : 0.f;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[c][i] = there && d + i < dim ? (float)from[d + i] : 0.f;
            }
            if (P::QUERY > 1)
#pragma unroll
                for (int i = 0; i < 16; ++i) largest = fmaxf(largest, fabsf(x[c][i]));
        }
        q_scale = 1.f;
        if (P::QUERY > 1) {
            largest = row_max(largest);
            // 2^(e - 13) of a largest element 1.f 2^e, at least 2^-100; 1 for rows of zeros, infinities and NaN
            const int e = max((int)(__float_as_uint(largest) >> 23) - 13, 27);
            if (largest > 0.f && largest < INFINITY) q_scale = __uint_as_float((unsigned)e << 23);
            const float back = 1.f / q_scale;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[c][i] *= back;
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) split<P::QUERY>(x[c], q[c]);
    }

    // where a lane's operands lie in a page and head: its key's row of tile t (16 bytes of chunk n; beyond the head any codes, times zeros of q),
    // its element's of tile i
    static __device__ __forceinline__ const i32x4 *key_at(const Pages &c, const signed char *page, int lane, int t, int n) {
        const int r = lane & 15, d = n * 64 + (lane >> 4) * 16;
        return (const i32x4 *)(page + ((r >> 2) * 16 + (r & 3) + 4 * t) * c.pitch + (d < c.pitch ? d : 0));
    }
    static __device__ __forceinline__ const i32x4 *value_at(const signed char *page, int lane, int i) {
        return (const i32x4 *)(page + (i * 16 + (lane & 15)) * PAGE + (lane >> 4) * 16);
    }

    // Scores of a page whose first place is `at` to weights; accumulators and sums to the new maximum.  hidden: some row does not see all of
    // the page (or there is none).  `into`: what the page's sums are scaled by, 0 where the lane's row sees none of it.
    __device__ __forceinline__ void weigh(const f32x4 (&sc)[4], int g, int at, bool there, bool hidden, float k_scale, float v_scale, f16x8 (&p)[P::WEIGHT][2], float &into) {
#pragma clang fp contract(off)  // (a fused product less its rounded maximum is off by half a step of that, which sum and result
        // share: 2^-15 at most below LARGE, but anything where scores are larger)
        constexpr float LARGE = 1024.f;
        float x[16], by = P::QUERY > 1 ? k_scale * q_scale : k_scale;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = sc[i >> 2][i & 3];
        into = v_scale;
        if (hidden || by < 0.f) {  // (below, the largest score is taken for the largest product)
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = there && at + g * 16 + i < limit ? x[i] * by : -INFINITY;
            by = 1.f;
            into = there && at < limit ? v_scale : 0.f;
        }
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, x[i]);
        top = fmaxf(row_max(top) * by, m);
        const float base = top == -INFINITY ? 0.f : top;
        if (__ballot(top != m)) {
            const float less = __builtin_amdgcn_exp2f(m - base);
            sum *= less;
#pragma unroll
            for (int i = 0; i < NC * 4; ++i) o[i] *= less;
            m = top;
        }
        float add = 0.f, shift = LIFT - base;
        if (__ballot(fabsf(base) >= LARGE)) {  // (nor is LIFT added to a maximum that large: from 2^25 on it would be rounded to 16, which is past half's range)
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = x[i] * by - base;
            by = 1.f, shift = LIFT;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], by, shift));
            add += x[i];
        }
        split<P::WEIGHT>(x, p);
        sum += add;
    }

    // 64 pages of a sequence: lane i has page, and scales, of number i (that of values for probabilities 2^LIFT times what they are)
    struct List {
        int ids, there;
        float ks, vs;
        __device__ __forceinline__ void load(const Pages &c, int s, int head, int first, int count, int step) {
            const int i = threadIdx.x & 63, p = i < count ? c.page_of(s, first + i * step) : -1;
            there = p >= 0, ids = max(p, 0), ks = vs = 0.f;
            if (p >= 0) ks = c.k_scales[(long)p * c.kv_heads + head], vs = c.v_scales[(long)p * c.kv_heads + head] * LOWER;
        }
        __device__ __forceinline__ int id(int n) const { return __builtin_amdgcn_readlane(ids, n); }
        __device__ __forceinline__ bool is(int n) const { return __builtin_amdgcn_readlane(there, n) != 0; }
        __device__ __forceinline__ float k(int n) const { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks), n)); }
        __device__ __forceinline__ float v(int n) const { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), n)); }
    };

    // pages that the wave's rows see at most (the later a row's query, the more)
    __device__ __forceinline__ int most() const {
        int n = limit;
        n = over_lanes<16>(n, [](int x, int y) { return max(x, y); });
        return uniform((n + PAGE - 1) / PAGE);
    }

    // KEYS: `count` pages, 64 at most, first, first + step, ... of sequence s, by this wave alone.  fresh: load the queries too
    __device__ __forceinline__ void pages(const AttArgs &a, int s, int head, int first, int count, int step, bool fresh) {
        const Pages &c = a.c;
        const int lane = fresh_lane(), least = uniform(limit);
        List list;
        list.load(c, s, head, first, count, step);
        i32x4 kr[4][NC], vr[NC * 4];
        auto fetch_keys = [&](int page) {
            const signed char *from = c.k_codes + c.tile(page, head);
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int n = 0; n < NC; ++n) kr[t][n] = *key_at(c, from, lane, t, n);
        };
        auto fetch_values = [&](int page) {
            const signed char *from = c.v_codes + c.tile(page, head);
#pragma unroll
            for (int i = 0; i < NC * 4; ++i)
                if (i * 16 < c.pitch) vr[i] = *value_at(from, lane, i);
        };
        fetch_keys(list.id(0)), fetch_values(list.id(0));
        if (fresh) load_queries(a);
        for (int n = 0; n < count; ++n) {
            const int at = (first + n * step) * PAGE;
            const bool there = list.is(n), more = n + 1 < count;
            const int next = list.id(more ? n + 1 : n);
            f32x4 sc[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < NC; ++i) {
                    f16x8 k[2];
                    to_halves(kr[t][i], k);
#pragma unroll
                    for (int e = 0; e < P::QUERY; ++e) sc[t] = mma(k[1], q[i][e][1], mma(k[0], q[i][e][0], sc[t]));
                }
            }
            if (more) fetch_keys(next);
            f16x8 p[P::WEIGHT][2];
            float into;
            weigh(sc, lane >> 4, at, there, !there || at + PAGE > least, list.k(n) * (a.scale * LOG2E), list.v(n), p, into);
#pragma unroll
            for (int i = 0; i < NC * 4; ++i) {
                if (i * 16 >= c.pitch) continue;
                f16x8 v[2];
                to_halves(vr[i], v);
                f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < P::WEIGHT; ++e) acc = mma(v[1], p[e][1], mma(v[0], p[e][0], acc));
                o[i] += acc * into;
            }
            if (more) fetch_values(next);
        }
    }

    // ROWS: `count` pages, 64 at most, from `first` on by all waves of a workgroup, each with rows of its own.  A page's codes are converted once, an
    // eighth by each wave, and go through LDS as operands, lane by lane: [keys' tile][chunk][half], then [values' tile][half], a buffer for every other page.
    __device__ __forceinline__ void pages_together(const AttArgs &a, int s, int head, int first, int count, int wave, f16x8 (*stages)[16 * NC][64]) {
        const Pages &c = a.c;
        const int lane = fresh_lane(), own_end = most(), least = uniform(limit);
        List list;
        list.load(c, s, head, first, count, 1);
        i32x4 share[NC];
        auto fetch = [&](int page) {
            const signed char *k = c.k_codes + c.tile(page, head), *v = c.v_codes + c.tile(page, head);
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                const int item = wave + ROWS_WAVES * n;
                if (item < 4 * NC) share[n] = *key_at(c, k, lane, item / NC, item % NC);
                else if ((item - 4 * NC) * 16 < c.pitch) share[n] = *value_at(v, lane, item - 4 * NC);
            }
        };
        auto stage = [&](int to) {
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                f16x8 x[2];
                to_halves(share[n], x);
                stages[to][(wave + ROWS_WAVES * n) * 2][lane] = x[0], stages[to][(wave + ROWS_WAVES * n) * 2 + 1][lane] = x[1];
            }
        };
        fetch(list.id(0));
        stage(0);
        if (count > 1) fetch(list.id(1));
        for (int n = 0; n < count; ++n) {
            __syncthreads();  // the page is in LDS, and nobody reads the one before it any more
            const f16x8 (*from)[64] = stages[n & 1];
            const int at = (first + n) * PAGE;
            const bool there = list.is(n);
            if (first + n < own_end) {
                // fragments in groups of four, the next on their way while one is multiplied; kept in that order (left to itself the compiler reads them
                // all at once, which takes more registers than four waves a SIMD leave)
                f16x8 ahead[2][4];
                auto group = [&](int k) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        ahead[k & 1][i] = from[4 * k + i][lane];
                };
                f32x4 sc[4];
                group(0);
#pragma unroll
                for (int t = 0; t < 4; ++t) sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < 2 * NC; ++k) {
                    group(k + 1);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int at = 4 * k + i, t = at / (2 * NC), c = at % (2 * NC);
#pragma unroll
                        for (int e = 0; e < P::QUERY; ++e) sc[t] = mma(ahead[k & 1][i], q[c >> 1][e][c & 1], sc[t]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                f16x8 p[P::WEIGHT][2];
                float into;
                weigh(sc, lane >> 4, at, there, !there || at + PAGE > least, list.k(n) * (a.scale * LOG2E), list.v(n), p, into);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int k = 0; k < 2 * NC; ++k) {
                    if (k + 1 < 2 * NC) group(2 * NC + k + 1);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {  // (elements beyond the head, whatever they are, are not stored)
                        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int e = 0; e < P::WEIGHT; ++e) acc = mma(ahead[k & 1][2 * i + 1], p[e][1], mma(ahead[k & 1][2 * i], p[e][0], acc));
                        o[k * 2 + i] += acc * into;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (n + 1 < count) stage((n + 1) & 1);
            if (n + 2 < count) fetch(list.id(n + 2));
        }
        __syncthreads();  // (the next pages take the same LDS)
    }
};

// A lane's four elements 4 g .. of a tile of 16 of row `row`'s result, divided by the sum.
template <class T>
__device__ __forceinline__ void put(const AttArgs &a, T *to, int d, const f32x4 &x, float by) {
    if (d + 4 <= a.c.dim && a.vec) {
        typedef T quad __attribute__((ext_vector_type(4)));
        quad v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)within<T>(x[e] * by);
        *(quad *)(to + d) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < a.c.dim) to[d + e] = (T)within<T>(x[e] * by);
    }
}

template <class T, int NC, bool ROWS>
__global__ __launch_bounds__((ROWS ? ROWS_WAVES : KEYS_WAVES) * 64, NC == 4 ? 1 : ROWS && sizeof(T) == 2 ? 4 : 2) void attention_cache_kernel(AttArgs a) {
    constexpr int WAVES = ROWS ? ROWS_WAVES : KEYS_WAVES, R = ROWS ? MANY_ROWS : KEYS_ROWS;  // rows of a tile
    // Queries are loaded once the loads of a tile's first page have set out, where registers leave room for both: 16 queries over 131072 keys take 1 us less so
    // in half, and 4 us more in single.
    constexpr bool LATE = !ROWS && sizeof(T) == 2;
    __shared__ f16x8 stages[ROWS ? 2 : 1][ROWS ? 16 * NC : 1][64];
    __shared__ f32x4 others[ROWS ? 1 : WAVES][ROWS ? 1 : NC * 4][64];
    __shared__ float2 stats[ROWS ? 1 : WAVES][16];
    const int wave = uniform((int)(threadIdx.x >> 6));
    const int head = blockIdx.x % a.c.kv_heads, run = blockIdx.x / a.c.kv_heads;
    Scan<R> scan;
    scan.begin(a);
    const long total = scan.cost, length = run_of<R>(total, scan.tiles, a.runs);
    const long last = min((run + 1) * length, total);
    long at = run * length;
    if (run == 0 && head == 0)  // tiles that the launch has room for and the sequences do not have
        for (long i = scan.tiles + threadIdx.x; i < a.units; i += WAVES * 64) a.joins[i].parts = 0;
    if (at >= last) return;
    Seq seq;
    int s;
    long base, tile_base;
    if (!scan.locate(a, at, seq, s, base, tile_base)) return;
    Wave<T, NC> w;
    for (;;) {
        const long after = base + seq.cost(), stop = min(fresh(last), after);
        while (at < stop) {
            const long ahead = at - base, tile = ahead < seq.pages ? 0 : ahead / fresh(seq.pages);
            const int first = (int)(at - base - tile * seq.pages), end = (int)min(seq.pages, first + (stop - at));
            const bool whole = first == 0 && end == seq.pages;
            const long rows = (long)seq.n * a.group, row0 = tile * R + (ROWS ? wave * 16 : 0), slot = run + tile_base + tile;
            if (first == 0 && head == 0 && threadIdx.x == 0) {  // (the tile's first page: every head's parts are alike)
                const long to = at + seq.pages - 1, run_length = fresh(length);
                const int parts = to < (run + 1) * run_length ? 1 : (int)(to / run_length) - run + 1;
                a.joins[tile_base + tile] = Join{parts == 1 ? 0 : parts, run, seq.q0, (int)(tile * R), (int)(rows - tile * R), {0, 0, 0}};
            }
            w.begin(a, seq, head, row0, rows);
            if (!LATE) w.load_queries(a);
            if constexpr (ROWS) {
                // what the tile's last row sees: all waves go through as many pages
                const int t = ((int)min((tile + 1) * R, rows) - 1) / fresh(a.group);
                const long sees = min(max(a.causal ? t + seq.len - seq.n + 1 : seq.len, 0L), (long)seq.keys);
                const int upto = min(end, (int)((sees + PAGE - 1) / PAGE));
                for (int i = first; i < upto; i += 64) w.pages_together(a, s, head, i, min(64, upto - i), wave, stages);
            } else {
                const int upto = min(end, w.most());
                for (int i = first + wave; i < upto; i += 64 * WAVES) w.pages(a, s, head, i, min(64, (upto - i + WAVES - 1) / WAVES), WAVES, LATE && i == first + wave);
            }
            const int lane = fresh_lane(), r = lane & 15, g = lane >> 4;
            at += end - first;
            w.sum = row_sum(w.sum) * LOWER;
            if constexpr (!ROWS) {
#pragma unroll
                for (int i = 0; i < NC * 4; ++i) others[wave][i][lane] = w.o[i];
                if (g == 0) stats[wave][r] = make_float2(w.m, w.sum);
                __syncthreads();
                float top = -INFINITY, by[WAVES];
#pragma unroll
                for (int k = 0; k < WAVES; ++k) top = fmaxf(top, stats[k][r].x);
                const float from = top == -INFINITY ? 0.f : top;
                w.m = top, w.sum = 0.f;
#pragma unroll
                for (int k = 0; k < WAVES; ++k) {
                    by[k] = __builtin_amdgcn_exp2f(stats[k][r].x - from);
                    w.sum += stats[k][r].y * by[k];
                }
#pragma unroll
                for (int i = 0; i < NC * 4; ++i) {
                    if (i % WAVES != wave) continue;
                    w.o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < WAVES; ++k) w.o[i] += others[k][i][lane] * by[k];
                }
                __syncthreads();
            }
            const long row = row0 + r;
            if (row >= rows) continue;
            if (whole) {
                const int group = fresh(a.group), t = (int)row / group, h = head * group + (int)row - t * group;
                T *to = (T *)a.o + (seq.q0 + (long)t) * a.ldo + (long)h * a.c.dim;
                const float inv = w.sum == 0.f ? 0.f : 1.f / w.sum;
#pragma unroll
                for (int i = 0; i < NC * 4; ++i)
                    if (ROWS || i % WAVES == wave) put<T>(a, to, i * 16 + g * 4, w.o[i], inv);
                if (a.lse && g == 0 && (ROWS || wave == 0)) a.lse[(long)h * a.c.tokens + seq.q0 + t] = w.sum == 0.f ? -INFINITY : (w.m + log2f(w.sum)) * LN2;
            } else {
                const long place = (slot * a.c.kv_heads + head) * R + (row - tile * R);
                float *to = a.part + place * a.part_ld;
#pragma unroll
                for (int i = 0; i < NC * 4; ++i)
                    if ((ROWS || i % WAVES == wave) && i * 16 + g * 4 < a.part_ld) *(f32x4 *)(to + i * 16 + g * 4) = w.o[i];
                if (g == 0 && (ROWS || wave == 0)) *(float2 *)(a.part_ml + place * 2) = make_float2(w.m, w.sum);
            }
        }
        if (at >= fresh(last)) return;
        base = after, tile_base += seq.tiles;
        if (!advance<R>(a, seq, s)) return;
    }
}

// The runs' sums of a tile's rows joined: half a wave a row, four elements a lane.  The first parts' sums are loaded before their maxima are known.
template <class T, int R>
__global__ __launch_bounds__(256) void attention_cache_join_kernel(AttArgs a) {
    const int half = threadIdx.x & 31, head = blockIdx.x % a.c.kv_heads, unit = blockIdx.x / a.c.kv_heads, row = blockIdx.y * 8 + (threadIdx.x >> 5);
    const Join join = a.joins[unit];
    const int parts = join.parts;
    if (!parts || row >= min(R, join.rows)) return;
    const long step = (long)a.c.kv_heads * R, place = (((long)join.run + unit) * a.c.kv_heads + head) * R + row;
    const float2 *ml = (const float2 *)a.part_ml + place;
    const float *from = a.part + place * a.part_ld;
    constexpr int BATCH = 8;
    f32x4 batch[BATCH];
    auto load = [&](int i, int d) {  // parts i .. (those beyond the last: it again, for weights of 0)
        const float *of = from + (d + half * 4 < a.part_ld ? d + half * 4 : 0);
#pragma unroll
        for (int k = 0; k < BATCH; ++k) batch[k] = *(const f32x4 *)(of + min(i + k, parts - 1) * step * a.part_ld);
    };
    load(0, 0);
    const float2 mine = half < parts ? ml[half * step] : make_float2(-INFINITY, 0.f);
    float top = mine.x;
    for (int i = half + 32; i < parts; i += 32) top = fmaxf(top, ml[i * step].x);
    top = over_lanes<32>(top, larger);
    const float at = top == -INFINITY ? 0.f : top, weight = __builtin_amdgcn_exp2f(mine.x - at);
    float sum = mine.y * weight;
    for (int i = half + 32; i < parts; i += 32) sum += ml[i * step].y * __builtin_amdgcn_exp2f(ml[i * step].x - at);
    sum = over_lanes<32>(sum, [](float x, float y) { return x + y; });
    const int t = (join.row0 + row) / a.group, h = head * a.group + join.row0 + row - t * a.group;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T *to = (T *)a.o + ((long)join.q0 + t) * a.ldo + (long)h * a.c.dim;
    for (int d = 0; d < a.c.dim; d += 128) {
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
        float w = weight;
        for (int i = 0; i < parts; i += BATCH) {
            if (i && !(i & 31)) w = i + half < parts ? __builtin_amdgcn_exp2f(ml[(i + half) * step].x - at) : 0.f;
            if (i || d) load(i, d);
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                const float by = __shfl(w, (i & 31) + k, 32);
                if (i + k < parts) x += batch[k] * by;
            }
        }
        if (d + half * 4 < a.c.dim) put<T>(a, to, d + half * 4, x, inv);
    }
    if (half == 0 && a.lse) a.lse[(long)h * a.c.tokens + join.q0 + t] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * LN2;
}

// How a call runs: rows of a tile, runs of a kv head, tiles of all sequences at most, and slots of partial sums (a run's and a tile's numbers added: each
// step from piece to piece of the list is to the next run or the next tile, so no two pieces share a slot).
struct Plan {
    bool rows;
    int tile, runs;
    long units, slots;
};

Plan plan_of(int dtype, int sequences, int tokens, int table_pages, int heads, int kv_heads, int dim) {
    Plan p;
    const long group = heads / kv_heads, all = (long)tokens * group, some = sequences < tokens ? sequences : tokens;
    // Rows of a sequence in the mean from which on ROWS is faster (us with and without: half, 48 over 4000 keys of 8 heads 16 / 18, 64 over 8192 of 4 sequences and
    // 8 heads 39 / 45, 32 over 16384 of 8 heads 25 / 22; single, whose ROWS leave two waves a SIMD, 64 as above 57 / 48, 80 over 16000 of 8 heads of 64 25 / 25).
    const int from = dtype == D8_FLOAT16 ? 33 : 96;
    p.rows = dim <= 128 && some && all / some >= from;
    p.tile = p.rows ? MANY_ROWS : KEYS_ROWS;
    p.units = all / p.tile + some;
    const int held = dim > 128 || (p.rows && dtype == D8_FLOAT32) ? 1 : 2;  // workgroups whose registers a compute unit holds
    const long at_once = ((long)held * cu_count() + kv_heads - 1) / kv_heads, most = p.units * (table_pages ? table_pages : 1);
    p.runs = (int)(at_once < most ? at_once : most);
    p.slots = p.units + p.runs;
    return p;
}

int part_ld_of(int dim) { return (dim + 3) / 4 * 4; }
size_t scratch_of(const Plan &p, int kv_heads, int dim) {
    return sizeof(Join) * p.units + sizeof(float) * (size_t)p.slots * kv_heads * p.tile * (part_ld_of(dim) + 2);
}

template <class T, int NC>
void launch(const AttArgs &a, const Plan &p, hipStream_t stream) {
    const dim3 grid((unsigned)(p.runs * a.c.kv_heads));
    if constexpr (NC <= 2) {
        if (p.rows) {
            hipLaunchKernelGGL((attention_cache_kernel<T, NC, true>), grid, dim3(ROWS_WAVES * 64), 0, stream, a);
            return;
        }
    }
    hipLaunchKernelGGL((attention_cache_kernel<T, NC, false>), grid, dim3(KEYS_WAVES * 64), 0, stream, a);
}

template <class T>
int launch_all(const AttArgs &a, const Plan &p, hipStream_t stream) {
    if (a.c.dim <= 64) launch<T, 1>(a, p, stream);
    else if (a.c.dim <= 128) launch<T, 2>(a, p, stream);
    else launch<T, 4>(a, p, stream);
    D8_LAUNCH_CHECK();
    const dim3 join((unsigned)(p.units * a.c.kv_heads), p.tile / 8);
    if (p.rows) hipLaunchKernelGGL((attention_cache_join_kernel<T, MANY_ROWS>), join, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((attention_cache_join_kernel<T, KEYS_ROWS>), join, dim3(256), 0, stream, a);
    D8_LAUNCH_CHECK();
    return 0;
}

bool sizes(int dtype, int sequences, int tokens, int heads, int kv_heads, int dim) {
    return (dtype == D8_FLOAT16 || dtype == D8_FLOAT32) && sequences >= 0 && sequences < (1 << 24) && tokens >= 0 && kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0 &&
           dim >= 1 && dim <= MOST_DIM && (long)tokens * heads < (1L << 30);
}

}  // namespace
}  // namespace cache
}  // namespace d8

using namespace d8;

extern "C" size_t d8_attention_cache_scratch_bytes(int dtype, int sequences, int q_tokens, int table_pages, int heads, int kv_heads, int dim) {
    if (!cache::sizes(dtype, sequences, q_tokens, heads, kv_heads, dim) || !sequences || !q_tokens || table_pages < 0 || table_pages >= (1 << 24)) return 0;
    return cache::scratch_of(cache::plan_of(dtype, sequences, q_tokens, table_pages, heads, kv_heads, dim), kv_heads, dim);
}

extern "C" int d8_attention_cache(int dtype, const void *q, long ldq, const signed char *k_codes, const float *k_scales, const signed char *v_codes,
                                  const float *v_scales, void *o, long ldo, float *lse, const int *starts, const int *lengths, const int *table, int sequences,
                                  int q_tokens, int table_pages, int pages, int heads, int kv_heads, int dim, float scale, int causal, void *scratch,
                                  size_t scratch_bytes, void *stream) {
    cache::AttArgs a;
    memset(&a, 0, sizeof(a));
    a.c = {(signed char *)k_codes, (signed char *)v_codes, (float *)k_scales, (float *)v_scales, starts, lengths, table, sequences, q_tokens, pages ? table_pages : 0, pages,
           kv_heads, dim, (int)cache::pitch_of(dim)};
    if (int rc = cache::check(a.c, dtype, "attention_cache")) return rc;
    D8_REQUIRE(heads >= kv_heads && heads % kv_heads == 0, "attention_cache: %d heads cannot share the keys of %d", heads, kv_heads);
    D8_REQUIRE(cache::sizes(dtype, sequences, q_tokens, heads, kv_heads, dim), "attention_cache: too many queries");
    D8_REQUIRE(scale == scale, "attention_cache: the scale is no number");
    if (!sequences || !q_tokens) return 0;
    D8_REQUIRE(q && o, "attention_cache: null tensor");
    D8_REQUIRE(ldq >= (long)heads * dim && ldo >= (long)heads * dim, "attention_cache: rows of %ld elements do not fit their leading dimensions", (long)heads * dim);
    const cache::Plan p = cache::plan_of(dtype, sequences, q_tokens, table_pages, heads, kv_heads, dim);
    const size_t need = cache::scratch_of(p, kv_heads, dim);
    D8_REQUIRE(scratch && scratch_bytes >= need && ((size_t)scratch & 15) == 0, "attention_cache: 16-byte aligned scratch of %zu bytes is needed, not %zu", need, scratch_bytes);
    D8_REQUIRE(p.units * kv_heads < (1L << 24), "attention_cache: too many tokens and sequences for a launch");
    const int v = 16 / (int)dtype_bytes(dtype);
    a.q = q, a.ldq = ldq, a.o = o, a.ldo = ldo, a.lse = lse, a.heads = heads, a.group = heads / kv_heads, a.causal = causal != 0, a.scale = scale, a.runs = p.runs;
    a.vec = dim % v == 0 && ldq % v == 0 && ldo % v == 0 && (((size_t)q | (size_t)o) & 15) == 0;
    a.part_ld = cache::part_ld_of(dim), a.units = p.units;
    a.joins = (cache::Join *)scratch, a.part = (float *)(a.joins + p.units), a.part_ml = a.part + (size_t)p.slots * kv_heads * p.tile * a.part_ld;
    return dtype == D8_FLOAT16 ? cache::launch_all<f16>(a, p, as_stream(stream)) : cache::launch_all<float>(a, p, as_stream(stream));
}
