// What the attention kernels share: their arguments, how a workgroup finds its sequence, operand fragments of the 32 x 32 matrix
// instructions in half and single precision.
//
// Rows.  The queries of all heads that share keys and values are one matrix: row r of a sequence is query r / group of head
// r % group of the kv head's group.  A tile of keys then serves every one of them, and a step of decoding (one query) has `group`
// rows instead of one.
//
// Products.  Both types use 32 x 32 accumulators: element (i, j) of a product of a 32 x k by a k x 32 matrix lies in lane
// j + 32 h, register 4 b + e with i = 8 b + 4 h + e (h = lane / 32).  An operand fragment is 16 bytes a lane: lane (i, h) holds row i of
// the left operand (column i of the right one) at k = 8 h .. 8 h + 7 of 16 (half) or k = 4 h .. 4 h + 3 of 8 (single, where four
// instructions take one value each).  The order of k within a product does not matter as long as both operands have the same one;
// that is what lets the accumulators of one product be the right operand of the next without leaving their lanes: registers
// 8 u .. 8 u + 7 (half), 4 u .. 4 u + 3 (single) of lane (j, h) are its fragment of step u, with k in the accumulators' order, and
// the left operand is read from LDS in that order too (read_cols).
#ifndef DEEP8_AMD_ATTENTION_H
#define DEEP8_AMD_ATTENTION_H

#include <initializer_list>

#include "common.h"

namespace d8 {
namespace attention {

enum { MOST_DIM = 256 };
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Args {
    const void *q, *k, *v;
    void *o;
    float *lse;  // [heads][q_tokens], natural logarithm
    const void *dout;
    void *dq, *dk, *dv;
    long ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
    const int *q_starts, *k_starts;
    int sequences, q_tokens, k_tokens, heads, kv_heads, group, dim, causal;
    unsigned group_rcp;  // floor((2^32 - 1) / group)
    float scale;
    int vec;        // rows of every tensor can be moved in 16-byte pieces
    int tiles;      // row tiles (key blocks) of all sequences at most
    int units;      // pieces of work that the launch has room for, of each kv head
    int pieces;     // ... that the keys (dk and dv: the rows) are cut into, about; 0: not at all
    int split_kv;   // gradient: keys of a workgroup are 128 over this
    int overwrite;
    float *part;    // partial sums of the pieces; forward: partial outputs [units * kv_heads][rows][dim] and [..][rows][2] maximum and sum
    float *part_ml;
    int4 *joins;    // ... what the second launch joins, by piece: chunks, first query, row tile, rows of the sequence
    float *delta;   // gradient: rowsum(do o) [heads][q_tokens]
    float *norms;   // gradient, half: norms of the rows of do [heads][q_tokens] and of v [kv_heads][k_tokens], 0 for one that is not finite
    float *v_norms;
};

// One sequence as its tensors have it.
struct Span {
    int q0, nq, k0, nk;
};
// The lane's sequence of the 64 from `first` on, an empty one beyond the last; q_top, k_top: the largest starts before them, and then up to
// their end.  Starts count as the tensors' ends where they leave the tensors, and as an earlier start where they lie before it: sequences never
// overlap, so what is counted here in tiles, blocks and chunks stays within what launches and scratch were sized by from the numbers of tokens,
// whatever the starts are.  All lanes of a wave take part.
__device__ __forceinline__ Span spans_from(const Args &a, int first, int &q_top, int &k_top) {
    const int lane = threadIdx.x & 63, at = min(first + lane, a.sequences), next = min(first + lane + 1, a.sequences);
    int q0 = min(max(a.q_starts[at], 0), a.q_tokens), q1 = min(max(a.q_starts[next], 0), a.q_tokens);
    int k0 = min(max(a.k_starts[at], 0), a.k_tokens), k1 = min(max(a.k_starts[next], 0), a.k_tokens);
    if (__ballot(q0 < q_top || q1 < q0 || k0 < k_top || k1 < k0)) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int q = __shfl_up(q0, d), k = __shfl_up(k0, d);
            q0 = lane >= d ? max(q0, q) : q0, k0 = lane >= d ? max(k0, k) : k0;
        }
        q0 = max(q0, q_top), k0 = max(k0, k_top);
        q1 = max(q1, q0), k1 = max(k1, k0);
    }
    q_top = __builtin_amdgcn_readlane(q1, 63), k_top = __builtin_amdgcn_readlane(k1, 63);
    return Span{q0, q1 - q0, k0, k1 - k0};
}

// Row r's query, r < 2^31: r times the reciprocal over 2^32 is the quotient or one less.
__device__ __forceinline__ int query_of(const Args &a, int r) {
    const int t = (int)__umulhi((unsigned)r, a.group_rcp);
    return t + (r - t * a.group >= a.group ? 1 : 0);
}

// Which sequence holds item `id` of a list in which sequence s has count(span) items (none if it is empty): sets s, the item's number in it and the span; false
// beyond the list.  All lanes of a wave take part, 64 sequences at a time.
template <class Count>
__device__ __forceinline__ bool locate(const Args &a, int id, Span &span, int &s, int &item, Count &&count) {
    const int lane = threadIdx.x & 63;
    int before = 0, q_top = 0, k_top = 0;
    for (int first = 0; first < a.sequences; first += 64) {
        const Span own = spans_from(a, first, q_top, k_top);
        const int n = count(own);
        int upto = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int other = __shfl_up(upto, d);
            upto += lane >= d ? other : 0;
        }
        const unsigned long long past = __ballot(before + upto > id);
        if (past) {
            const int l = __ffsll((long long)past) - 1;
            s = first + l;
            item = id - before - (__shfl(upto, l) - __shfl(n, l));
            s = __builtin_amdgcn_readfirstlane(s);
            item = __builtin_amdgcn_readfirstlane(item);
            const int from = __builtin_amdgcn_readfirstlane(l);
            span.q0 = __builtin_amdgcn_readlane(own.q0, from), span.nq = __builtin_amdgcn_readlane(own.nq, from);
            span.k0 = __builtin_amdgcn_readlane(own.k0, from), span.nk = __builtin_amdgcn_readlane(own.nk, from);
            return true;
        }
        before += __shfl(upto, 63);
    }
    return false;
}

template <class T>
struct Type;

typedef __fp16 tr_f16x4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
#define ATTN_LDS(T, p) ((__attribute__((address_space(3))) T *)(__attribute__((address_space(3))) void *)(p))

template <>
struct Type<f16> {
    typedef f16x8 frag;
    static constexpr int V = 8;      // elements of 16 bytes
    static constexpr int STEP = 16;  // k of one fragment product
    static constexpr int REGS = 8;   // accumulator registers that make one fragment
    static __device__ __forceinline__ void mma(f32x16 &acc, const frag &a, const frag &b) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0);
    }
    static __device__ __forceinline__ frag pack(const f32x16 &s, int u) {
        frag r;
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = (f16)s[8 * u + e];
        return r;
    }
    // columns c0 .. c0 + 31 of a tile (row r at tile + r * pitch bytes) as left operand: lane (i, h) column c0 + i, rows r0 + 4 h + e and
    // r0 + 8 + 4 h + e: two transposing reads, in which 16 lanes together read 4 rows of 16 columns and each gets a column
    // (IN_ROW_ORDER: rows r0 + 8 h + e, the order of read_rows)
    template <bool IN_ROW_ORDER = false>
    static __device__ __forceinline__ frag read_cols(const char *tile, int pitch, int r0, int c0, int lane) {
        const int i = lane & 15, j = lane >> 4;
        const char *p = tile + (r0 + (IN_ROW_ORDER ? 8 : 4) * (j >> 1) + (i >> 2)) * pitch + (c0 + 16 * (j & 1) + 4 * (i & 3)) * 2;
        const tr_f16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16(ATTN_LDS(tr_f16x4, p));
        const tr_f16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4f16(ATTN_LDS(tr_f16x4, p + (IN_ROW_ORDER ? 4 : 8) * pitch));
        return __builtin_bit_cast(frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

template <>
struct Type<float> {
    typedef f32x4 frag;
    static constexpr int V = 4;
    static constexpr int STEP = 8;
    static constexpr int REGS = 4;
    static __device__ __forceinline__ void mma(f32x16 &acc, const frag &a, const frag &b) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], acc, 0, 0, 0);
    }
    static __device__ __forceinline__ frag pack(const f32x16 &s, int u) {
        frag r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = s[4 * u + e];
        return r;
    }
    // lane (i, h): column c0 + i of rows r0 + 4 h + e, which is the order of read_rows too
    template <bool IN_ROW_ORDER = false>
    static __device__ __forceinline__ frag read_cols(const char *tile, int pitch, int r0, int c0, int lane) {
        const char *p = tile + (r0 + 4 * (lane >> 5)) * pitch + (c0 + (lane & 31)) * 4;
        frag r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = *(const float *)(p + e * pitch);
        return r;
    }
};

// 16 bytes of a row from element d on, zero beyond `dim` and where the row is not there
template <class T>
__device__ __forceinline__ typename Type<T>::frag load_piece(const T *row, int d, int dim, bool there, int vec) {
    typename Type<T>::frag r;
#pragma unroll
    for (int e = 0; e < Type<T>::V; ++e) r[e] = (T)0.f;
    if (!there || d >= dim) return r;
    if (vec) return *(const typename Type<T>::frag *)(row + d);
#pragma unroll
    for (int e = 0; e < Type<T>::V; ++e)
        if (d + e < dim) r[e] = row[d + e];
    return r;
}

// the lane's fragment of row (lane & 31) of a tile, step u: the left operand whose k runs along the row (or the right operand whose
// columns are the tile's rows)
template <class T>
__device__ __forceinline__ typename Type<T>::frag read_rows(const char *tile, int pitch, int u, int lane) {
    return *(const typename Type<T>::frag *)(tile + (lane & 31) * pitch + u * 32 + (lane >> 5) * 16);
}

// ---- tiles that go from memory straight into LDS ----------------------------------------------------------------------
// A row takes PB bytes (a power of two) in LDS, its 16-byte piece c at position c ^ swizzle(row): the lanes of a load land 16 bytes
// apart, so rows cannot be padded, and the exclusive-or keeps what a read's lanes want in different banks, both along rows (one piece of
// sixteen rows, in whatever order the lanes are served) and along columns (four rows of four pieces each, or a row's neighbours).
template <int PB>
__device__ __forceinline__ int swizzle(int row) {
    // of the 256 bytes that the banks span, a row takes PB: the rows of a column read, four in a row, go to different quarters, sixteen rows to
    // different sixteenths
    constexpr int PER_SPAN = PB >= 256 ? 1 : 256 / PB;
    return (((row & 3) / PER_SPAN) << 2) | ((row >> 2) & 3);
}

template <class T, int DP>
constexpr int row_bytes() {  // the power of two that holds DP elements
    int b = 64;
    while (b < DP * (int)sizeof(T)) b *= 2;
    return b;
}

// read_rows and read_cols of such a tile, whose address is a multiple of PB; r0 a multiple of 16, c0 of 32
template <class T, int PB>
__device__ __forceinline__ typename Type<T>::frag rows_frag(const char *tile, int r0, int u, int lane) {
    const int row = r0 + (lane & 31);
    return *(const typename Type<T>::frag *)(tile + row * PB + (((2 * u + (lane >> 5)) ^ swizzle<PB>(row)) << 4));
}
template <class T, int PB>
__device__ __forceinline__ typename Type<T>::frag cols_frag(const char *tile, int r0, int c0, int lane) {
    typename Type<T>::frag r;
    if constexpr (sizeof(T) == 2) {
        const int i = lane & 15, j = lane >> 4, row = r0 + 4 * (j >> 1) + (i >> 2), at = c0 * 2 + 32 * (j & 1) + 8 * (i & 3);
        const char *p = tile + row * PB + ((((at >> 4) ^ swizzle<PB>(row)) << 4) | (at & 15));
        const char *q = tile + (row + 8) * PB + ((((at >> 4) ^ swizzle<PB>(row + 8)) << 4) | (at & 15));
        const tr_f16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16(ATTN_LDS(tr_f16x4, p));
        const tr_f16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4f16(ATTN_LDS(tr_f16x4, q));
        r = __builtin_bit_cast(typename Type<T>::frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
        const int at = (c0 + (lane & 31)) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = r0 + 4 * (lane >> 5) + e;
            r[e] = *(const float *)(tile + row * PB + ((((at >> 4) ^ swizzle<PB>(row)) << 4) | (at & 15)));
        }
    }
    return r;
}

typedef unsigned desc_t __attribute__((ext_vector_type(4)));

// s_waitcnt: at most n vector-memory instructions outstanding; all LDS reads have arrived
#define ATTN_VMCNT(n) __builtin_amdgcn_s_waitcnt(((n) & 15) | (((n) >> 4) << 14) | 0x0f70)
__device__ __forceinline__ void lds_reads_done() {
    __builtin_amdgcn_s_waitcnt(0xc07f);
    asm volatile("" ::: "memory");
}

// One 16-byte piece a lane from memory into LDS at `target` + 16 * lane.  asm, so that the compiler does not hold every later LDS read
// until it has landed; the kernels wait by count.  Beyond the descriptor's bytes zeros are written.  (s_nop 4: the
// hardware does not interlock scalars that a vector instruction has just written, nor m0.)
__device__ __forceinline__ void load_to_lds(const desc_t &desc, unsigned voffset, unsigned target) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(target), "v"(voffset), "s"(desc) : "memory");
}

// Rows of one tensor on their way into tiles: `first` is the first row's head, rows are `ld` elements apart.
template <class T, int PB>
struct TileLoader {
    unsigned voff;  // the lane's row and piece within 1 KB of LDS, as an offset from the tile's first row, before the swizzle
    unsigned row_stride;
    int lane_row, lane_pos, pieces;
    static constexpr int ROWS = PB >= 1024 ? 1 : 1024 / PB;  // rows of one load

    __device__ __forceinline__ void init(long ld, int dim, int lane) {
        static_assert(PB <= 1024, "a row is one load at most");
        lane_row = lane / (PB / 16), lane_pos = lane % (PB / 16);
        row_stride = (unsigned)(ld * sizeof(T));
        voff = lane_row * row_stride;
        pieces = dim / Type<T>::V;
    }
    // descriptor over the head's part of `rows` rows from `first` on
    static __device__ __forceinline__ desc_t desc(const T *first, int rows, long ld, int dim) {
        const unsigned long p = (unsigned long)first;
        const unsigned bytes = rows > 0 ? (unsigned)((rows - 1) * (unsigned)(ld * sizeof(T)) + dim * (int)sizeof(T)) : 0u;
        return desc_t{(unsigned)__builtin_amdgcn_readfirstlane((int)p), (unsigned)__builtin_amdgcn_readfirstlane((int)(p >> 32)) & 0xffffu,
                      (unsigned)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
    }
    // load t of a tile: rows t * ROWS .. of it, to LDS byte address `tile`
    __device__ __forceinline__ void load(const desc_t &d, int t, unsigned tile) const {
        const int piece = lane_pos ^ swizzle<PB>(t * ROWS + lane_row);
        const unsigned at = piece < pieces ? voff + t * ROWS * row_stride + piece * 16 : 0x80000000u;
        load_to_lds(d, at, __builtin_amdgcn_readfirstlane(tile + t * 1024));
    }
};

__device__ __forceinline__ unsigned lds_address(const void *p) { return (unsigned)(size_t)ATTN_LDS(const char, p); }

// ---- the running softmax of a lane's row ---------------------------------------------------------------------------------
// Scores times c (log2 e times the scale, positive) enter as powers of two relative to `base`, which follows their maximum only when that has
// grown by more than 8: sums and outputs are then up to 2^8 larger than they would be, which fp32 (and a half up to 256) does
// not notice, and most tiles need no pass over the accumulators.
struct Softmax {
    float base, sum;
    __device__ __forceinline__ void init() { base = -INFINITY, sum = 0.f; }
    // scores -> powers; returns what the accumulators have to be multiplied by, 1 for every lane if nothing changes
    template <int N>
    __device__ __forceinline__ bool step(f32x16 (&s)[N], float c, float &keep) {
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < N; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, s[b][e]);
        top = fmaxf(top, __shfl_xor(top, 32)) * c;
        const bool moved = __ballot(top > base + 8.f) != 0;
        keep = 1.f;
        if (moved) {
            const float next = fmaxf(base, top);
            keep = next == base ? 1.f : __builtin_amdgcn_exp2f(base - next);
            sum *= keep;
            base = next;
        }
        const float at = base == -INFINITY ? 0.f : base;
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < N; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[b][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][e], c, -at));
                part[e & 3] += s[b][e];
            }
        sum += (part[0] + part[1]) + (part[2] + part[3]);
        return moved;
    }
};

int check(const Args &a, int dtype, const char *name);
inline void set_group(Args &a) { a.group = a.heads / a.kv_heads, a.group_rcp = 0xffffffffu / (unsigned)a.group; }
bool in_pieces(int dtype, int dim, std::initializer_list<const void *> p, std::initializer_list<long> ld);
size_t grad_scratch_bytes(int dtype, int sequences, int q_tokens, int k_tokens, int heads, int kv_heads, int dim, bool causal);

template <int DP, class T>
constexpr int pitch_of() { return DP * (int)sizeof(T) + 16; }  // the 16 bytes keep a column's rows in different banks

}  // namespace attention
}  // namespace d8

#endif
