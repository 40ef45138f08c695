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
    float scale;
    int vec;        // rows of every tensor can be moved in 16-byte pieces
    int tiles;      // row tiles (key blocks) of all sequences at most
    int units;      // split forward: pieces of work that the launch has room for, of each kv head
    int pieces;     // ... that the keys are cut into, about
    int overwrite;
    float *part;    // split forward: partial outputs [units * kv_heads][rows][dim] and [..][rows][2] maximum and sum
    float *part_ml;
    float *delta;   // gradient: rowsum(do o) [heads][q_tokens]
    float *norms;   // gradient, half: largest squared norms of rows of do and of v, by workgroup of the first pass
};

// One sequence as its tensors have it.  Starts that run backwards or leave the tensors are cut to what is there.
struct Span {
    int q0, nq, k0, nk;
};
__device__ __forceinline__ Span span_of(const Args &a, int s) {
    Span r;
    r.q0 = min(max(a.q_starts[s], 0), a.q_tokens);
    r.nq = max(min(a.q_starts[s + 1], a.q_tokens) - r.q0, 0);
    r.k0 = min(max(a.k_starts[s], 0), a.k_tokens);
    r.nk = max(min(a.k_starts[s + 1], a.k_tokens) - r.k0, 0);
    return r;
}

// Which sequence holds item `id` of a list in which sequence s has count(span) items: sets s, the item's number in it and the span; false
// beyond the list.  All lanes of a wave take part, 64 sequences at a time.
template <class Count>
__device__ __forceinline__ bool locate(const Args &a, int id, Span &span, int &s, int &item, Count &&count) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int first = 0; first < a.sequences; first += 64) {
        int n = 0;
        if (first + lane < a.sequences) n = count(span_of(a, first + lane));
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
            span = span_of(a, s);
            return true;
        }
        before += __shfl(upto, 63);
    }
    return false;
}

// sum of count(span) over the sequences
template <class Count>
__device__ __forceinline__ long total_of(const Args &a, Count &&count) {
    const int lane = threadIdx.x & 63;
    long n = 0;
    for (int s = lane; s < a.sequences; s += 64) n += count(span_of(a, s));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d);
    return n;
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

int check(const Args &a, int dtype, const char *name);
bool in_pieces(int dtype, int dim, std::initializer_list<const void *> p, std::initializer_list<long> ld);
size_t grad_scratch_bytes(int q_tokens, int heads);

template <int DP, class T>
constexpr int pitch_of() { return DP * (int)sizeof(T) + 16; }  // the 16 bytes keep a column's rows in different banks

}  // namespace attention
}  // namespace d8

#endif
