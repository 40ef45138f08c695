// Tokens' keys and values written into a cache of 8-bit pages, and read back.
//
// A page and head have one scale, a power of two: the least of which 127 reach the largest element.  New tokens raise it if they have to, and
// then the codes that are there are rounded to the new scale, halves to the even one; a page's first token begins a new one.  Powers of two, though a
// scale of max / 127 would be finer by half a bit in the mean: growing tokenwise, a page meets about five new maxima, each of them one
// more rounding of all its codes at scales that go as they like, but one or two at powers of two; and a code is then the exact quotient's
// rounding, whatever the order of tokens in a call.
//
// One workgroup writes the tokens that a call brings to one page of one head: the elements are read twice (the largest, then the codes; the
// second time out of cache), values are transposed through LDS, and a page that holds tokens already is read and written whole.  Bound
// by memory where pages are filled (8192 tokens of 8 heads of 128 halves: 13 us written, 11.5 read back, 3.9 and 4.4 TB/s), by the chain of its loads
// (sequence, page, scale, codes) where they get a token each: 5 us.
#include <type_traits>

#include "cache.h"
#include "lanes.h"

namespace d8 {
namespace cache {

int check(const Pages &p, int dtype, const char *name) {
    if (dtype != D8_FLOAT16 && dtype != D8_FLOAT32) return fail(D8_ERR_DTYPE, "%s: type %d is not support", name, dtype);
    D8_REQUIRE(p.sequences >= 0 && p.tokens >= 0 && p.table_pages >= 0 && p.pages >= 0, "%s: %d sequences, %d tokens, %d of %d pages", name, p.sequences, p.tokens,
               p.table_pages, p.pages);
    D8_REQUIRE(p.kv_heads >= 1 && p.dim >= 1 && p.dim <= MOST_DIM, "%s: %d heads of %d elements (1 to %d)", name, p.kv_heads, p.dim, (int)MOST_DIM);
    D8_REQUIRE(p.table_pages < (1 << 24) && p.sequences < (1 << 24) && (long)p.tokens * p.kv_heads < (1L << 30), "%s: too many tokens, sequences or pages", name);
    if (!p.sequences || !p.tokens) return 0;
    D8_REQUIRE(p.starts && p.lengths && (p.table || !p.table_pages), "%s: null tensor", name);
    D8_REQUIRE(!p.pages || (p.k_codes && p.k_scales && p.v_codes && p.v_scales), "%s: null cache", name);
    D8_REQUIRE((((size_t)p.k_codes | (size_t)p.v_codes) & 15) == 0, "%s: codes must be 16-byte aligned", name);
    return 0;
}

namespace {

struct Args {
    Pages c;
    void *k, *v;
    long ldk, ldv;
};

__device__ __forceinline__ unsigned size_of(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// the least power of two of which 127 reach a value of this size (2^-100 at least); NaN for one that is not finite
__device__ __forceinline__ float scale_for(unsigned size) {
    if (size >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    // size = 1.f 2^e: 127 2^(e - 6) = 1.984375 2^e reaches it unless f is larger than that
    const int e = (int)(size >> 23) - 127 - 6 + ((size & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    return __uint_as_float((unsigned)(max(e, -100) + 127) << 23);
}

// four codes in a word at another scale
__device__ __forceinline__ int rescaled(int word, float by) {
    unsigned out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) out |= ((unsigned)(int)rintf((float)(signed char)(word >> (8 * i)) * by) & 255u) << (8 * i);
    return (int)out;
}

template <class T, int V>
struct Piece {
    typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));  // (rows may start anywhere)
};
template <class T>
struct Piece<T, 1> {
    typedef T type;
};
__device__ __forceinline__ unsigned code_of(float x, float back) { return (unsigned)(int)rintf(x * back) & 255u; }  // (exact but for the rounding)

enum { WORDS = 17 };  // words of LDS between two elements' 16 of tokens: four elements of one token in different banks

// Rows r .. r + rows - 1 of the call are places slot .. of `page`, which holds `slot` tokens already (or none that count).  V: elements of a piece of a
// row (in_pieces).  An item is a piece of four tokens, of keys and of values: a word of codes of each of its elements.
template <class T, int V>
__device__ __forceinline__ void append(const Args &a, int r, int rows, int slot, int page, int head, unsigned *sizes, unsigned *words) {
    const Pages &c = a.c;
    typedef typename Piece<T, V>::type piece;
    const int tid = threadIdx.x, pieces = c.dim / V, first = slot >> 2, items = (((slot + rows - 1) >> 2) - first + 1) * pieces;
    const T *k = (const T *)a.k + (long)r * a.ldk + (long)head * c.dim, *v = (const T *)a.v + (long)r * a.ldv + (long)head * c.dim;
    float *ks = c.k_scales + (long)page * c.kv_heads + head, *vs = c.v_scales + (long)page * c.kv_heads + head;
    piece kx[4], vx[4];
    auto load = [&](int i) {  // (rows that are not there: zeros)
        const int word = i / pieces, d = (i - word * pieces) * V, row = (first + word) * 4 - slot;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            kx[j] = vx[j] = piece{};
            if (row + j >= 0 && row + j < rows) kx[j] = *(const piece *)(k + (row + j) * a.ldk + d), vx[j] = *(const piece *)(v + (row + j) * a.ldv + d);
        }
    };
    auto at = [&](const piece &x, int e) {
        if constexpr (V == 1) return (float)x;
        else return (float)x[e];
    };
    // the largest of both; a thread's last item stays in its registers
    unsigned k_size = 0, v_size = 0;
    int held = -1;
    for (int i = tid; i < items; i += 256) {
        load(i);
        held = i;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) k_size = max(k_size, size_of(at(kx[j], e))), v_size = max(v_size, size_of(at(vx[j], e)));
    }
    if (tid == 0) sizes[8] = slot ? __float_as_uint(*ks) : 0u, sizes[9] = slot ? __float_as_uint(*vs) : 0u;
    const auto larger = [](unsigned x, unsigned y) { return max(x, y); };
    k_size = over_lanes<64>(k_size, larger), v_size = over_lanes<64>(v_size, larger);
    if ((tid & 63) == 0) sizes[tid >> 6] = k_size, sizes[4 + (tid >> 6)] = v_size;
    for (int i = tid; i < c.pitch * WORDS; i += 256) words[i] = 0;
    __syncthreads();
    const float k_old = __uint_as_float(sizes[8]), v_old = __uint_as_float(sizes[9]);
    k_size = max(max(sizes[0], sizes[1]), max(sizes[2], sizes[3])), v_size = max(max(sizes[4], sizes[5]), max(sizes[6], sizes[7]));
    const float k_need = scale_for(k_size), v_need = scale_for(v_size);
    // (a scale that is no number stays so until the page begins anew)
    const float k_scale = k_need != k_need || k_old != k_old ? __uint_as_float(0x7fc00000u) : fmaxf(k_need, k_old);
    const float v_scale = v_need != v_need || v_old != v_old ? __uint_as_float(0x7fc00000u) : fmaxf(v_need, v_old);
    if (tid == 0) *ks = k_scale, *vs = v_scale;
    const float k_back = k_scale == k_scale ? 1.f / k_scale : 0.f, v_back = v_scale == v_scale ? 1.f / v_scale : 0.f;
    const bool k_good = k_size < 0x7f800000u, v_good = v_size < 0x7f800000u;
    signed char *k_to = c.k_codes + c.tile(page, head), *v_to = c.v_codes + c.tile(page, head);
    for (int i = held; i >= 0; i -= 256) {
        if (i != held) load(i);
        const int word = i / pieces, d = (i - word * pieces) * V;
        unsigned w[V] = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int place = (first + word) * 4 + j;
            if (v_good)
#pragma unroll
                for (int e = 0; e < V; ++e) w[e] |= code_of(at(vx[j], e), v_back) << (8 * j);
            if (place < slot || place >= slot + rows) continue;
            signed char *to = k_to + place * c.pitch + d;
            if constexpr (V == 1) {
                *to = (signed char)(k_good ? code_of(at(kx[j], 0), k_back) : 0u);
            } else {
                unsigned q[V / 4];
#pragma unroll
                for (int e = 0; e < V; e += 4)
                    q[e / 4] = !k_good ? 0u : code_of(at(kx[j], e), k_back) | code_of(at(kx[j], e + 1), k_back) << 8 | code_of(at(kx[j], e + 2), k_back) << 16 | code_of(at(kx[j], e + 3), k_back) << 24;
                if constexpr (V == 8) *(uint2 *)to = make_uint2(q[0], q[1]);
                else *(unsigned *)to = q[0];
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) words[(d + e) * WORDS + first + word] = w[e];
    }
    // keys that were there
    const float k_by = k_old * k_back, v_by = v_old * v_back;
    if (slot && k_by != 1.f) {
        for (int i = tid; i < slot * c.pitch / 16; i += 256) {
            i32x4 w = *(const i32x4 *)(k_to + i * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = rescaled(w[e], k_scale == k_scale && k_old == k_old ? k_by : 0.f);
            *(i32x4 *)(k_to + i * 16) = w;
        }
    }
    __syncthreads();
    // values: 16 tokens of an element a thread; those before `slot` as they were, at the new scale
    for (int i = tid; i < c.pitch * 4; i += 256) {
        const int d = i >> 2, t = (i & 3) * 16;
        if (t + 16 <= slot && v_by == 1.f) continue;
        if (t >= slot + rows) continue;
        i32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (int)words[d * WORDS + t / 4 + e];
        if (t < slot) {
            const i32x4 old = *(const i32x4 *)(v_to + i * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int there = min(max(slot - t - 4 * e, 0), 4);
                const unsigned mask = there == 4 ? 0xffffffffu : (1u << (8 * there)) - 1;
                const unsigned o = v_by == 1.f ? (unsigned)old[e] : (unsigned)rescaled(old[e], v_scale == v_scale && v_old == v_old ? v_by : 0.f);
                w[e] = (int)((o & mask) | ((unsigned)w[e] & ~mask));
            }
        }
        *(i32x4 *)(v_to + i * 16) = w;
    }
}

// The workgroup's share of a call: rows row .. row + rows - 1 are places slot .. of `page` (-1: none) of one sequence, all that the call brings to it.
struct Share {
    int row, rows, slot, page;
};

// Share number `id` of the call, sequence by sequence and page by page; false beyond the last.  A start that lies before an earlier one counts
// as that one.  All lanes of a wave take part, 64 sequences at a time.
__device__ __forceinline__ bool share_of(const Pages &c, int id, Share &share) {
    const int lane = threadIdx.x & 63;
    int before = 0, top = 0;
    for (int from = 0; from < c.sequences; from += 64) {
        const int at = min(from + lane, c.sequences), next = min(from + lane + 1, c.sequences);
        int first = min(max(c.starts[at], 0), c.tokens), end = min(max(c.starts[next], 0), c.tokens);
        const long length = at < c.sequences ? max(c.lengths[at], 0) : 0;
        if (__ballot(first < top || end < first)) {
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int other = __shfl_up(first, d);
                first = lane >= d ? max(first, other) : first;
            }
            first = max(first, top), end = max(end, first);
        }
        top = __builtin_amdgcn_readlane(end, 63);
        const int n = end - first;
        const long place = length - n;  // of the first row; before 0 where the cache holds fewer tokens than the call brings
        const int pages = n ? (int)((place & (PAGE - 1)) + n + PAGE - 1) / PAGE : 0;
        const int upto = sum_upto_lane(pages);
        const unsigned long long past = __ballot(before + upto > id);
        if (past) {
            const int l = __builtin_amdgcn_readfirstlane(__ffsll((long long)past) - 1), s = from + l;
            const int number = id - before - __builtin_amdgcn_readlane(upto - pages, l), slot0 = __builtin_amdgcn_readlane((int)(place & (PAGE - 1)), l);
            const int page0 = __builtin_amdgcn_readlane((int)(place >> 6), l), rows = __builtin_amdgcn_readlane(n, l);
            const int skipped = number ? number * PAGE - slot0 : 0;
            share.row = __builtin_amdgcn_readlane(first, l) + skipped;
            share.slot = number ? 0 : slot0;
            share.rows = min(PAGE - share.slot, rows - skipped);
            share.page = c.page_of(s, page0 + number);
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

template <class T, int V>
__global__ __launch_bounds__(256) void cache_append_kernel(Args a) {
    __shared__ unsigned sizes[10];  // of four waves' keys and values, and the scales before
    __shared__ unsigned words[MOST_DIM * WORDS];
    Share s;
    if (share_of(a.c, blockIdx.x / a.c.kv_heads, s) && s.page >= 0) append<T, V>(a, s.row, s.rows, s.slot, s.page, blockIdx.x % a.c.kv_heads, sizes, words);
}

template <class T, int V>
__device__ __forceinline__ void store(T *p, const float (&x)[V]) {
    typename Piece<T, V>::type v;
    if constexpr (V == 1) {
        v = (T)x[0];
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (T)x[e];
    }
    *(typename Piece<T, V>::type *)p = v;
}

// Rows r .. of the call: the values of places slot .. of `page`, zeros if there is none.
template <class T, int V>
__device__ __forceinline__ void read(const Args &a, int r, int rows, int slot, int page, int head, unsigned *words) {
    const Pages &c = a.c;
    const int tid = threadIdx.x, pieces = c.dim / V;
    T *k = (T *)a.k + (long)r * a.ldk + (long)head * c.dim, *v = (T *)a.v + (long)r * a.ldv + (long)head * c.dim;
    const bool there = page >= 0;
    float ks = 0.f, vs = 0.f;
    const signed char *kc = nullptr;
    if (there) {
        ks = c.k_scales[(long)page * c.kv_heads + head], vs = c.v_scales[(long)page * c.kv_heads + head];
        kc = c.k_codes + c.tile(page, head);
        const signed char *vc = c.v_codes + c.tile(page, head);
        for (int i = tid; i < c.pitch * 4; i += 256) {
            const i32x4 w = *(const i32x4 *)(vc + i * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) words[(i >> 2) * WORDS + (i & 3) * 4 + e] = (unsigned)w[e];
        }
        __syncthreads();
    }
#pragma unroll 4
    for (int i = tid; i < rows * pieces; i += 256) {
        const int row = i / pieces, d = (i - row * pieces) * V, t = slot + row;
        float x[V] = {}, y[V] = {};
        if (there) {
            signed char code[V];
            const signed char *from = kc + t * c.pitch + d;
            if constexpr (V == 8) *(uint2 *)code = *(const uint2 *)from;
            else if constexpr (V == 4) *(unsigned *)code = *(const unsigned *)from;
            else code[0] = *from;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                x[e] = within<T>((float)code[e] * ks);
                y[e] = within<T>((float)(signed char)(words[(d + e) * WORDS + (t >> 2)] >> (8 * (t & 3))) * vs);
            }
        }
        store<T, V>(k + row * a.ldk + d, x), store<T, V>(v + row * a.ldv + d, y);
    }
}

template <class T, int V>
__global__ __launch_bounds__(256) void cache_read_kernel(Args a) {
    __shared__ unsigned words[MOST_DIM * WORDS];
    Share s;
    if (share_of(a.c, blockIdx.x / a.c.kv_heads, s)) read<T, V>(a, s.row, s.rows, s.slot, s.page, blockIdx.x % a.c.kv_heads, words);
}

// Workgroups of a call, for each head: n rows of a sequence reach (n + 62) / 64 + 1 pages at most, and each at least one.
long shares_of(const Pages &c) {
    const long some = c.sequences < c.tokens ? c.sequences : c.tokens, shares = (c.tokens + 62 * some) / 64 + some;
    return shares < c.tokens ? shares : c.tokens;
}

int check_rows(const Args &a, const char *name) {
    const long row = (long)a.c.kv_heads * a.c.dim;
    D8_REQUIRE(a.k && a.v, "%s: null tensor", name);
    D8_REQUIRE(a.ldk >= row && a.ldv >= row, "%s: rows of %ld elements do not fit their leading dimensions", name, row);
    D8_REQUIRE(shares_of(a.c) * a.c.kv_heads < (1L << 24), "%s: too many tokens and sequences for a launch", name);
    return 0;
}

// fn(V) for the largest pieces of 16 or 8 bytes that heads are made of, or single elements
template <class T, class F>
void in_pieces(int dim, F &&fn) {
    constexpr int V = 16 / (int)sizeof(T);
    if (dim % V == 0) return fn(std::integral_constant<int, V>());
    if constexpr (V == 8)
        if (dim % 4 == 0) return fn(std::integral_constant<int, 4>());
    fn(std::integral_constant<int, 1>());
}

template <class T>
void launch_append(const Args &a, dim3 grid, hipStream_t stream) {
    in_pieces<T>(a.c.dim, [&](auto v) { hipLaunchKernelGGL((cache_append_kernel<T, decltype(v)::value>), grid, dim3(256), 0, stream, a); });
}

template <class T>
void launch_read(const Args &a, dim3 grid, hipStream_t stream) {
    in_pieces<T>(a.c.dim, [&](auto v) { hipLaunchKernelGGL((cache_read_kernel<T, decltype(v)::value>), grid, dim3(256), 0, stream, a); });
}

}  // namespace
}  // namespace cache
}  // namespace d8

using namespace d8;

extern "C" int d8_cache_append(int dtype, const void *k, long ldk, const void *v, long ldv, signed char *k_codes, float *k_scales, signed char *v_codes,
                               float *v_scales, const int *starts, const int *lengths, const int *table, int sequences, int tokens, int table_pages, int pages,
                               int kv_heads, int dim, void *stream) {
    cache::Args a = {{k_codes, v_codes, k_scales, v_scales, starts, lengths, table, sequences, tokens, table_pages, pages, kv_heads, dim, (int)cache::pitch_of(dim)},
                     (void *)k, (void *)v, ldk, ldv};
    if (int rc = cache::check(a.c, dtype, "cache_append")) return rc;
    if (!sequences || !tokens) return 0;
    if (int rc = cache::check_rows(a, "cache_append")) return rc;
    if (!pages || !table_pages) return 0;
    const dim3 grid((unsigned)(cache::shares_of(a.c) * kv_heads));
    if (dtype == D8_FLOAT16) cache::launch_append<f16>(a, grid, as_stream(stream));
    else cache::launch_append<float>(a, grid, as_stream(stream));
    D8_LAUNCH_CHECK();
    return 0;
}

extern "C" int d8_cache_read(int dtype, void *k, long ldk, void *v, long ldv, const signed char *k_codes, const float *k_scales, const signed char *v_codes,
                             const float *v_scales, const int *starts, const int *lengths, const int *table, int sequences, int tokens, int table_pages, int pages,
                             int kv_heads, int dim, void *stream) {
    cache::Args a = {{(signed char *)k_codes, (signed char *)v_codes, (float *)k_scales, (float *)v_scales, starts, lengths, table, sequences, tokens, table_pages, pages,
                      kv_heads, dim, (int)cache::pitch_of(dim)},
                     k, v, ldk, ldv};
    if (int rc = cache::check(a.c, dtype, "cache_read")) return rc;
    if (!sequences || !tokens) return 0;
    if (int rc = cache::check_rows(a, "cache_read")) return rc;
    const dim3 grid((unsigned)(cache::shares_of(a.c) * kv_heads));
    if (dtype == D8_FLOAT16) cache::launch_read<f16>(a, grid, as_stream(stream));
    else cache::launch_read<float>(a, grid, as_stream(stream));
    D8_LAUNCH_CHECK();
    return 0;
}
