// Norm of each query and key head and its rotation by the position of its token, both tensors in one launch, and the way back.
//
//   r = 1 / sqrt(mean(x^2) + epsilon),  n = x r w,  (y_a, y_b) = (n_a c - n_b s, n_a s + n_b c) for the pairs (a, b) of the first
//   `rotary` elements, y = n for the others
//   back: g = the pairs of dy turned the other way,  dx = r (w g - x r mean(w g x r)),  dw = sum over tokens and heads of g x r
//
// Bound by memory: x is read and y written once (back: x and dy read, dx written).  A head is held by a group of 2^k lanes, each
// with two 16-byte pieces, chosen so that the two elements of a pair meet in one lane in either layout (half: piece p and the one
// rotary / 2 further on; neighbours: any two pieces), so that nothing but the two sums crosses lanes.  A group goes through several
// heads of one token and keeps the token's cosines and sines, which would otherwise be read from L2 once a head, as many bytes
// as the heads themselves.  Heads that cannot be moved in 16-byte pieces go through LDS, one wave each.
//
// Half, 8192 tokens of 32 + 8 heads of 128: 38 us, 172 MB at 4.5 TB/s (a large copy 5.1).  Back, single, 4099 tokens of 12 + 4 heads of 96: 17 us,
// 77 MB at 4.5 TB/s, and 4 for the weights' sums.  8 tokens: 4 us, a launch.
//
// All sums are fp32.  The sums behind dw go over workgroups through scratch and are added in a fixed order.
#include "common.h"

namespace d8 {
namespace {

enum { GENERAL_MOST_DIM = 2048 };  // elements of a head that the general kernel stages in LDS
enum { GRAD_GROUPS = 1024 };       // workgroups of a gradient call at most: rows of partial sums of dw

struct Side {  // queries or keys
    const void *x;
    const void *dy;
    void *out;  // y, or dx
    const void *weight;
    void *dweight;
    long ldx, lddy, ldout;
    int heads;
};

struct RotaryArgs {
    Side side[2];
    const int *positions;
    const float2 *table;
    float *partial;  // gradient: [workgroups][dim] sums behind dw
    float epsilon;
    int tokens, dim, norm, table_positions, rotary, interleaved;
    int chunk;             // heads that a group goes through
    int chunks[2];         // ... groups a token of each side
    int lanes;             // lanes a group
    int overwrite;
    int side_groups[2];    // gradient: workgroups of each side
};

template <class T>
struct Piece;
template <>
struct Piece<f16> {
    static constexpr int N = 8;
    typedef f16x8 vec;
};
template <>
struct Piece<float> {
    static constexpr int N = 4;
    typedef f32x4 vec;
};

template <class T>
__device__ __forceinline__ void load_piece(const T *p, float (&v)[Piece<T>::N]) {
    const typename Piece<T>::vec w = *(const typename Piece<T>::vec *)p;
#pragma unroll
    for (int e = 0; e < Piece<T>::N; ++e) v[e] = (float)w[e];
}
template <class T>
__device__ __forceinline__ void store_piece(T *p, const float (&v)[Piece<T>::N]) {
    typename Piece<T>::vec w;
#pragma unroll
    for (int e = 0; e < Piece<T>::N; ++e) w[e] = (T)v[e];
    *(typename Piece<T>::vec *)p = w;
}

// Where a lane's two pieces lie in a head (elements; -1: it has none) and whether they are turned.
struct LanePieces {
    int at[2];
    bool turned;
    int angle;  // first of its angles
    template <int V>
    __device__ __forceinline__ void init(const RotaryArgs &a, int l) {
        const int pairs = a.rotary / (2 * V), all = a.dim / V;
        turned = l < pairs;
        angle = l * V;  // V angles: of V pairs across two pieces, or of the neighbours in two pieces that follow each other
        if (turned) {
            at[0] = a.interleaved ? 2 * l * V : l * V;
            at[1] = a.interleaved ? at[0] + V : at[0] + a.rotary / 2;
        } else {
            const int p = 2 * pairs + 2 * (l - pairs);
            at[0] = p < all ? p * V : -1;
            at[1] = p + 1 < all ? (p + 1) * V : -1;
        }
    }
};

// turn the lane's pairs; back: the other way
template <int V>
__device__ __forceinline__ void turn(float (&a)[V], float (&b)[V], const float (&c)[V], const float (&s)[V], bool interleaved, bool back) {
    if (!interleaved) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float sn = back ? -s[e] : s[e], p = a[e], q = b[e];
            a[e] = p * c[e] - q * sn;
            b[e] = p * sn + q * c[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float &x = e < V / 2 ? a[2 * e % V] : b[2 * e % V];
            float &y = e < V / 2 ? a[2 * e % V + 1] : b[2 * e % V + 1];
            const float sn = back ? -s[e] : s[e], p = x, q = y;
            x = p * c[e] - q * sn;
            y = p * sn + q * c[e];
        }
    }
}

__device__ __forceinline__ int position_of(const RotaryArgs &a, int token) {
    const int p = a.positions ? a.positions[token] : token;
    return min(max(p, 0), a.table_positions - 1);
}

template <int V>
__device__ __forceinline__ void load_angles(const RotaryArgs &a, int token, const LanePieces &lp, float (&c)[V], float (&s)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) c[e] = 1.f, s[e] = 0.f;
    if (!lp.turned) return;
    const f32x4 *t = (const f32x4 *)(a.table + (long)position_of(a, token) * (a.rotary / 2) + lp.angle);
#pragma unroll
    for (int e = 0; e < V / 2; ++e) {
        const f32x4 w = t[e];
        c[2 * e] = w[0], s[2 * e] = w[1], c[2 * e + 1] = w[2], s[2 * e + 1] = w[3];
    }
}

__device__ __forceinline__ float group_sum(float v, int lanes) {
    for (int m = 1; m < lanes; m <<= 1) v += __shfl_xor(v, m);
    return v;
}

template <class T>
__device__ __forceinline__ void load_two(const T *x, const LanePieces &lp, float (&a)[Piece<T>::N], float (&b)[Piece<T>::N], float otherwise) {
#pragma unroll
    for (int e = 0; e < Piece<T>::N; ++e) a[e] = b[e] = otherwise;
    if (x && lp.at[0] >= 0) load_piece<T>(x + lp.at[0], a);
    if (x && lp.at[1] >= 0) load_piece<T>(x + lp.at[1], b);
}

template <class T>
__global__ __launch_bounds__(256) void head_norm_rotary_kernel(RotaryArgs a) {
    constexpr int V = Piece<T>::N;
    const int l = threadIdx.x & (a.lanes - 1);
    const long group = ((long)blockIdx.x * 256 + threadIdx.x) / a.lanes;
    const int per_token = a.chunks[0] + a.chunks[1];
    const long token = group / per_token;
    if (token >= a.tokens) return;  // (whole groups: the sums below stay inside one)
    int c = (int)(group - token * per_token);
    const int which = c >= a.chunks[0];
    c -= which ? a.chunks[0] : 0;
    const Side &S = a.side[which];
    LanePieces lp;
    lp.init<V>(a, l);
    float cs[V], sn[V], wa[V], wb[V];
    load_angles<V>(a, (int)token, lp, cs, sn);
    load_two<T>((const T *)S.weight, lp, wa, wb, 1.f);
    const int h0 = c * a.chunk, h1 = min(h0 + a.chunk, S.heads);
    const T *x = (const T *)S.x + token * S.ldx;
    T *y = (T *)S.out + token * S.ldout;
    for (int h = h0; h < h1; ++h) {
        float p[V], q[V];
        load_two<T>(x + (long)h * a.dim, lp, p, q, 0.f);
        if (a.norm) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) sum += p[e] * p[e] + q[e] * q[e];
            const float r = rsqrtf(group_sum(sum, a.lanes) / a.dim + a.epsilon);
#pragma unroll
            for (int e = 0; e < V; ++e) p[e] = p[e] * r * wa[e], q[e] = q[e] * r * wb[e];
        }
        if (lp.turned) turn<V>(p, q, cs, sn, a.interleaved, false);
        if (lp.at[0] >= 0) store_piece<T>(y + (long)h * a.dim + lp.at[0], p);
        if (lp.at[1] >= 0) store_piece<T>(y + (long)h * a.dim + lp.at[1], q);
    }
}

// Workgroups 0 .. side_groups[0] - 1 have the queries, the others the keys; each walks its share of (token, heads) and keeps its
// sums behind dw in registers.
template <class T>
__global__ __launch_bounds__(256) void head_norm_rotary_grad_kernel(RotaryArgs a) {
    constexpr int V = Piece<T>::N;
    __shared__ float sums[256 * 2 * V];
    const int l = threadIdx.x & (a.lanes - 1), groups = 256 / a.lanes;
    const int which = (int)blockIdx.x >= a.side_groups[0];
    const int block = blockIdx.x - (which ? a.side_groups[0] : 0);
    const Side &S = a.side[which];
    LanePieces lp;
    lp.init<V>(a, l);
    float wa[V], wb[V], da[V], db[V];
    load_two<T>((const T *)S.weight, lp, wa, wb, 1.f);
#pragma unroll
    for (int e = 0; e < V; ++e) da[e] = db[e] = 0.f;
    const long units = (long)a.tokens * a.chunks[which];
    for (long u = (long)block * groups + threadIdx.x / a.lanes; u < units; u += (long)a.side_groups[which] * groups) {
        const long token = u / a.chunks[which];
        const int h0 = (int)(u - token * a.chunks[which]) * a.chunk, h1 = min(h0 + a.chunk, S.heads);
        float cs[V], sn[V];
        load_angles<V>(a, (int)token, lp, cs, sn);
        const T *x = (const T *)S.x + token * S.ldx, *dy = (const T *)S.dy + token * S.lddy;
        T *dx = (T *)S.out + token * S.ldout;
        for (int h = h0; h < h1; ++h) {
            float p[V], q[V], ga[V], gb[V];
            load_two<T>(a.norm ? x + (long)h * a.dim : nullptr, lp, p, q, 0.f);
            load_two<T>(dy + (long)h * a.dim, lp, ga, gb, 0.f);
            if (lp.turned) turn<V>(ga, gb, cs, sn, a.interleaved, true);
            if (a.norm) {
                float sum = 0.f, dot = 0.f;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    sum += p[e] * p[e] + q[e] * q[e];
                    dot += wa[e] * ga[e] * p[e] + wb[e] * gb[e] * q[e];
                }
                const float r = rsqrtf(group_sum(sum, a.lanes) / a.dim + a.epsilon);
                const float m = group_sum(dot, a.lanes) * r / a.dim;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float ua = p[e] * r, ub = q[e] * r;
                    da[e] += ga[e] * ua, db[e] += gb[e] * ub;
                    ga[e] = r * (wa[e] * ga[e] - ua * m), gb[e] = r * (wb[e] * gb[e] - ub * m);
                }
            }
            T *to = dx + (long)h * a.dim;
            if (!(a.overwrite & 1)) {
                load_two<T>(to, lp, p, q, 0.f);
#pragma unroll
                for (int e = 0; e < V; ++e) ga[e] += p[e], gb[e] += q[e];
            }
            if (lp.at[0] >= 0) store_piece<T>(to + lp.at[0], ga);
            if (lp.at[1] >= 0) store_piece<T>(to + lp.at[1], gb);
        }
    }
    if (!S.dweight) return;  // uniform over the workgroup
#pragma unroll
    for (int e = 0; e < V; ++e) sums[(2 * e) * 256 + threadIdx.x] = da[e], sums[(2 * e + 1) * 256 + threadIdx.x] = db[e];
    __syncthreads();
    float *to = a.partial + (long)blockIdx.x * a.dim;
    if ((int)threadIdx.x < a.lanes) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (lp.at[k] < 0) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float s = 0.f;
                for (int g = 0; g < groups; ++g) s += sums[(2 * e + k) * 256 + g * a.lanes + l];
                to[lp.at[k] + e] = s;
            }
        }
    }
}

// One wave a head, through LDS: heads of any size, alignment and layout.
template <class T>
__global__ __launch_bounds__(64) void head_norm_rotary_general_kernel(RotaryArgs a) {
    __shared__ float head[GENERAL_MOST_DIM];
    const int lane = threadIdx.x, per_token = a.side[0].heads + a.side[1].heads;
    const long token = blockIdx.x / per_token;
    int h = (int)(blockIdx.x - token * per_token);
    const int which = h >= a.side[0].heads;
    h -= which ? a.side[0].heads : 0;
    const Side &S = a.side[which];
    const T *x = (const T *)S.x + token * S.ldx + (long)h * a.dim, *w = (const T *)S.weight;
    T *y = (T *)S.out + token * S.ldout + (long)h * a.dim;
    float sum = 0.f;
    for (int i = lane; i < a.dim; i += 64) {
        const float v = (float)x[i];
        head[i] = v, sum += v * v;
    }
    const float r = a.norm ? rsqrtf(group_sum(sum, 64) / a.dim + a.epsilon) : 1.f;
    __syncthreads();
    const int half = a.rotary / 2;
    const float2 *t = a.rotary ? a.table + (long)position_of(a, (int)token) * half : nullptr;
    for (int i = lane; i < a.dim; i += 64) {
        float v = head[i] * r * (w && a.norm ? (float)w[i] : 1.f);
        if (i < a.rotary) {
            const int pair = a.interleaved ? i / 2 : i % half;
            const bool second = a.interleaved ? i & 1 : i >= half;
            const int o = a.interleaved ? i ^ 1 : (second ? i - half : i + half);
            const float u = head[o] * r * (w && a.norm ? (float)w[o] : 1.f);
            const float2 cs = t[pair];
            v = second ? u * cs.y + v * cs.x : v * cs.x - u * cs.y;
        }
        y[i] = (T)v;
    }
}

template <class T>
__global__ __launch_bounds__(64) void head_norm_rotary_grad_general_kernel(RotaryArgs a) {
    __shared__ float head[GENERAL_MOST_DIM], grad[GENERAL_MOST_DIM], sums[GENERAL_MOST_DIM];
    const int lane = threadIdx.x;
    const int which = (int)blockIdx.x >= a.side_groups[0];
    const int block = blockIdx.x - (which ? a.side_groups[0] : 0);
    const Side &S = a.side[which];
    const T *w = a.norm ? (const T *)S.weight : nullptr;
    for (int i = lane; i < a.dim; i += 64) sums[i] = 0.f;
    const int half = a.rotary / 2;
    const long units = (long)a.tokens * S.heads;
    for (long u = block; u < units; u += a.side_groups[which]) {
        const long token = u / S.heads;
        const int h = (int)(u - token * S.heads);
        const T *x = (const T *)S.x + token * S.ldx + (long)h * a.dim, *dy = (const T *)S.dy + token * S.lddy + (long)h * a.dim;
        T *dx = (T *)S.out + token * S.ldout + (long)h * a.dim;
        for (int i = lane; i < a.dim; i += 64) grad[i] = (float)dy[i];
        __syncthreads();
        const float2 *t = a.rotary ? a.table + (long)position_of(a, (int)token) * half : nullptr;
        float sum = 0.f, dot = 0.f;
        for (int i = lane; i < a.dim; i += 64) {
            float g = grad[i];
            if (i < a.rotary) {
                const int pair = a.interleaved ? i / 2 : i % half;
                const bool second = a.interleaved ? i & 1 : i >= half;
                const float o = grad[a.interleaved ? i ^ 1 : (second ? i - half : i + half)];
                const float2 cs = t[pair];
                g = second ? g * cs.x - o * cs.y : g * cs.x + o * cs.y;
            }
            head[i] = g;
            const float v = a.norm ? (float)x[i] : 0.f;
            sum += v * v, dot += (w ? (float)w[i] : 1.f) * g * v;
        }
        __syncthreads();
        const float r = a.norm ? rsqrtf(group_sum(sum, 64) / a.dim + a.epsilon) : 1.f, m = group_sum(dot, 64) * r / a.dim;
        for (int i = lane; i < a.dim; i += 64) {
            const float g = head[i], v = a.norm ? (float)x[i] * r : 0.f;
            sums[i] += g * v;
            // (a head of one element: the two terms cancel but for epsilon, 1 - (x r)^2 = epsilon r^2)
            const float wg = (w ? (float)w[i] : 1.f) * g;
            const float d = !a.norm ? g : a.dim == 1 ? wg * r * r * r * a.epsilon : r * (wg - v * m);
            dx[i] = (T)((a.overwrite & 1) ? d : d + (float)dx[i]);
        }
        __syncthreads();
    }
    if (!S.dweight) return;
    for (int i = lane; i < a.dim; i += 64) a.partial[(long)blockIdx.x * a.dim + i] = sums[i];
}

// dw = (what it holds) + the sums of the side's workgroups, element by element: 64 threads an element, each its share of the
// workgroups in order, their sums joined in one order.
template <class T>
__global__ __launch_bounds__(256) void head_norm_weight_grad_kernel(RotaryArgs a) {
    __shared__ float part[4][4];
    const int which = blockIdx.y, col = threadIdx.x & 3, i = blockIdx.x * 4 + col, share = threadIdx.x >> 2;
    T *dw = (T *)a.side[which].dweight;
    if (!dw) return;
    const float *from = a.partial + (which ? (long)a.side_groups[0] * a.dim : 0);
    const int rows = a.side_groups[which];
    float s = 0.f;
    if (i < a.dim) {
        // (eight loads in flight: one after the other they cost 0.2 us each)
        for (int g = share; g < rows; g += 64 * 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = g + u * 64 < rows ? from[(long)(g + u * 64) * a.dim + i] : 0.f;
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
    }
#pragma unroll
    for (int m = 4; m < 64; m <<= 1) s += __shfl_xor(s, m);
    if ((threadIdx.x & 63) < 4) part[threadIdx.x >> 6][col] = s;
    __syncthreads();
    if (threadIdx.x < 4 && i < a.dim) {
        s = (part[0][col] + part[1][col]) + (part[2][col] + part[3][col]);
        dw[i] = (T)((a.overwrite & 2) ? s : s + (float)dw[i]);
    }
}

bool in_pieces(const RotaryArgs &a, int dtype, bool grad) {
    const int v = 16 / (int)dtype_bytes(dtype);
    if (a.dim % v || a.rotary % (2 * v)) return false;
    size_t any = (size_t)a.table;
    for (const Side &s : a.side) {
        if (!s.heads) continue;
        any |= (size_t)s.x | (size_t)s.out | (size_t)s.weight | (size_t)s.dy;
        if (s.ldx % v || s.ldout % v || (grad && s.lddy % v)) return false;
    }
    if (any & 15) return false;
    return a.rotary / (2 * v) + (a.dim / v - a.rotary / v + 1) / 2 <= 64;
}

void set_lanes(RotaryArgs &a, int dtype) {
    const int v = 16 / (int)dtype_bytes(dtype);
    const int need = a.rotary / (2 * v) + (a.dim / v - a.rotary / v + 1) / 2;
    for (a.lanes = 1; a.lanes < need;) a.lanes *= 2;
}

// How many heads of a token a group goes through: one while that leaves compute units idle, else up to eight.
void set_chunks(RotaryArgs &a) {
    const long rows = (long)a.tokens * (a.side[0].heads + a.side[1].heads), at_once = 256 / a.lanes * 8L * cu_count();
    a.chunk = (int)(rows / at_once);
    a.chunk = a.chunk < 1 ? 1 : a.chunk > 8 ? 8 : a.chunk;
    for (int i = 0; i < 2; ++i) a.chunks[i] = ceil_div(a.side[i].heads, a.chunk);
}

int check(const RotaryArgs &a, int dtype, bool grad) {
    if (dtype != D8_FLOAT16 && dtype != D8_FLOAT32) return fail(D8_ERR_DTYPE, "head_norm_rotary: type %d is not support", dtype);
    D8_REQUIRE(a.tokens >= 0 && a.dim >= 1, "head_norm_rotary: %d tokens of heads of %d", a.tokens, a.dim);
    D8_REQUIRE(a.dim <= GENERAL_MOST_DIM, "head_norm_rotary: a head has at most %d elements, not %d", (int)GENERAL_MOST_DIM, a.dim);
    D8_REQUIRE(a.rotary >= 0 && a.rotary <= a.dim && a.rotary % 2 == 0, "head_norm_rotary: %d of the %d elements of a head cannot be turned in pairs", a.rotary, a.dim);
    D8_REQUIRE(a.rotary == 0 || (a.table && a.table_positions >= 1), "head_norm_rotary: rotation needs a table of angles");
    D8_REQUIRE(((size_t)a.table & 7) == 0, "head_norm_rotary: the table of angles must be 8-byte aligned");
    for (const Side &s : a.side) {
        D8_REQUIRE(s.heads >= 0, "head_norm_rotary: %d heads", s.heads);
        if (!s.heads || !a.tokens) continue;
        D8_REQUIRE(s.out && (grad ? s.dy && (s.x || !a.norm) : s.x != nullptr), "head_norm_rotary: null tensor");
        const long row = (long)s.heads * a.dim;
        D8_REQUIRE(((grad && !a.norm) || s.ldx >= row) && s.ldout >= row && (!grad || s.lddy >= row), "head_norm_rotary: rows of %ld elements do not fit their leading dimension", row);
        D8_REQUIRE(a.norm || (!s.weight && !s.dweight), "head_norm_rotary: a weight without a norm");
    }
    D8_REQUIRE((long)a.tokens * (a.side[0].heads + (long)a.side[1].heads) < (1L << 31), "head_norm_rotary: too many heads");
    return 0;
}

// workgroups of the gradient kernels, by side
void grad_groups(RotaryArgs &a, long per_group) {
    long want[2], most = GRAD_GROUPS;
    for (int i = 0; i < 2; ++i) want[i] = a.tokens ? ((long)a.tokens * a.chunks[i] + per_group - 1) / per_group : 0;
    const long all = want[0] + want[1];
    for (int i = 0; i < 2; ++i) {
        a.side_groups[i] = (int)(all <= most ? want[i] : want[i] * most / all);
        if (want[i] && !a.side_groups[i]) a.side_groups[i] = 1;
    }
}

}  // namespace
}  // namespace d8

using namespace d8;

extern "C" int d8_head_norm_rotary(int dtype, const void *q, long ldq, int q_heads, const void *q_weight, void *q_out, long ldq_out,
                                   const void *k, long ldk, int k_heads, const void *k_weight, void *k_out, long ldk_out,
                                   int tokens, int dim, int norm, float epsilon, const int *positions, const float *table,
                                   int table_positions, int rotary, int interleaved, void *stream) {
    RotaryArgs a;
    memset(&a, 0, sizeof(a));
    a.side[0].x = q, a.side[0].ldx = ldq, a.side[0].heads = q_heads, a.side[0].weight = q_weight, a.side[0].out = q_out, a.side[0].ldout = ldq_out;
    a.side[1].x = k, a.side[1].ldx = ldk, a.side[1].heads = k_heads, a.side[1].weight = k_weight, a.side[1].out = k_out, a.side[1].ldout = ldk_out;
    a.tokens = tokens, a.dim = dim, a.norm = norm != 0, a.epsilon = epsilon, a.positions = positions, a.table = (const float2 *)table;
    a.table_positions = table_positions, a.rotary = rotary, a.interleaved = interleaved != 0;
    if (int rc = check(a, dtype, false)) return rc;
    const long rows = (long)tokens * (q_heads + k_heads);
    if (!rows) return 0;
    if (in_pieces(a, dtype, false)) {
        set_lanes(a, dtype);
        set_chunks(a);
        const long threads = (long)tokens * (a.chunks[0] + a.chunks[1]) * a.lanes;
        const dim3 grid(ceil_div(threads, 256));
        if (dtype == D8_FLOAT16) hipLaunchKernelGGL(head_norm_rotary_kernel<f16>, grid, dim3(256), 0, as_stream(stream), a);
        else hipLaunchKernelGGL(head_norm_rotary_kernel<float>, grid, dim3(256), 0, as_stream(stream), a);
    } else {
        if (dtype == D8_FLOAT16) hipLaunchKernelGGL(head_norm_rotary_general_kernel<f16>, dim3(rows), dim3(64), 0, as_stream(stream), a);
        else hipLaunchKernelGGL(head_norm_rotary_general_kernel<float>, dim3(rows), dim3(64), 0, as_stream(stream), a);
    }
    D8_LAUNCH_CHECK();
    return 0;
}

extern "C" size_t d8_head_norm_rotary_grad_scratch_bytes(int dtype, int tokens, int q_heads, int k_heads, int dim) {
    if ((dtype != D8_FLOAT16 && dtype != D8_FLOAT32) || tokens < 0 || q_heads < 0 || k_heads < 0 || dim < 1 || dim > GENERAL_MOST_DIM) return 0;
    return sizeof(float) * (GRAD_GROUPS + 2) * (size_t)dim;
}

extern "C" int d8_head_norm_rotary_grad(int dtype, const void *q, long ldq, int q_heads, const void *q_weight, const void *dq_out, long lddq_out,
                                        void *dq, long lddq, void *dq_weight, const void *k, long ldk, int k_heads, const void *k_weight,
                                        const void *dk_out, long lddk_out, void *dk, long lddk, void *dk_weight, int tokens, int dim, int norm,
                                        float epsilon, const int *positions, const float *table, int table_positions, int rotary,
                                        int interleaved, int overwrite, void *scratch, size_t scratch_bytes, void *stream) {
    RotaryArgs a;
    memset(&a, 0, sizeof(a));
    Side &s0 = a.side[0], &s1 = a.side[1];
    s0.x = q, s0.ldx = ldq, s0.heads = q_heads, s0.weight = q_weight, s0.dy = dq_out, s0.lddy = lddq_out, s0.out = dq, s0.ldout = lddq, s0.dweight = dq_weight;
    s1.x = k, s1.ldx = ldk, s1.heads = k_heads, s1.weight = k_weight, s1.dy = dk_out, s1.lddy = lddk_out, s1.out = dk, s1.ldout = lddk, s1.dweight = dk_weight;
    a.tokens = tokens, a.dim = dim, a.norm = norm != 0, a.epsilon = epsilon, a.positions = positions, a.table = (const float2 *)table;
    a.table_positions = table_positions, a.rotary = rotary, a.interleaved = interleaved != 0, a.overwrite = overwrite;
    if (int rc = check(a, dtype, true)) return rc;
    const bool sums = dq_weight || dk_weight;
    const size_t need = d8_head_norm_rotary_grad_scratch_bytes(dtype, tokens, q_heads, k_heads, dim);
    D8_REQUIRE(!sums || (scratch && scratch_bytes >= need && ((size_t)scratch & 3) == 0), "head_norm_rotary_grad: scratch of %zu bytes, %zu needed", scratch_bytes, need);
    a.partial = (float *)scratch;
    const bool pieces = in_pieces(a, dtype, true);
    if (pieces) {
        set_lanes(a, dtype);
        set_chunks(a);
        grad_groups(a, 256 / a.lanes);
    } else {
        a.chunk = 1, a.chunks[0] = q_heads, a.chunks[1] = k_heads;
        grad_groups(a, 1);
    }
    const int groups = a.side_groups[0] + a.side_groups[1];
    if (groups) {
        if (pieces && dtype == D8_FLOAT16) hipLaunchKernelGGL(head_norm_rotary_grad_kernel<f16>, dim3(groups), dim3(256), 0, as_stream(stream), a);
        else if (pieces) hipLaunchKernelGGL(head_norm_rotary_grad_kernel<float>, dim3(groups), dim3(256), 0, as_stream(stream), a);
        else if (dtype == D8_FLOAT16) hipLaunchKernelGGL(head_norm_rotary_grad_general_kernel<f16>, dim3(groups), dim3(64), 0, as_stream(stream), a);
        else hipLaunchKernelGGL(head_norm_rotary_grad_general_kernel<float>, dim3(groups), dim3(64), 0, as_stream(stream), a);
        D8_LAUNCH_CHECK();
    }
    if (sums) {  // (with no token at all the sums are zero)
        const dim3 grid(ceil_div(dim, 4), 2);
        if (dtype == D8_FLOAT16) hipLaunchKernelGGL(head_norm_weight_grad_kernel<f16>, grid, dim3(256), 0, as_stream(stream), a);
        else hipLaunchKernelGGL(head_norm_weight_grad_kernel<float>, grid, dim3(256), 0, as_stream(stream), a);
        D8_LAUNCH_CHECK();
    }
    return 0;
}

namespace d8 {
namespace {

// table[p][i] = (cos, sin)(p f_i), f_i = base^(-2 i / rotary), slowed down for long contexts (see the header).  In fp64: at
// position 10^5 an fp32 angle is off by up to 4e-3.
__global__ __launch_bounds__(256) void rotary_table_kernel(float2 *table, int positions, int half, double base, double factor, double keep_below,
                                                           double slow_above) {
    const long n = (long)positions * half;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
        const long p = i / half;
        const int pair = (int)(i - p * half);
        double f = pow(base, -(double)pair / half);
        if (factor != 1.0) {
            const double wave = 6.283185307179586 / f;
            double keep = 0.0;  // share of the frequency that stays as it is
            if (slow_above > 0.0) keep = wave <= keep_below ? 1.0 : wave >= slow_above ? 0.0 : (slow_above / wave - 1.0) / (slow_above / keep_below - 1.0);
            f *= keep + (1.0 - keep) / factor;
        }
        double s, c;
        sincos((double)p * f, &s, &c);
        table[i] = make_float2((float)c, (float)s);
    }
}

}  // namespace
}  // namespace d8

extern "C" int d8_rotary_table(float *table, int positions, int rotary, double base, double factor, double keep_below, double slow_above, void *stream) {
    D8_REQUIRE(table && ((size_t)table & 7) == 0, "rotary_table: the table must be 8-byte aligned memory");
    D8_REQUIRE(positions >= 1 && rotary >= 2 && rotary % 2 == 0, "rotary_table: %d positions, %d elements turned", positions, rotary);
    D8_REQUIRE(base > 0.0 && factor > 0.0, "rotary_table: base %g, factor %g", base, factor);
    D8_REQUIRE(slow_above == 0.0 || (keep_below > 0.0 && slow_above > keep_below), "rotary_table: wave lengths %g and %g", keep_below, slow_above);
    const long n = (long)positions * (rotary / 2);
    const long groups = (n + 255) / 256;
    hipLaunchKernelGGL(rotary_table_kernel, dim3(groups < 4096 ? groups : 4096), dim3(256), 0, as_stream(stream), (float2 *)table, positions, rotary / 2, base,
                       factor, keep_below, slow_above);
    D8_LAUNCH_CHECK();
    return 0;
}
