/*
 * dev_train.hip - the operators of a training step beside the combine
 * (ucg_builtin_dev.h): the sum of several operands with dropout in its
 * epilogue, a router's balance loss and the clipped policy loss, each with its
 * gradient. All of them stream their operands from HBM once; sums are held in
 * fp32 over a few rows and joined in fp64 in an order that depends on the
 * sizes alone, so a call gives the same bits every time (no float atomics).
 */
#include <hip/hip_runtime.h>

#include <math.h>

#include "ucg_builtin_dev.h"
#include "dev_internal.h"
#include "dev_kernels.h"

namespace {

using ucgdev::kMaxMulti;
using ucgdev::rd_tree;
using ucgdev::SrcList;

typedef __bf16 bf16;
typedef _Float16 f16;

constexpr int kThreads = 256;         /* 4 waves */

/* ---- loads and stores of V neighbouring elements -------------------------- */
/* A vector only has to be element-aligned: gfx950 takes global accesses at any
 * address, so an odd row length costs split lines and no other kernel. */
template <typename T, int V>
struct Vec {
    static_assert(sizeof(T) * V % 4 == 0, "whole words");
    typedef unsigned type __attribute__((ext_vector_type(sizeof(T) * V / 4),
                                         aligned(sizeof(T)), __may_alias__));
};

template <typename T, int V>
__device__ __forceinline__ void load_raw(const T *p, T (&o)[V])
{
    typedef typename Vec<T, V>::type W;
    const W w = __builtin_nontemporal_load(reinterpret_cast<const W*>(p));
    __builtin_memcpy(o, &w, sizeof(o));
}

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T *p, float (&o)[V])
{
    T t[V];
    load_raw<T, V>(p, t);
#pragma unroll
    for (int k = 0; k < V; k++) {
        o[k] = (float)t[k];
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T *p, const float (&x)[V])
{
    typedef typename Vec<T, V>::type W;
    T t[V];
#pragma unroll
    for (int k = 0; k < V; k++) {
        t[k] = (T)x[k];               /* round to nearest even, once */
    }
    W w;
    __builtin_memcpy(&w, t, sizeof(w));
    __builtin_nontemporal_store(w, reinterpret_cast<W*>(p));
}

/* elements [c, c + V) of a row of n, `fill` past its end */
template <typename T, int V>
__device__ __forceinline__ void load_row(const T *row, size_t c, size_t n, float fill,
                                         float (&o)[V])
{
    if (c + V <= n) {
        load_vec<T, V>(row + c, o);
    } else {
#pragma unroll
        for (int k = 0; k < V; k++) {
            o[k] = c + k < n ? (float)row[c + k] : fill;
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_row(T *row, size_t c, size_t n, const float (&x)[V])
{
    if (c + V <= n) {
        store_vec<T, V>(row + c, x);
    } else {
#pragma unroll
        for (int k = 0; k < V; k++) {
            if (c + k < n) {
                row[c + k] = (T)x[k];
            }
        }
    }
}

/* ---- wavefront sums over G neighbouring lanes, the result in each ---------- */
template <typename X, typename F>
__device__ __forceinline__ X lanes_all(X x, unsigned lo, unsigned hi, F f)
{
    for (unsigned o = lo; o < hi; o <<= 1) {
        x = f(x, __shfl_xor(x, o, 64));
    }
    return x;
}

template <int CTRL>
__device__ __forceinline__ float dpp(float x)
{
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, true));
}

/* The same for a float over G lanes known at compile time, without LDS: after
 * the quads agree, a mirrored half row holds another quad's value, and so on. */
template <int G, typename F>
__device__ __forceinline__ float group_all(float x, F f)
{
    if constexpr (G >= 2) {
        x = f(x, dpp<0xB1>(x));       /* quad_perm 1,0,3,2 */
    }
    if constexpr (G >= 4) {
        x = f(x, dpp<0x4E>(x));       /* quad_perm 2,3,0,1 */
    }
    if constexpr (G >= 8) {
        x = f(x, dpp<0x141>(x));      /* row_half_mirror */
    }
    if constexpr (G >= 16) {
        x = f(x, dpp<0x140>(x));      /* row_mirror */
    }
    if constexpr (G >= 32) {
        x = f(x, __shfl_xor(x, 16, 64));
    }
    if constexpr (G >= 64) {
        x = f(x, __shfl_xor(x, 32, 64));
    }
    return x;
}

struct Add {
    template <typename X>
    __device__ __forceinline__ X operator()(X a, X b) const { return a + b; }
};
struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

/* sum over the block's 256 threads in thread order of halves; every thread
 * calls it, thread 0 has the result */
template <typename X>
__device__ __forceinline__ X block_sum(X x, X *lds)
{
    x = lanes_all(x, 1, 64, Add());
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        lds[threadIdx.x >> 6] = x;
    }
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

/* True in every thread of the last block to arrive, with the other blocks'
 * writes visible. *done is 0 before the launch (the kernel before it on the
 * stream writes that), so nothing has to be cleared between calls. */
__device__ __forceinline__ bool last_block(unsigned *done, unsigned *lds)
{
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        *lds = __hip_atomic_fetch_add(done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    const bool last = *lds == gridDim.x - 1;
    if (last) {
        __threadfence();
    }
    return last;
}

/* ======================================================================== */
/* dropout                                                                  */
/* ======================================================================== */
struct Rng {
    uint64_t        seed, tag, offset;
    const uint64_t *dev;
    uint32_t        threshold;   /* 0 .. 65536 */
    float           scale;
};

/* Philox-4x32-10 for counter (group, tag): eight 16-bit numbers. One round is
 * two 32 x 32 -> 64 bit products and two three-way xors; ten rounds for eight
 * elements keep it below the time the elements' own bytes take (a 32-bit
 * number for each element would double it). */
__device__ __forceinline__ void philox(uint64_t group, uint64_t tag, uint64_t seed,
                                       uint32_t (&w)[4])
{
    uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32);
    uint32_t c2 = (uint32_t)tag, c3 = (uint32_t)(tag >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    w[0] = c0;
    w[1] = c1;
    w[2] = c2;
    w[3] = c3;
}

__device__ __forceinline__ void rng_state(const Rng &r, uint64_t &seed, uint64_t &tag)
{
    seed = r.seed;
    tag  = r.tag;
    if (r.dev != nullptr) {
        seed = r.dev[0];
        tag  = r.dev[1];
    }
}

/* the 16-bit numbers of elements [at, at + V) of the tensor, two to a word.
 * ALIGNED: at is a multiple of V, so they lie in one group of eight. */
template <int V, bool ALIGNED>
__device__ __forceinline__ void draw(uint64_t at, uint64_t tag, uint64_t seed,
                                     uint32_t (&o)[V / 2])
{
    uint32_t w[4];
    philox(at >> 3, tag, seed, w);
    const unsigned sub = (unsigned)at & 7;
    if constexpr (ALIGNED && V == 8) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            o[k] = w[k];
        }
    } else if constexpr (ALIGNED) {
        static_assert(V == 4, "a vector is a group or half of one");
        o[0] = sub ? w[2] : w[0];
        o[1] = sub ? w[3] : w[1];
    } else {
        uint32_t x[9] = {w[0], w[1], w[2], w[3], 0, 0, 0, 0, 0};
        if (sub + V > 8) {
            philox((at >> 3) + 1, tag, seed, w);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                x[4 + k] = w[k];
            }
        }
        /* shift the eight words right by sub halves */
#pragma unroll
        for (int k = 0; k < 6; k++) {
            x[k] = sub & 4 ? x[k + 2] : x[k];
        }
#pragma unroll
        for (int k = 0; k < 6; k++) {
            x[k] = sub & 2 ? x[k + 1] : x[k];
        }
#pragma unroll
        for (int k = 0; k < V / 2; k++) {
            o[k] = sub & 1 ? (x[k] >> 16) | (x[k + 1] << 16) : x[k];
        }
    }
}

template <int V>
__device__ __forceinline__ bool kept(const uint32_t (&u)[V / 2], int k, uint32_t threshold)
{
    return ((u[k >> 1] >> (16 * (k & 1))) & 0xffffu) >= threshold;
}

/* N > 0: that many sources, in registers at once; 0: any number, one by one */
template <typename T, int N, typename L>
__device__ __forceinline__ float sum_sources(const SrcList &srcs, unsigned nsrc, L at)
{
    if constexpr (N == 0) {
        float s = at(static_cast<const T*>(srcs.p[0]));
        for (unsigned m = 1; m < nsrc; m++) {
            s = at(static_cast<const T*>(srcs.p[m])) + s;
        }
        return s;
    } else {
        float v[N];
#pragma unroll
        for (int m = 0; m < N; m++) {
            v[m] = at(static_cast<const T*>(srcs.p[m]));
        }
        if constexpr ((N & (N - 1)) == 0) {
            return rd_tree<N>(v, Add());
        } else {
            float s = v[0];
#pragma unroll
            for (int m = 1; m < N; m++) {
                s = v[m] + s;
            }
            return s;
        }
    }
}

/*
 * One lane does the V elements whose place in the whole tensor starts at a
 * multiple of V, so that one Philox group serves them; the first and the last
 * lane of a call may have fewer and go element by element. `inv` is
 * 2^64 / cols rounded up (unused for one column): the quotient by cols is its
 * high product, or one less (the rounding adds i * e / 2^64 < 1 with e <= 1).
 */
template <typename T, typename R, int V, int N>
__global__ void __launch_bounds__(kThreads)
k_sum_dropout(R *dst, SrcList srcs, unsigned nsrc, const T *bias, const R *residual,
              uint64_t n, uint64_t first, uint64_t cols, uint64_t inv, Rng rng)
{
    const unsigned phase = (unsigned)(rng.offset % V);
    const uint64_t g     = first + (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t  i     = (int64_t)(g * V) - phase;
    if (i >= (int64_t)n) {
        return;
    }
    uint64_t seed, tag;
    rng_state(rng, seed, tag);
    uint32_t u[V / 2] = {};
    const uint64_t at = rng.offset - phase + g * V;
    uint64_t col = 0;
    if (bias != nullptr) {
        const uint64_t j = i > 0 ? (uint64_t)i : 0;
        const uint64_t q = __umul64hi(j, inv);
        col = j - q * cols;
        col = cols == 1 ? 0 : (int64_t)col < 0 ? col + cols : col;
    }
    if (i >= 0 && i + V <= (int64_t)n) {
        float s[V];
        if constexpr (N == 0) {
            load_vec<T, V>(static_cast<const T*>(srcs.p[0]) + i, s);
#pragma unroll 4
            for (unsigned m = 1; m < nsrc; m++) {
                float x[V];
                load_vec<T, V>(static_cast<const T*>(srcs.p[m]) + i, x);
#pragma unroll
                for (int k = 0; k < V; k++) {
                    s[k] = x[k] + s[k];
                }
            }
        } else {
            float x[N][V];
#pragma unroll
            for (int m = 0; m < N; m++) {
                load_vec<T, V>(static_cast<const T*>(srcs.p[m]) + i, x[m]);
            }
#pragma unroll
            for (int k = 0; k < V; k++) {
                float v[N];
#pragma unroll
                for (int m = 0; m < N; m++) {
                    v[m] = x[m][k];
                }
                if constexpr ((N & (N - 1)) == 0) {
                    s[k] = rd_tree<N>(v, Add());
                } else {
                    s[k] = v[0];
#pragma unroll
                    for (int m = 1; m < N; m++) {
                        s[k] = v[m] + s[k];
                    }
                }
            }
        }
        float r[V] = {};
        if (residual != nullptr) {
            load_vec<R, V>(residual + i, r);
        }
        if (bias != nullptr) {
            float b[V];
            if (col + V <= cols) {
                T t[V];
                __builtin_memcpy(t, bias + col, sizeof(t));   /* temporal: read by every row */
#pragma unroll
                for (int k = 0; k < V; k++) {
                    b[k] = (float)t[k];
                }
            } else {
                uint64_t c = col;
#pragma unroll
                for (int k = 0; k < V; k++) {
                    b[k] = (float)bias[c];
                    c = c + 1 == cols ? 0 : c + 1;
                }
            }
#pragma unroll
            for (int k = 0; k < V; k++) {
                s[k] += b[k];
            }
        }
        if (rng.threshold != 0) {
            draw<V, true>(at, tag, seed, u);
        }
#pragma unroll
        for (int k = 0; k < V; k++) {
            const float d = kept<V>(u, k, rng.threshold) ? s[k] * rng.scale : 0.f;
            s[k] = residual != nullptr ? d + r[k] : d;
        }
        store_vec<R, V>(dst + i, s);
        return;
    }
    if (rng.threshold != 0) {
        draw<V, true>(at, tag, seed, u);
    }
    for (int k = 0; k < V; k++) {
        const int64_t j = i + k;
        if (j < 0 || j >= (int64_t)n) {
            continue;
        }
        float s = sum_sources<T, N>(srcs, nsrc, [&](const T *p) { return (float)p[j]; });
        if (bias != nullptr) {
            s += (float)bias[col];
            col = col + 1 == cols ? 0 : col + 1;
        }
        const float d = kept<V>(u, k, rng.threshold) ? s * rng.scale : 0.f;
        dst[j] = (R)(residual != nullptr ? d + (float)residual[j] : d);
    }
}

/*
 * The gradient with the bias' part: a lane keeps V columns over the rows of
 * its chunk, tx lanes side by side and kThreads / tx rows at once, and the
 * block's rows are joined in LDS. A row may start anywhere in a group of eight
 * (ALIGNED 0: the columns or the offset are no multiple of V): then V numbers
 * come from two groups.
 */
template <typename R, typename T, int V, bool ALIGNED>
__global__ void __launch_bounds__(kThreads)
k_dropout_grad(T *dsrc, const R *grad, float *dbias, uint64_t rows, uint64_t cols,
               unsigned tx, uint64_t chunk, Rng rng)
{
    __shared__ float lds[kThreads * V];
    const unsigned x  = threadIdx.x % tx, y = threadIdx.x / tx, ty = kThreads / tx;
    const uint64_t c  = ((uint64_t)blockIdx.x * tx + x) * V;
    const uint64_t r0 = (uint64_t)blockIdx.y * chunk;
    const uint64_t r1 = r0 + chunk < rows ? r0 + chunk : rows;
    uint64_t seed, tag;
    rng_state(rng, seed, tag);
    float sum[V] = {};
    if (c < cols) {
        constexpr int U = 4;          /* rows in flight */
        for (uint64_t r = r0 + y; r < r1; r += (uint64_t)U * ty) {
            float g[U][V];
#pragma unroll
            for (int j = 0; j < U; j++) {
                const uint64_t q = r + (uint64_t)j * ty;
                if (q < r1) {
                    load_row<R, V>(grad + q * cols, c, cols, 0.f, g[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < U; j++) {
                const uint64_t q = r + (uint64_t)j * ty;
                if (q < r1) {
                    uint32_t u[V / 2] = {};
                    if (rng.threshold != 0) {
                        draw<V, ALIGNED>(rng.offset + q * cols + c, tag, seed, u);
                    }
#pragma unroll
                    for (int k = 0; k < V; k++) {
                        g[j][k] = kept<V>(u, k, rng.threshold) ? g[j][k] * rng.scale : 0.f;
                        sum[k] += g[j][k];
                    }
                    store_row<T, V>(dsrc + q * cols, c, cols, g[j]);
                }
            }
        }
    }
#pragma unroll
    for (int k = 0; k < V; k++) {
        lds[threadIdx.x * V + k] = sum[k];
    }
    __syncthreads();
    /* column j of the block's tx * V: its rows y = 0, 1, .. in order */
    for (unsigned j = threadIdx.x; j < tx * V; j += kThreads) {
        const uint64_t at = (uint64_t)blockIdx.x * tx * V + j;
        if (at < cols) {
            float s = 0.f;
            for (unsigned q = 0; q < ty; q++) {
                s += lds[q * tx * V + j];
            }
            dbias[(uint64_t)blockIdx.y * cols + at] = s;
        }
    }
}

/* 16 columns by 16 parts of the partials' rows */
template <typename X, typename S>
__device__ __forceinline__ S join_columns(const X *part, uint64_t nparts, uint64_t stride,
                                          uint64_t col, uint64_t cols, S *lds)
{
    const unsigned x = threadIdx.x & 15, y = threadIdx.x >> 4;
    S s = 0;
    if (col < cols) {
#pragma unroll 8
        for (uint64_t p = y; p < nparts; p += 16) {
            s += (S)part[p * stride + col];
        }
    }
    __syncthreads();
    lds[threadIdx.x] = s;
    __syncthreads();
    S t = 0;
    for (unsigned q = 0; q < 16; q++) {
        t += lds[q * 16 + x];
    }
    return t;
}

__global__ void __launch_bounds__(kThreads)
k_join_bias(float *dbias, const float *part, uint64_t nparts, uint64_t cols)
{
    __shared__ double lds[kThreads];
    const uint64_t col = (uint64_t)blockIdx.x * 16 + (threadIdx.x & 15);
    const double s     = join_columns<float, double>(part, nparts, cols, col, cols, lds);
    if (threadIdx.x < 16 && col < cols) {
        dbias[col] = (float)s;
    }
}

/* ======================================================================== */
/* balance loss                                                             */
/* ======================================================================== */
constexpr int kMaxExperts = 1024;

/* exp and log through the hardware's base-2 functions (1 ulp). The difference
 * x - max is taken first and scaled afterwards, so that logits of the type's
 * lowest value (a usual mask) meet no overflow: a row of them alone is uniform. */
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

/* softmax of one row held by G lanes: x becomes exp(x - max); returns the
 * factor that makes it a probability and the log of the sum of exponentials,
 * both 0 for a row of -inf alone */
template <int G, int C>
__device__ __forceinline__ void row_softmax(float (&x)[C], float &inv, float &lse)
{
    float top = x[0];
#pragma unroll
    for (int k = 1; k < C; k++) {
        top = fmaxf(top, x[k]);
    }
    top = group_all<G>(top, Max());
    const float shift = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < C; k++) {
        x[k] = __builtin_amdgcn_exp2f((x[k] - shift) * kLog2e);
        sum += x[k];
    }
    sum = group_all<G>(sum, Add());
    const bool none = sum == 0.f;
    inv = none ? 0.f : 1.f / sum;
    lse = none ? 0.f : __builtin_fmaf(__builtin_amdgcn_logf(sum), kLn2, top);
}

/* the loss' three values from whole counts and sums, by one block */
__device__ __forceinline__ void balance_loss_block(const int64_t *counts, const float *sums,
                                                   unsigned experts, double balance,
                                                   double z_coef, float *loss, double *lds)
{
    double dot = 0;
    for (unsigned e = threadIdx.x; e < experts; e += kThreads) {
        dot += (double)counts[e] * (double)sums[e];
    }
    dot = block_sum(dot, lds);
    if (threadIdx.x == 0) {
        const double n = (double)counts[experts];
        const double b = n > 0 ? balance * dot / (n * n) : 0;
        const double z = n > 0 && z_coef != 0 ? z_coef * (double)sums[experts] / n : 0;
        loss[0] = (float)(b + z);
        loss[1] = (float)b;
        loss[2] = (float)z;
    }
}

struct Balance {
    uint64_t tokens, ld, ld_index, ld_out;
    unsigned experts, topk;
    uint64_t chunk;              /* rows of a block */
    double   balance;            /* balance_coef * experts / topk */
    double   z_coef;
};

/* the partials of all blocks: floats [blocks][experts + 1], then counts of the
 * same shape, then the counter of the joining blocks */
struct BalancePart {
    float    *sums;
    unsigned *counts;
    unsigned *done;
};

/* A row lies in G lanes, V neighbouring columns to a lane and vector, so a
 * wave has 64 / G rows at once and a lane keeps the sums of its columns over
 * all rows of the block. Counts are integers, so their LDS atomics give the
 * same in any order. */
template <typename T, typename I, int G, int NV>
__global__ void __launch_bounds__(kThreads)
k_balance(const T *logits, const I *index, const uint8_t *mask, Balance p, BalancePart out,
          int64_t *counts, float *sums, float *loss)
{
    constexpr int V = 16 / sizeof(T), C = NV * V, R = 64 / G;
    __shared__ float psum[4][G * C + 1];
    __shared__ unsigned hist[G * C + 1];
    __shared__ double join[4];
    const unsigned E    = p.experts;
    const unsigned wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const unsigned l    = lane % G, sub = lane / G;
    for (unsigned e = threadIdx.x; e <= G * C; e += kThreads) {
        hist[e] = 0;
    }
    __syncthreads();
    const uint64_t r0 = (uint64_t)blockIdx.x * p.chunk;
    const uint64_t r1 = r0 + p.chunk < p.tokens ? r0 + p.chunk : p.tokens;
    float acc[C] = {}, zsum = 0.f;
    unsigned live_rows = 0;
    for (uint64_t t = r0 + wave * R + sub; t < r1; t += 4 * R) {
        if (mask != nullptr && mask[t] == 0) {
            continue;                 /* the same for a row's G lanes */
        }
        float x[C];
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float v[V];
            load_row<T, V>(logits + t * p.ld, (j * G + l) * V, E, -INFINITY, v);
#pragma unroll
            for (int k = 0; k < V; k++) {
                x[j * V + k] = v[k];
            }
        }
        for (unsigned k = l; k < p.topk; k += G) {
            const int64_t e = (int64_t)index[t * p.ld_index + k];
            if (e >= 0 && e < (int64_t)E) {
                atomicAdd(&hist[e], 1u);
            }
        }
        float inv, lse;
        row_softmax<G, C>(x, inv, lse);
#pragma unroll
        for (int k = 0; k < C; k++) {
            acc[k] = __builtin_fmaf(x[k], inv, acc[k]);
        }
        zsum = __builtin_fmaf(lse, lse, zsum);
        live_rows++;
    }
    /* rows of the wave, then waves, in a fixed order */
#pragma unroll
    for (int k = 0; k < C; k++) {
        acc[k] = lanes_all(acc[k], G, 64, Add());
    }
    zsum      = lanes_all(zsum, G, 64, Add());
    live_rows = lanes_all(live_rows, G, 64, Add());
    if (sub == 0) {
#pragma unroll
        for (int k = 0; k < C; k++) {
            psum[wave][((k / V) * G + l) * V + k % V] = acc[k];
        }
    }
    if (lane == 0) {
        psum[wave][G * C] = zsum;
        atomicAdd(&hist[G * C], live_rows);
    }
    __syncthreads();
    for (unsigned e = threadIdx.x; e <= E; e += kThreads) {
        const unsigned at = e == E ? G * C : e;
        const double s    = ((double)psum[0][at] + (double)psum[1][at]) +
                         ((double)psum[2][at] + (double)psum[3][at]);
        if (counts != nullptr) {      /* the only block */
            counts[e] = hist[at];
            sums[e]   = (float)s;
        } else {
            out.sums[(uint64_t)blockIdx.x * (E + 1) + e]   = (float)s;
            out.counts[(uint64_t)blockIdx.x * (E + 1) + e] = hist[at];
        }
    }
    if (counts != nullptr) {
        if (loss != nullptr) {
            __syncthreads();
            balance_loss_block(counts, sums, E, p.balance, p.z_coef, loss, join);
        }
    } else if (blockIdx.x == 0 && threadIdx.x == 0) {
        *out.done = 0;
    }
}

__global__ void __launch_bounds__(kThreads)
k_balance_join(BalancePart part, unsigned nparts, Balance p, int64_t *counts, float *sums,
               float *loss)
{
    __shared__ double lds[kThreads];
    __shared__ uint64_t lds_n[kThreads];
    __shared__ unsigned arrived;
    const unsigned n   = p.experts + 1;
    const uint64_t col = (uint64_t)blockIdx.x * 16 + (threadIdx.x & 15);
    const double s     = join_columns<float, double>(part.sums, nparts, n, col, n, lds);
    const uint64_t c   = join_columns<unsigned, uint64_t>(part.counts, nparts, n, col, n, lds_n);
    if (threadIdx.x < 16 && col < n) {
        sums[col]   = (float)s;
        counts[col] = (int64_t)c;
    }
    if (loss != nullptr && last_block(part.done, &arrived)) {
        balance_loss_block(counts, sums, p.experts, p.balance, p.z_coef, loss, lds);
    }
}

__global__ void __launch_bounds__(kThreads)
k_balance_loss(const int64_t *counts, const float *sums, Balance p, float *loss)
{
    __shared__ double lds[4];
    balance_loss_block(counts, sums, p.experts, p.balance, p.z_coef, loss, lds);
}

/* dx_e = grad * p_e ( a (c_e - sum_j p_j c_j) + 2 b lse ), a = balance / N^2,
 * b = z_coef / N. The counts enter less their mean, which the p (that sum to
 * one) cancel: near balance that keeps the digits that the difference needs. */
template <typename T, int G, int NV>
__global__ void __launch_bounds__(kThreads)
k_balance_grad(const T *logits, const uint8_t *mask, const int64_t *counts, const T *base,
               const float *grad_loss, T *dlogits, Balance p)
{
    constexpr int V = 16 / sizeof(T), C = NV * V, R = 64 / G;
    const unsigned E    = p.experts;
    const unsigned wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const unsigned l    = lane % G, sub = lane / G;
    const int64_t tokens = counts[E];
    const int64_t mean   = (int64_t)((double)tokens * p.topk / E);
    const double g       = grad_loss != nullptr ? (double)*grad_loss : 1.0;
    const float a = tokens > 0 ? (float)(g * p.balance / ((double)tokens * (double)tokens)) : 0.f;
    const float b = tokens > 0 ? (float)(g * 2 * p.z_coef / (double)tokens) : 0.f;
    float c[C];
#pragma unroll
    for (int k = 0; k < C; k++) {
        const unsigned e = ((k / V) * G + l) * V + k % V;
        c[k] = e < E ? (float)(counts[e] - mean) : 0.f;
    }
    for (uint64_t t = ((uint64_t)blockIdx.x * 4 + wave) * R + sub; t < p.tokens;
         t += (uint64_t)gridDim.x * 4 * R) {
        const bool live = mask == nullptr || mask[t] != 0;
        float x[C], d[C];
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float v[V] = {}, w[V] = {};
            if (live) {
                load_row<T, V>(logits + t * p.ld, (j * G + l) * V, E, -INFINITY, v);
            }
            if (base != nullptr) {
                load_row<T, V>(base + t * p.ld_out, (j * G + l) * V, E, 0.f, w);
            }
#pragma unroll
            for (int k = 0; k < V; k++) {
                x[j * V + k] = live ? v[k] : -INFINITY;
                d[j * V + k] = w[k];
            }
        }
        float inv, lse;
        row_softmax<G, C>(x, inv, lse);
        float dot = 0.f;
#pragma unroll
        for (int k = 0; k < C; k++) {
            x[k] *= inv;
            dot = __builtin_fmaf(x[k], c[k], dot);
        }
        dot = group_all<G>(dot, Add());
        const float z = b * lse;
#pragma unroll
        for (int k = 0; k < C; k++) {
            const float s = __builtin_fmaf(x[k], __builtin_fmaf(a, c[k] - dot, z), d[k]);
            d[k] = live ? s : d[k];   /* whatever grad_loss is */
        }
#pragma unroll
        for (int j = 0; j < NV; j++) {
            float v[V];
#pragma unroll
            for (int k = 0; k < V; k++) {
                v[k] = d[j * V + k];
            }
            if ((unsigned)(j * G + l) * V < E) {
                store_row<T, V>(dlogits + t * p.ld_out, (j * G + l) * V, E, v);
            }
        }
    }
}

/* ======================================================================== */
/* policy loss                                                              */
/* ======================================================================== */
struct Policy {
    uint64_t rows, cols, ld;
    int      adv_per_row, per_sequence;
    unsigned lanes;              /* that share a row: a power of two */
    unsigned steps;              /* vectors of a lane */
    uint64_t chunks;             /* parts of a row */
    float    up, down;           /* log(1 + clip_high), log(1 - clip_low) */
    float    ratio_up, ratio_down;
    float    kl_coef;
    double   kl_coef64;
};

struct PolicyPart {              /* of one part of a row */
    float    pg, kl;
    unsigned tokens, cut;
};

struct PolicySum {
    double   pg, kl;
    uint64_t tokens, rows, cut;
};

/* exp(q) - q - 1, by its series near nought, where the subtractions would
 * leave nothing (to q^10 / 10!: the rest is below 5e-9 of it there) */
__device__ __forceinline__ float exp_less(float q)
{
    float s = 1.f / 3628800.f;
    s = __builtin_fmaf(s, q, 1.f / 362880.f);
    s = __builtin_fmaf(s, q, 1.f / 40320.f);
    s = __builtin_fmaf(s, q, 1.f / 5040.f);
    s = __builtin_fmaf(s, q, 1.f / 720.f);
    s = __builtin_fmaf(s, q, 1.f / 120.f);
    s = __builtin_fmaf(s, q, 1.f / 24.f);
    s = __builtin_fmaf(s, q, 1.f / 6.f);
    s = __builtin_fmaf(s, q, 0.5f);
    return fabsf(q) < 0.75f ? s * q * q : expf(q) - q - 1.f;
}

/* whether a token is cut goes by d itself, not by its rounded exponential */
__device__ __forceinline__ bool is_cut(float a, float d, const Policy &p)
{
    return (a > 0.f && d > p.up) || (a < 0.f && d < p.down);
}

/* the operands of V tokens of a row, and which of them count */
template <typename T, int V>
struct Tokens {
    float logp[V], old[V], ref[V], adv[V];
    bool  live[V];

    __device__ __forceinline__ void load(const T *lp, const T *op, const T *rp,
                                         const float *ap, const uint8_t *mp, const Policy &p,
                                         uint64_t row, uint64_t c)
    {
        const uint64_t at = row * p.ld;
        load_row<T, V>(lp + at, c, p.cols, 0.f, logp);
        load_row<T, V>(op + at, c, p.cols, 0.f, old);
        if (rp != nullptr) {
            load_row<T, V>(rp + at, c, p.cols, 0.f, ref);
        }
        if (p.adv_per_row) {
            const float a = ap[row];
#pragma unroll
            for (int k = 0; k < V; k++) {
                adv[k] = a;
            }
        } else {
            load_row<float, V>(ap + at, c, p.cols, 0.f, adv);
        }
        if (mp == nullptr) {
#pragma unroll
            for (int k = 0; k < V; k++) {
                live[k] = c + k < p.cols;
            }
        } else if (c + V <= p.cols) {
            uint8_t m[V];
            load_raw<uint8_t, V>(mp + at + c, m);
#pragma unroll
            for (int k = 0; k < V; k++) {
                live[k] = m[k] != 0;
            }
        } else {
#pragma unroll
            for (int k = 0; k < V; k++) {
                live[k] = c + k < p.cols && mp[at + c + k] != 0;
            }
        }
    }
};

/* the join of a row's parts, of the rows, and the results; by blocks that each
 * take rows b, b + gridDim.x, .. groups of them */
__device__ __forceinline__ PolicySum policy_rows(const PolicyPart *part, const Policy &p,
                                                 int32_t *row_tokens, unsigned lanes)
{
    PolicySum sum = {};
    const unsigned l = threadIdx.x % lanes, per = kThreads / lanes;
    for (uint64_t r = (uint64_t)blockIdx.x * per + threadIdx.x / lanes; r < p.rows;
         r += (uint64_t)gridDim.x * per) {
        double pg = 0, kl = 0;
        unsigned long long tokens = 0, cut = 0;
        for (uint64_t w = l; w < p.chunks; w += lanes) {
            const PolicyPart &x = part[r * p.chunks + w];
            pg += x.pg;
            kl += x.kl;
            tokens += x.tokens;
            cut += x.cut;
        }
        pg     = lanes_all(pg, 1, lanes, Add());
        kl     = lanes_all(kl, 1, lanes, Add());
        tokens = lanes_all(tokens, 1, lanes, Add());
        cut    = lanes_all(cut, 1, lanes, Add());
        if (l == 0) {
            const double w = p.per_sequence && tokens ? 1.0 / (double)tokens : 1.0;
            sum.pg += pg * w;
            sum.kl += kl * w;
            sum.tokens += tokens;
            sum.rows += tokens != 0;
            sum.cut += cut;
            if (row_tokens != nullptr) {
                row_tokens[r] = (int32_t)tokens;
            }
        }
    }
    return sum;
}

__device__ __forceinline__ PolicySum policy_block(PolicySum s, double *lds)
{
    unsigned long long *n = reinterpret_cast<unsigned long long*>(lds + 4);
    PolicySum t;
    t.pg     = block_sum(s.pg, lds);
    t.kl     = block_sum(s.kl, lds);
    t.tokens = block_sum((unsigned long long)s.tokens, n);
    t.rows   = block_sum((unsigned long long)s.rows, n);
    t.cut    = block_sum((unsigned long long)s.cut, n);
    return t;
}

__device__ __forceinline__ void policy_loss_values(double pg, double kl, int64_t n,
                                                   double kl_coef, float *loss)
{
    pg = n > 0 ? pg / (double)n : 0;
    kl = n > 0 ? kl / (double)n : 0;
    loss[0] = (float)(pg + kl_coef * kl);
    loss[1] = (float)pg;
    loss[2] = (float)kl;
}

__device__ __forceinline__ void policy_write(const PolicySum &s, const Policy &p, float *sums,
                                             int64_t *counts, float *loss)
{
    sums[0]   = (float)s.pg;
    sums[1]   = (float)s.kl;
    counts[0] = (int64_t)s.tokens;
    counts[1] = (int64_t)s.rows;
    counts[2] = (int64_t)s.cut;
    if (loss != nullptr) {
        policy_loss_values(s.pg, s.kl, p.per_sequence ? counts[1] : counts[0], p.kl_coef64, loss);
    }
}

/* A wave does one part of 64 / lanes rows at a time: `steps` vectors of each
 * of the lanes that share the row. One block (single): it joins them too. */
template <typename T>
__global__ void __launch_bounds__(kThreads)
k_policy(const T *logp, const T *old, const T *ref, const float *adv, const uint8_t *mask,
         Policy p, PolicyPart *part, unsigned *done, int single, float *sums, int64_t *counts,
         int32_t *row_tokens, float *loss)
{
    constexpr int V = 16 / sizeof(T);
    __shared__ double lds[8];
    const unsigned lane = threadIdx.x & 63, l = lane % p.lanes, per = 64 / p.lanes;
    const uint64_t tiles = (p.rows + per - 1) / per, items = tiles * p.chunks;
    for (uint64_t it = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); it < items;
         it += (uint64_t)gridDim.x * 4) {
        const uint64_t chunk = it % p.chunks;
        const uint64_t row   = it / p.chunks * per + lane / p.lanes;
        float pg = 0.f, kl = 0.f;
        unsigned tokens = 0, cut = 0;
        if (row < p.rows) {
            const uint64_t c0 = chunk * p.steps * p.lanes * V + l * V;
#pragma unroll 2
            for (unsigned j = 0; j < p.steps; j++) {
                const uint64_t c = c0 + (uint64_t)j * p.lanes * V;
                if (c >= p.cols) {
                    break;
                }
                Tokens<T, V> t;
                t.load(logp, old, ref, adv, mask, p, row, c);
#pragma unroll
                for (int k = 0; k < V; k++) {
                    const float d = t.logp[k] - t.old[k];
                    const bool is = is_cut(t.adv[k], d, p);
                    const float r = is ? (t.adv[k] > 0.f ? p.ratio_up : p.ratio_down) : expf(d);
                    const float e = ref != nullptr ? exp_less(t.ref[k] - t.logp[k]) : 0.f;
                    pg += t.live[k] ? -t.adv[k] * r : 0.f;
                    kl += t.live[k] ? e : 0.f;
                    tokens += t.live[k];
                    cut += t.live[k] && is;
                }
            }
        }
        pg     = lanes_all(pg, 1, p.lanes, Add());
        kl     = lanes_all(kl, 1, p.lanes, Add());
        tokens = lanes_all(tokens, 1, p.lanes, Add());
        cut    = lanes_all(cut, 1, p.lanes, Add());
        if (l == 0 && row < p.rows) {
            part[row * p.chunks + chunk] = {pg, kl, tokens, cut};
        }
    }
    if (single) {
        __threadfence();
        __syncthreads();
        const PolicySum s = policy_block(policy_rows(part, p, row_tokens, 1), lds);
        if (threadIdx.x == 0) {
            policy_write(s, p, sums, counts, loss);
        }
    } else if (blockIdx.x == 0 && threadIdx.x == 0) {
        *done = 0;
    }
}

__global__ void __launch_bounds__(kThreads)
k_policy_join(const PolicyPart *part, PolicySum *block, unsigned *done, Policy p, unsigned lanes,
              float *sums, int64_t *counts, int32_t *row_tokens, float *loss)
{
    __shared__ double lds[8];
    __shared__ unsigned arrived;
    PolicySum s = policy_block(policy_rows(part, p, row_tokens, lanes), lds);
    if (threadIdx.x == 0) {
        block[blockIdx.x] = s;
    }
    if (last_block(done, &arrived)) {
        PolicySum t = {};
        if (threadIdx.x < gridDim.x) {
            t = block[threadIdx.x];
        }
        t = policy_block(t, lds);
        if (threadIdx.x == 0) {
            policy_write(t, p, sums, counts, loss);
        }
    }
}

__global__ void k_policy_loss(const float *sums, const int64_t *counts, int per_sequence,
                              double kl_coef, float *loss)
{
    policy_loss_values(sums[0], sums[1], per_sequence ? counts[1] : counts[0], kl_coef, loss);
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
k_policy_grad(const T *logp, const T *old, const T *ref, const float *adv, const uint8_t *mask,
              const int32_t *row_tokens, const int64_t *counts, const float *grad_loss, T *dlogp,
              Policy p)
{
    constexpr int V = 16 / sizeof(T);
    const unsigned lane = threadIdx.x & 63, l = lane % p.lanes, per = 64 / p.lanes;
    const uint64_t tiles = (p.rows + per - 1) / per, items = tiles * p.chunks;
    const double g   = grad_loss != nullptr ? (double)*grad_loss : 1.0;
    const int64_t n  = p.per_sequence ? counts[1] : counts[0];
    const double all = n > 0 ? g / (double)n : 0;
    for (uint64_t it = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); it < items;
         it += (uint64_t)gridDim.x * 4) {
        const uint64_t chunk = it % p.chunks;
        const uint64_t row   = it / p.chunks * per + lane / p.lanes;
        if (row >= p.rows) {
            continue;
        }
        float w = (float)all;
        if (p.per_sequence) {
            const int32_t m = row_tokens[row];
            w = m > 0 ? (float)(all / m) : 0.f;
        }
        const uint64_t c0 = chunk * p.steps * p.lanes * V + l * V;
#pragma unroll 2
        for (unsigned j = 0; j < p.steps; j++) {
            const uint64_t c = c0 + (uint64_t)j * p.lanes * V;
            if (c >= p.cols) {
                break;
            }
            Tokens<T, V> t;
            t.load(logp, old, ref, adv, mask, p, row, c);
            float o[V];
#pragma unroll
            for (int k = 0; k < V; k++) {
                const float d = t.logp[k] - t.old[k];
                float x = is_cut(t.adv[k], d, p) ? 0.f : -t.adv[k] * expf(d);
                if (ref != nullptr) {
                    const float q = t.ref[k] - t.logp[k];
                    x = __builtin_fmaf(-p.kl_coef, exp_less(q) + q, x);   /* 1 - exp(q) */
                }
                o[k] = t.live[k] ? x * w : 0.f;
            }
            store_row<T, V>(dlogp + row * p.ld, c, p.cols, o);
        }
    }
}

/* ======================================================================== */
/* host side                                                                */
/* ======================================================================== */
/* the context's device current for the call, the caller's one afterwards */
struct OnDevice {
    int        before = -1;
    hipError_t err;

    explicit OnDevice(int device)
    {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) {
            err = hipSetDevice(device);
        } else {
            before = -1;
        }
    }
    ~OnDevice()
    {
        if (before >= 0) {
            (void)hipSetDevice(before);
        }
    }
};

inline uint64_t div_up(uint64_t a, uint64_t b) { return a / b + (a % b != 0); }

ucs_status_t invalid(const char *what, const char *why)
{
    return set_error(UCS_ERR_INVALID_PARAM, what, why);
}

bool is_float_dt(int dt)
{
    return dt == UCG_DEV_DT_FLOAT32 || dt == UCG_DEV_DT_BFLOAT16 || dt == UCG_DEV_DT_FLOAT16;
}

size_t size_of(int dt)
{
    return dt == UCG_DEV_DT_FLOAT32 ? 4 : 2;
}

bool misaligned(const void *p, size_t size)
{
    return ((uintptr_t)p % size) != 0;
}

/* whether two ranges share bytes */
bool overlap(const void *a, size_t na, const void *b, size_t nb)
{
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return na != 0 && nb != 0 && x < y + nb && y < x + na;
}

/* rows x cols elements of `size` bytes, a row every ld: their span in bytes.
 * False when that does not fit in 63 bits. */
bool span(uint64_t rows, uint64_t cols, uint64_t ld, size_t size, size_t *bytes)
{
    uint64_t n = 0;
    if (rows != 0 && cols != 0 &&
        (__builtin_mul_overflow(rows - 1, ld, &n) || __builtin_add_overflow(n, cols, &n) ||
         __builtin_mul_overflow(n, (uint64_t)size, &n) || n > (uint64_t)INT64_MAX)) {
        return false;
    }
    *bytes = n;
    return true;
}

hipStream_t stream_of(ucg_builtin_dev_ctx_t *ctx)
{
    return (hipStream_t)ucg_builtin_dev_ctx_stream(ctx);
}

template <typename F>
void with_float(int dt, F f)
{
    if (dt == UCG_DEV_DT_FLOAT32) {
        f(float());
    } else if (dt == UCG_DEV_DT_BFLOAT16) {
        f(bf16());
    } else {
        f(f16());
    }
}

/* (T of dt, R of out_dt): out_dt is dt or FLOAT32 */
template <typename F>
void with_pair(int dt, int out_dt, F f)
{
    with_float(dt, [&](auto t) {
        typedef decltype(t) T;
        if (out_dt == dt) {
            f(T(), T());
        } else {
            f(T(), float());
        }
    });
}

/* ---- dropout ---- */
/* elements of a lane: a whole group of eight where 16 bytes hold it, half a
 * group where a 32-bit operand would need two loads for it */
template <typename T, typename R>
constexpr int drop_vec()
{
    return sizeof(T) == 2 && sizeof(R) == 2 ? 8 : 4;
}

/* work-items of one launch (a dispatch counts them in 32 bits) */
constexpr uint64_t kMaxItems = (uint64_t)1 << 31;
/* columns of a bias whose gradient one launch can join (16 to a block) */
constexpr uint64_t kMaxBias = (uint64_t)1 << 27;

template <typename T, typename R, int N>
void launch_sum(hipStream_t st, R *dst, const SrcList &srcs, unsigned nsrc, const T *bias,
                const R *residual, uint64_t n, uint64_t cols, const Rng &rng)
{
    constexpr int V = drop_vec<T, R>();
    const uint64_t inv    = cols == 1 ? 0 : UINT64_MAX / cols + 1;
    const uint64_t groups = div_up(n + rng.offset % V, V);
    for (uint64_t first = 0; first < groups; first += kMaxItems) {
        const uint64_t left = groups - first < kMaxItems ? groups - first : kMaxItems;
        hipLaunchKernelGGL((k_sum_dropout<T, R, V, N>), dim3((unsigned)div_up(left, kThreads)),
                           dim3(kThreads), 0, st, dst, srcs, nsrc, bias, residual, n, first,
                           cols, inv, rng);
    }
}

template <typename T, typename R>
void launch_sum_n(hipStream_t st, R *dst, const SrcList &srcs, unsigned nsrc, const T *bias,
                  const R *residual, uint64_t n, uint64_t cols, const Rng &rng)
{
    switch (nsrc) {
    case 1: launch_sum<T, R, 1>(st, dst, srcs, nsrc, bias, residual, n, cols, rng); break;
    case 2: launch_sum<T, R, 2>(st, dst, srcs, nsrc, bias, residual, n, cols, rng); break;
    case 3: launch_sum<T, R, 3>(st, dst, srcs, nsrc, bias, residual, n, cols, rng); break;
    case 4: launch_sum<T, R, 4>(st, dst, srcs, nsrc, bias, residual, n, cols, rng); break;
    case 8: launch_sum<T, R, 8>(st, dst, srcs, nsrc, bias, residual, n, cols, rng); break;
    case 16: launch_sum<T, R, 16>(st, dst, srcs, nsrc, bias, residual, n, cols, rng); break;
    default: launch_sum<T, R, 0>(st, dst, srcs, nsrc, bias, residual, n, cols, rng); break;
    }
}

/* how the gradient with the bias' part cuts its rows: the same for every type,
 * so that the workspace goes by the sizes alone (V = 4 gives the most parts) */
struct GradPlan {
    unsigned tx;                 /* lanes side by side */
    uint64_t blocks_x, parts, chunk;
};

GradPlan grad_plan(uint64_t rows, uint64_t cols, int V)
{
    GradPlan g;
    const uint64_t groups = div_up(cols, V);
    g.tx = 1;
    while (g.tx < (unsigned)kThreads && g.tx < groups) {
        g.tx *= 2;
    }
    g.blocks_x        = div_up(groups, g.tx);
    const uint64_t ty = kThreads / g.tx;
    /* 1024 blocks, at most 256 parts to join, four rows a lane at least */
    uint64_t parts = div_up(1024, g.blocks_x);
    parts   = parts < 256 ? parts : 256;
    const uint64_t most = div_up(rows, ty * 4);
    parts   = parts < most ? parts : most;
    parts   = parts > 0 ? parts : 1;
    g.chunk = div_up(rows, parts);
    g.parts = g.chunk ? div_up(rows, g.chunk) : 1;
    return g;
}

ucs_status_t dropout_rng(const ucg_builtin_dev_dropout_params_t *p, const char *what, Rng *rng,
                         uint64_t *n)
{
    if (p == nullptr) {
        return invalid(what, "params is NULL");
    }
    if (!is_float_dt(p->dt) || (p->out_dt != p->dt && p->out_dt != UCG_DEV_DT_FLOAT32)) {
        return set_error(UCS_ERR_UNSUPPORTED, what,
                         "dt must be float32, bfloat16 or float16, out_dt dt or float32");
    }
    if (!(p->p >= 0.0 && p->p <= 1.0)) {
        return invalid(what, "p must be in [0, 1]");
    }
    size_t bytes;
    if (!span(p->rows, p->cols, p->cols, 4, &bytes)) {
        return invalid(what, "rows x cols does not fit");
    }
    *n = (uint64_t)p->rows * p->cols;
    if (p->offset + *n < p->offset || p->offset + *n > (uint64_t)INT64_MAX) {
        return invalid(what, "offset + rows x cols must be below 2^63");
    }
    if (misaligned(p->rng, 8)) {
        return invalid(what, "misaligned rng");
    }
    rng->seed      = p->seed;
    rng->tag       = p->tag;
    rng->offset    = p->offset;
    rng->dev       = p->rng;
    rng->threshold = (uint32_t)lrint(p->p * 65536.0);
    rng->scale     = rng->threshold < 65536 ? (float)(65536.0 / (65536 - rng->threshold)) : 0.f;
    return UCS_OK;
}

/* ---- balance ---- */
ucs_status_t balance_check(const ucg_builtin_dev_balance_params_t *p, const char *what,
                           Balance *b)
{
    if (p == nullptr) {
        return invalid(what, "params is NULL");
    }
    if (!is_float_dt(p->dt) ||
        (p->index_dt != UCG_DEV_DT_INT32 && p->index_dt != UCG_DEV_DT_INT64)) {
        return set_error(UCS_ERR_UNSUPPORTED, what,
                         "dt must be float32, bfloat16 or float16, index_dt int32 or int64");
    }
    if (p->experts < 1 || p->experts > (size_t)kMaxExperts || p->topk < 1 ||
        p->topk > p->experts) {
        return invalid(what, "experts must be 1..1024 and topk 1..experts");
    }
    if (!isfinite(p->balance_coef) || !isfinite(p->z_coef)) {
        return invalid(what, "the coefficients must be finite");
    }
    b->tokens   = p->tokens;
    b->experts  = (unsigned)p->experts;
    b->topk     = (unsigned)p->topk;
    b->ld       = p->ld ? p->ld : p->experts;
    b->ld_index = p->ld_index ? p->ld_index : p->topk;
    b->ld_out   = p->ld_out ? p->ld_out : p->experts;
    b->chunk    = 0;
    b->balance  = p->balance_coef * (double)p->experts / (double)p->topk;
    b->z_coef   = p->z_coef;
    if (b->ld < p->experts || b->ld_index < p->topk || b->ld_out < p->experts) {
        return invalid(what, "a row step is smaller than the row");
    }
    return UCS_OK;
}

/* blocks of k_balance: enough for every CU, few enough to join; a multiple of
 * 64 rows each, so that no more than one of them is short whatever G is */
void balance_plan(uint64_t tokens, uint64_t *blocks, uint64_t *chunk)
{
    constexpr uint64_t kMost = 512;
    uint64_t c = div_up(div_up(tokens, kMost), 64) * 64;
    c       = c ? c : 64;
    *chunk  = c;
    *blocks = tokens ? div_up(tokens, c) : 1;
}

/* f(T, G lanes to a row, NV vectors to a lane) for `experts` columns */
template <typename T, typename F>
void with_layout(unsigned experts, F f)
{
    constexpr unsigned V = 16 / sizeof(T);
    const unsigned groups = (unsigned)div_up(experts, V);
    typedef std::integral_constant<int, 1> one;
    if (groups <= 1) {
        f(one(), one());
    } else if (groups <= 2) {
        f(std::integral_constant<int, 2>(), one());
    } else if (groups <= 4) {
        f(std::integral_constant<int, 4>(), one());
    } else if (groups <= 8) {
        f(std::integral_constant<int, 8>(), one());
    } else if (groups <= 16) {
        f(std::integral_constant<int, 16>(), one());
    } else if (groups <= 32) {
        f(std::integral_constant<int, 32>(), one());
    } else if (groups <= 64) {
        f(std::integral_constant<int, 64>(), one());
    } else if (groups <= 128) {
        f(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
    } else if constexpr (V == 4) {
        f(std::integral_constant<int, 64>(), std::integral_constant<int, 4>());
    }
}

/* ---- policy ---- */
constexpr unsigned kPolicyJoin = 64;      /* joining blocks at most */

void policy_split(uint64_t cols, int V, Policy *p)
{
    const uint64_t groups = div_up(cols, V);
    p->lanes = 1;
    while (p->lanes < 64 && p->lanes < groups) {
        p->lanes *= 2;
    }
    const uint64_t vecs = div_up(groups, p->lanes);
    p->steps  = (unsigned)(vecs < 4 ? (vecs ? vecs : 1) : 4);
    p->chunks = vecs ? div_up(vecs, p->steps) : 1;
}

ucs_status_t policy_check(const ucg_builtin_dev_policy_params_t *q, const char *what, Policy *p,
                          size_t *bytes)
{
    if (q == nullptr) {
        return invalid(what, "params is NULL");
    }
    if (!is_float_dt(q->dt)) {
        return set_error(UCS_ERR_UNSUPPORTED, what, "dt must be float32, bfloat16 or float16");
    }
    if (!(q->clip_low >= 0.0 && q->clip_low <= 1.0) ||
        !(q->clip_high >= 0.0 && isfinite(q->clip_high)) || !isfinite(q->kl_coef)) {
        return invalid(what, "clip_low must be in [0, 1], clip_high finite and not negative, "
                             "kl_coef finite");
    }
    p->rows = q->rows;
    p->cols = q->cols;
    p->ld   = q->ld ? q->ld : q->cols;
    if (p->ld < q->cols) {
        return invalid(what, "a row step is smaller than the row");
    }
    if (q->cols > (size_t)INT32_MAX || q->rows > ((size_t)1 << 48) || !span(q->rows, q->cols, p->ld, 4, bytes)) {
        return invalid(what, "rows x cols does not fit");
    }
    p->adv_per_row  = q->adv_per_row;
    p->per_sequence = q->per_sequence;
    p->up           = (float)log1p(q->clip_high);
    p->down         = (float)log1p(-q->clip_low);
    p->ratio_up     = (float)(1 + q->clip_high);
    p->ratio_down   = (float)(1 - q->clip_low);
    p->kl_coef      = (float)q->kl_coef;
    p->kl_coef64    = q->kl_coef;
    policy_split(q->cols, 16 / (int)size_of(q->dt), p);
    return UCS_OK;
}

unsigned policy_grid(const Policy &p)
{
    const uint64_t items = div_up(p.rows, 64 / p.lanes) * p.chunks;
    const uint64_t b     = div_up(items, 4);
    return (unsigned)(b < (1u << 20) ? (b ? b : 1) : (1u << 20));
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

}  // namespace

extern "C" {

/* ------------------------------------------------------------------------ */
ucs_status_t ucg_builtin_dev_sum_dropout(ucg_builtin_dev_ctx_t *ctx,
                                         const ucg_builtin_dev_dropout_params_t *params,
                                         void *dst, const void *const *srcs, unsigned nsrc,
                                         const void *bias, const void *residual)
{
    static const char what[] = "sum_dropout";
    Rng rng;
    uint64_t n;
    ucs_status_t st = dropout_rng(params, what, &rng, &n);
    if (st != UCS_OK) {
        return st;
    }
    if (nsrc == 0 || nsrc > (unsigned)kMaxMulti || srcs == nullptr) {
        return invalid(what, "nsrc must be 1..16 and srcs non-NULL");
    }
    const size_t ts = size_of(params->dt), rs = size_of(params->out_dt);
    SrcList list;
    for (unsigned i = 0; i < (unsigned)kMaxMulti; i++) {
        list.p[i] = i < nsrc ? srcs[i] : nullptr;
    }
    if (n != 0) {
        if (dst == nullptr || misaligned(dst, rs) || misaligned(residual, rs) ||
            misaligned(bias, ts)) {
            return invalid(what, "NULL dst or a misaligned buffer");
        }
        for (unsigned i = 0; i < nsrc; i++) {
            if (list.p[i] == nullptr || misaligned(list.p[i], ts)) {
                return invalid(what, "NULL or misaligned source");
            }
            if ((list.p[i] != dst || ts != rs) && overlap(dst, n * rs, list.p[i], n * ts)) {
                return invalid(what, "dst overlaps a source");
            }
        }
        if ((residual != dst && residual != nullptr && overlap(dst, n * rs, residual, n * rs)) ||
            (bias != nullptr && overlap(dst, n * rs, bias, params->cols * ts))) {
            return invalid(what, "dst overlaps the residual or the bias");
        }
    }
    if (ctx == nullptr) {
        return invalid(what, "ctx is NULL");
    }
    if (n == 0) {
        return UCS_OK;
    }
    OnDevice dev(dev_ctx_device(ctx));
    HIP_TRY(dev.err);
    with_pair(params->dt, params->out_dt, [&](auto t, auto r) {
        typedef decltype(t) T;
        typedef decltype(r) R;
        launch_sum_n<T, R>(stream_of(ctx), static_cast<R*>(dst), list, nsrc,
                           static_cast<const T*>(bias), static_cast<const R*>(residual), n,
                           params->cols, rng);
    });
    HIP_TRY(hipGetLastError());
    dev_ctx_count(ctx, 1, n * (nsrc * ts + (residual ? 2 : 1) * rs));
    return UCS_OK;
}

size_t ucg_builtin_dev_sum_dropout_grad_workspace(size_t rows, size_t cols)
{
    size_t most = 0;
    if (cols == 0 || cols > kMaxBias) {
        return 0;
    }
    for (int v : {4, 8}) {
        const GradPlan g   = grad_plan(rows, cols, v);
        const size_t bytes = g.parts > 1 ? g.parts * cols * sizeof(float) : 0;
        most = bytes > most ? bytes : most;
    }
    return round16(most);
}

ucs_status_t ucg_builtin_dev_sum_dropout_grad(ucg_builtin_dev_ctx_t *ctx,
                                              const ucg_builtin_dev_dropout_params_t *params,
                                              void *dsrc, const void *grad, float *dbias,
                                              void *workspace, size_t workspace_bytes)
{
    static const char what[] = "sum_dropout_grad";
    Rng rng;
    uint64_t n;
    ucs_status_t st = dropout_rng(params, what, &rng, &n);
    if (st != UCS_OK) {
        return st;
    }
    const size_t ts = size_of(params->dt), rs = size_of(params->out_dt);
    const uint64_t rows = params->rows, cols = params->cols;
    if (dbias != nullptr && cols > kMaxBias) {
        return invalid(what, "a bias of more than 2^27 columns");
    }
    const size_t need = dbias ? ucg_builtin_dev_sum_dropout_grad_workspace(rows, cols) : 0;
    if (n != 0 && (dsrc == nullptr || grad == nullptr || misaligned(dsrc, ts) ||
                   misaligned(grad, rs))) {
        return invalid(what, "NULL or misaligned dsrc or grad");
    }
    if (misaligned(dbias, 4) || misaligned(workspace, 16)) {
        return invalid(what, "misaligned dbias or workspace");
    }
    if (need != 0 && (workspace == nullptr || workspace_bytes < need)) {
        return invalid(what, "the workspace is missing or too small");
    }
    if (((dsrc != grad || ts != rs) && overlap(dsrc, n * ts, grad, n * rs)) ||
        (dbias != nullptr &&
         (overlap(dbias, cols * 4, dsrc, n * ts) || overlap(dbias, cols * 4, grad, n * rs))) ||
        (need != 0 && (overlap(workspace, need, dsrc, n * ts) ||
                       overlap(workspace, need, grad, n * rs) ||
                       overlap(workspace, need, dbias, cols * 4)))) {
        return invalid(what, "overlapping buffers");
    }
    if (ctx == nullptr) {
        return invalid(what, "ctx is NULL");
    }
    if (cols == 0 || (n == 0 && dbias == nullptr)) {
        return UCS_OK;
    }
    OnDevice dev(dev_ctx_device(ctx));
    HIP_TRY(dev.err);
    hipStream_t stream = stream_of(ctx);
    with_pair(params->dt, params->out_dt, [&](auto t, auto r) {
        typedef decltype(t) T;
        typedef decltype(r) R;
        T *d       = static_cast<T*>(dsrc);
        const R *g = static_cast<const R*>(grad);
        if (dbias == nullptr) {
            SrcList list = {};
            list.p[0]    = grad;
            launch_sum<R, T, 1>(stream, d, list, 1, nullptr, nullptr, n, cols, rng);
            dev_ctx_count(ctx, 1, 0);
            return;
        }
        constexpr int V     = drop_vec<T, R>();
        const GradPlan plan = grad_plan(rows, cols, V);
        float *out          = plan.parts > 1 ? static_cast<float*>(workspace) : dbias;
        const dim3 grid((unsigned)plan.blocks_x, (unsigned)plan.parts);
        if (cols % V == 0 && rng.offset % V == 0) {
            hipLaunchKernelGGL((k_dropout_grad<R, T, V, true>), grid, dim3(kThreads), 0, stream,
                               d, g, out, rows, cols, plan.tx, plan.chunk, rng);
        } else {
            hipLaunchKernelGGL((k_dropout_grad<R, T, V, false>), grid, dim3(kThreads), 0, stream,
                               d, g, out, rows, cols, plan.tx, plan.chunk, rng);
        }
        if (plan.parts > 1) {
            hipLaunchKernelGGL(k_join_bias, dim3((unsigned)div_up(cols, 16)), dim3(kThreads), 0,
                               stream, dbias, out, plan.parts, cols);
        }
        dev_ctx_count(ctx, plan.parts > 1 ? 2 : 1, 0);
    });
    HIP_TRY(hipGetLastError());
    return UCS_OK;
}

/* ------------------------------------------------------------------------ */
size_t ucg_builtin_dev_balance_workspace(size_t tokens, size_t experts)
{
    uint64_t blocks, chunk;
    balance_plan(tokens, &blocks, &chunk);
    return blocks > 1 ? round16(blocks * (experts + 1) * 8 + 4) : 0;
}

ucs_status_t ucg_builtin_dev_balance(ucg_builtin_dev_ctx_t *ctx,
                                     const ucg_builtin_dev_balance_params_t *params,
                                     const void *logits, const void *index, const uint8_t *mask,
                                     int64_t *counts, float *sums, float *loss, void *workspace,
                                     size_t workspace_bytes)
{
    static const char what[] = "balance";
    Balance b;
    ucs_status_t st = balance_check(params, what, &b);
    if (st != UCS_OK) {
        return st;
    }
    const size_t ts = size_of(params->dt), is = params->index_dt == UCG_DEV_DT_INT32 ? 4 : 8;
    size_t bytes, index_bytes;
    if (!span(b.tokens, b.experts, b.ld, ts, &bytes) ||
        !span(b.tokens, b.topk, b.ld_index, is, &index_bytes)) {
        return invalid(what, "tokens x row step does not fit");
    }
    if (counts == nullptr || sums == nullptr ||
        (b.tokens != 0 && (logits == nullptr || index == nullptr))) {
        return invalid(what, "NULL buffer");
    }
    if (misaligned(logits, ts) || misaligned(index, is) || misaligned(counts, 8) ||
        misaligned(sums, 4) || misaligned(loss, 4) || misaligned(workspace, 16)) {
        return invalid(what, "misaligned buffer");
    }
    const size_t need = ucg_builtin_dev_balance_workspace(b.tokens, b.experts);
    if (need != 0 && (workspace == nullptr || workspace_bytes < need)) {
        return invalid(what, "the workspace is missing or too small");
    }
    if (ctx == nullptr) {
        return invalid(what, "ctx is NULL");
    }
    uint64_t blocks;
    balance_plan(b.tokens, &blocks, &b.chunk);
    BalancePart part = {};
    if (blocks > 1) {
        part.sums   = static_cast<float*>(workspace);
        part.counts = reinterpret_cast<unsigned*>(part.sums + blocks * (b.experts + 1));
        part.done   = part.counts + blocks * (b.experts + 1);
    }
    OnDevice dev(dev_ctx_device(ctx));
    HIP_TRY(dev.err);
    hipStream_t stream = stream_of(ctx);
    int64_t *direct    = blocks > 1 ? nullptr : counts;
    with_float(params->dt, [&](auto t) {
        typedef decltype(t) T;
        with_layout<T>(b.experts, [&](auto g, auto nv) {
            constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
            if (is == 4) {
                hipLaunchKernelGGL((k_balance<T, int32_t, G, NV>), dim3((unsigned)blocks),
                                   dim3(kThreads), 0, stream, static_cast<const T*>(logits),
                                   static_cast<const int32_t*>(index), mask, b, part, direct,
                                   sums, loss);
            } else {
                hipLaunchKernelGGL((k_balance<T, int64_t, G, NV>), dim3((unsigned)blocks),
                                   dim3(kThreads), 0, stream, static_cast<const T*>(logits),
                                   static_cast<const int64_t*>(index), mask, b, part, direct,
                                   sums, loss);
            }
        });
    });
    if (blocks > 1) {
        hipLaunchKernelGGL(k_balance_join, dim3((unsigned)div_up(b.experts + 1, 16)),
                           dim3(kThreads), 0, stream, part, (unsigned)blocks, b, counts, sums,
                           loss);
    }
    HIP_TRY(hipGetLastError());
    dev_ctx_count(ctx, blocks > 1 ? 2 : 1, 0);
    return UCS_OK;
}

ucs_status_t ucg_builtin_dev_balance_loss(ucg_builtin_dev_ctx_t *ctx,
                                          const ucg_builtin_dev_balance_params_t *params,
                                          const int64_t *counts, const float *sums, float *loss)
{
    static const char what[] = "balance_loss";
    Balance b;
    ucs_status_t st = balance_check(params, what, &b);
    if (st != UCS_OK) {
        return st;
    }
    if (counts == nullptr || sums == nullptr || loss == nullptr || misaligned(counts, 8) ||
        misaligned(sums, 4) || misaligned(loss, 4)) {
        return invalid(what, "NULL or misaligned buffer");
    }
    if (ctx == nullptr) {
        return invalid(what, "ctx is NULL");
    }
    OnDevice dev(dev_ctx_device(ctx));
    HIP_TRY(dev.err);
    hipLaunchKernelGGL(k_balance_loss, dim3(1), dim3(kThreads), 0, stream_of(ctx), counts, sums,
                       b, loss);
    HIP_TRY(hipGetLastError());
    dev_ctx_count(ctx, 1, 0);
    return UCS_OK;
}

ucs_status_t ucg_builtin_dev_balance_grad(ucg_builtin_dev_ctx_t *ctx,
                                          const ucg_builtin_dev_balance_params_t *params,
                                          const void *logits, const uint8_t *mask,
                                          const int64_t *counts, const void *base,
                                          const float *grad_loss, void *dlogits)
{
    static const char what[] = "balance_grad";
    Balance b;
    ucs_status_t st = balance_check(params, what, &b);
    if (st != UCS_OK) {
        return st;
    }
    const size_t ts = size_of(params->dt);
    size_t bytes, out_bytes;
    if (!span(b.tokens, b.experts, b.ld, ts, &bytes) ||
        !span(b.tokens, b.experts, b.ld_out, ts, &out_bytes)) {
        return invalid(what, "tokens x row step does not fit");
    }
    if (counts == nullptr || (b.tokens != 0 && (logits == nullptr || dlogits == nullptr))) {
        return invalid(what, "NULL buffer");
    }
    if (misaligned(logits, ts) || misaligned(dlogits, ts) || misaligned(base, ts) ||
        misaligned(counts, 8) || misaligned(grad_loss, 4)) {
        return invalid(what, "misaligned buffer");
    }
    if (((dlogits != logits || b.ld != b.ld_out) && overlap(dlogits, out_bytes, logits, bytes)) ||
        (base != nullptr && dlogits != base && overlap(dlogits, out_bytes, base, out_bytes)) ||
        (mask != nullptr && overlap(dlogits, out_bytes, mask, b.tokens)) ||
        overlap(dlogits, out_bytes, counts, (b.experts + 1) * 8) ||
        (grad_loss != nullptr && overlap(dlogits, out_bytes, grad_loss, 4))) {
        return invalid(what, "dlogits overlaps an input");
    }
    if (ctx == nullptr) {
        return invalid(what, "ctx is NULL");
    }
    if (b.tokens == 0) {
        return UCS_OK;
    }
    OnDevice dev(dev_ctx_device(ctx));
    HIP_TRY(dev.err);
    hipStream_t stream = stream_of(ctx);
    with_float(params->dt, [&](auto t) {
        typedef decltype(t) T;
        with_layout<T>(b.experts, [&](auto g, auto nv) {
            constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
            const uint64_t want = div_up(b.tokens, 4 * (64 / G));
            const unsigned grid = (unsigned)(want < 2048 ? want : 2048);
            hipLaunchKernelGGL((k_balance_grad<T, G, NV>), dim3(grid), dim3(kThreads), 0, stream,
                               static_cast<const T*>(logits), mask, counts,
                               static_cast<const T*>(base), grad_loss, static_cast<T*>(dlogits),
                               b);
        });
    });
    HIP_TRY(hipGetLastError());
    dev_ctx_count(ctx, 1, 0);
    return UCS_OK;
}

/* ------------------------------------------------------------------------ */
size_t ucg_builtin_dev_policy_workspace(size_t rows, size_t cols)
{
    size_t most = 1;
    for (int v : {4, 8}) {
        Policy p;
        policy_split(cols, v, &p);
        most = p.chunks > most ? p.chunks : most;
    }
    return round16(rows * most * sizeof(PolicyPart)) + round16(kPolicyJoin * sizeof(PolicySum)) +
           16;
}

ucs_status_t ucg_builtin_dev_policy(ucg_builtin_dev_ctx_t *ctx,
                                    const ucg_builtin_dev_policy_params_t *params,
                                    const void *logp, const void *old, const void *ref,
                                    const float *adv, const uint8_t *mask, float *sums,
                                    int64_t *counts, int32_t *row_tokens, float *loss,
                                    void *workspace, size_t workspace_bytes)
{
    static const char what[] = "policy";
    Policy p;
    size_t bytes;
    ucs_status_t st = policy_check(params, what, &p, &bytes);
    if (st != UCS_OK) {
        return st;
    }
    const size_t ts = size_of(params->dt);
    if (sums == nullptr || counts == nullptr ||
        (bytes != 0 && (logp == nullptr || old == nullptr || adv == nullptr))) {
        return invalid(what, "NULL buffer");
    }
    if (misaligned(logp, ts) || misaligned(old, ts) || misaligned(ref, ts) ||
        misaligned(adv, 4) || misaligned(sums, 4) || misaligned(counts, 8) ||
        misaligned(row_tokens, 4) || misaligned(loss, 4) || misaligned(workspace, 16)) {
        return invalid(what, "misaligned buffer");
    }
    const size_t need = ucg_builtin_dev_policy_workspace(p.rows, p.cols);
    if (workspace == nullptr || workspace_bytes < need) {
        return invalid(what, "the workspace is missing or too small");
    }
    if (ctx == nullptr) {
        return invalid(what, "ctx is NULL");
    }
    PolicyPart *part = static_cast<PolicyPart*>(workspace);
    char *tail       = static_cast<char*>(workspace) + round16(p.rows * p.chunks *
                                                               sizeof(PolicyPart));
    PolicySum *block = reinterpret_cast<PolicySum*>(tail);
    unsigned *done   = reinterpret_cast<unsigned*>(tail + round16(kPolicyJoin *
                                                                  sizeof(PolicySum)));
    OnDevice dev(dev_ctx_device(ctx));
    HIP_TRY(dev.err);
    hipStream_t stream = stream_of(ctx);
    unsigned grid      = policy_grid(p);
    /* one block does a few parts by itself: a second launch costs more */
    const int single = grid <= 4 && p.rows <= (uint64_t)kThreads;
    grid = single ? 1 : grid;
    with_float(params->dt, [&](auto t) {
        typedef decltype(t) T;
        hipLaunchKernelGGL((k_policy<T>), dim3(grid), dim3(kThreads), 0, stream,
                           static_cast<const T*>(logp), static_cast<const T*>(old),
                           static_cast<const T*>(ref), adv, mask, p, part, done, single, sums,
                           counts, row_tokens, loss);
    });
    if (!single) {
        unsigned lanes = 1;
        while (lanes < 64 && lanes < p.chunks) {
            lanes *= 2;
        }
        const uint64_t want = div_up(p.rows * lanes, kThreads);
        hipLaunchKernelGGL(k_policy_join, dim3((unsigned)(want < kPolicyJoin ? want : kPolicyJoin)),
                           dim3(kThreads), 0, stream, part, block, done, p, lanes, sums, counts,
                           row_tokens, loss);
    }
    HIP_TRY(hipGetLastError());
    dev_ctx_count(ctx, single ? 1 : 2, 0);
    return UCS_OK;
}

ucs_status_t ucg_builtin_dev_policy_loss(ucg_builtin_dev_ctx_t *ctx,
                                         const ucg_builtin_dev_policy_params_t *params,
                                         const float *sums, const int64_t *counts, float *loss)
{
    static const char what[] = "policy_loss";
    Policy p;
    size_t bytes;
    ucs_status_t st = policy_check(params, what, &p, &bytes);
    if (st != UCS_OK) {
        return st;
    }
    if (sums == nullptr || counts == nullptr || loss == nullptr || misaligned(counts, 8) ||
        misaligned(sums, 4) || misaligned(loss, 4)) {
        return invalid(what, "NULL or misaligned buffer");
    }
    if (ctx == nullptr) {
        return invalid(what, "ctx is NULL");
    }
    OnDevice dev(dev_ctx_device(ctx));
    HIP_TRY(dev.err);
    hipLaunchKernelGGL(k_policy_loss, dim3(1), dim3(1), 0, stream_of(ctx), sums, counts,
                       p.per_sequence, p.kl_coef64, loss);
    HIP_TRY(hipGetLastError());
    dev_ctx_count(ctx, 1, 0);
    return UCS_OK;
}

ucs_status_t ucg_builtin_dev_policy_grad(ucg_builtin_dev_ctx_t *ctx,
                                         const ucg_builtin_dev_policy_params_t *params,
                                         const void *logp, const void *old, const void *ref,
                                         const float *adv, const uint8_t *mask,
                                         const int32_t *row_tokens, const int64_t *counts,
                                         const float *grad_loss, void *dlogp)
{
    static const char what[] = "policy_grad";
    Policy p;
    size_t bytes;
    ucs_status_t st = policy_check(params, what, &p, &bytes);
    if (st != UCS_OK) {
        return st;
    }
    const size_t ts = size_of(params->dt);
    const size_t nb = bytes / 4 * ts;
    if (counts == nullptr || (p.per_sequence && p.rows != 0 && row_tokens == nullptr) ||
        (bytes != 0 && (logp == nullptr || old == nullptr || adv == nullptr ||
                        dlogp == nullptr))) {
        return invalid(what, "NULL buffer (per_sequence needs row_tokens)");
    }
    if (misaligned(logp, ts) || misaligned(old, ts) || misaligned(ref, ts) ||
        misaligned(dlogp, ts) || misaligned(adv, 4) || misaligned(counts, 8) ||
        misaligned(row_tokens, 4) || misaligned(grad_loss, 4)) {
        return invalid(what, "misaligned buffer");
    }
    if ((dlogp != logp && overlap(dlogp, nb, logp, nb)) ||
        (dlogp != old && overlap(dlogp, nb, old, nb)) ||
        (ref != nullptr && dlogp != ref && overlap(dlogp, nb, ref, nb)) ||
        overlap(dlogp, nb, adv, p.adv_per_row ? p.rows * 4 : bytes) ||
        (mask != nullptr && overlap(dlogp, nb, mask, bytes / 4)) ||
        (row_tokens != nullptr && overlap(dlogp, nb, row_tokens, p.rows * 4)) ||
        (grad_loss != nullptr && overlap(dlogp, nb, grad_loss, 4)) ||
        overlap(dlogp, nb, counts, 24)) {
        return invalid(what, "dlogp overlaps an input");
    }
    if (ctx == nullptr) {
        return invalid(what, "ctx is NULL");
    }
    if (bytes == 0) {
        return UCS_OK;
    }
    OnDevice dev(dev_ctx_device(ctx));
    HIP_TRY(dev.err);
    with_float(params->dt, [&](auto t) {
        typedef decltype(t) T;
        hipLaunchKernelGGL((k_policy_grad<T>), dim3(policy_grid(p)), dim3(kThreads), 0,
                           stream_of(ctx), static_cast<const T*>(logp),
                           static_cast<const T*>(old), static_cast<const T*>(ref), adv, mask,
                           row_tokens, counts, grad_loss, static_cast<T*>(dlogp), p);
    });
    HIP_TRY(hipGetLastError());
    dev_ctx_count(ctx, 1, 0);
    return UCS_OK;
}

}  /* extern "C" */
