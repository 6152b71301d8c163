/*
 * dev_train.hip - the operators of a training step beside the combine
 * (ucg_builtin_dev.h): the sum of several operands with dropout in its
 * epilogue, a router's balance loss and the clipped policy loss, each with its
 * gradient. All of them stream their operands from HBM once; sums are held in
 * fp32 over at most 32 rows of a lane (one vector in the policy terms) and
 * joined in fp64 in an order that depends on the sizes alone, so a call gives
 * the same bits every time (no float atomics).
 */
#include <hip/hip_runtime.h>

#include <math.h>

#include <initializer_list>

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

template <typename T, int V, bool NT = true>
__device__ __forceinline__ void load_raw(const T *p, T (&o)[V])
{
    typedef typename Vec<T, V>::type W;
    W w;
    if constexpr (NT) {
        w = __builtin_nontemporal_load(reinterpret_cast<const W*>(p));
    } else {
        w = *reinterpret_cast<const W*>(p);
    }
    __builtin_memcpy(o, &w, sizeof(o));
}

/* elements [c, c + V) of a row of n, `fill` past its end. The values stay as
 * they were loaded: a conversion here would wait for them, and the loads that
 * a caller issues next would not be in flight together. */
template <typename T, int V>
__device__ __forceinline__ void load_row(const T *row, uint64_t c, uint64_t n, T fill, T (&o)[V])
{
    if (c + V <= n) {
        load_raw<T, V>(row + c, o);
    } else {
#pragma unroll
        for (int k = 0; k < V; k++) {
            o[k] = c + k < n ? row[c + k] : fill;
        }
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
    if constexpr (G >= 32) {          /* rows 0, 2 beside rows 1, 3 */
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x),
                                                        false, false);
        x = f(__uint_as_float(s[0]), __uint_as_float(s[1]));
    }
    if constexpr (G >= 64) {          /* the lower half beside the upper */
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x),
                                                        false, false);
        x = f(__uint_as_float(s[0]), __uint_as_float(s[1]));
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

/* sum over the block's NT threads, in every thread; lds holds NT / 64 values */
template <int NT, typename X>
__device__ __forceinline__ X block_sum(X x, X *lds)
{
    x = lanes_all(x, 1, 64, Add());
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        lds[threadIdx.x >> 6] = x;
    }
    __syncthreads();
    x = lds[0];
#pragma unroll
    for (int w = 1; w < NT / 64; w++) {
        x += lds[w];
    }
    return x;
}

/* True in every thread of the last block to arrive, with the other blocks'
 * writes visible. *done is 0 before the launch (the kernel before it on the
 * stream writes that), so nothing has to be cleared between calls. Thread 0's
 * one atomic releases what its block has written (ordered before it by the
 * barrier) to the device and acquires what the others have released; the
 * barrier after it orders the block's reads. (A fence of every thread before
 * and after it as well took 2 us more: each writes back and drops its XCD's L2.) */
__device__ __forceinline__ bool last_block(unsigned *done, unsigned *lds)
{
    __syncthreads();
    if (threadIdx.x == 0) {
        *lds = __hip_atomic_fetch_add(done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return *lds == gridDim.x - 1;
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

/* Philox-4x32-10 for counter (group, tag): eight 16-bit numbers. A round is two
 * 32 x 32 -> 64 bit products and two three-way xors (bitop3 0x96), 40
 * instructions in all for eight elements; a 32-bit number for each element
 * would take twice that and leave the bandwidth. */
__device__ __forceinline__ void philox(uint64_t group, uint64_t tag, uint64_t seed,
                                       uint32_t (&w)[4])
{
    uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32);
    uint32_t c2 = (uint32_t)tag, c3 = (uint32_t)(tag >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = __builtin_amdgcn_bitop3_b32((uint32_t)(b >> 32), c1, k0, 0x96);
        c1 = (uint32_t)b;
        c2 = __builtin_amdgcn_bitop3_b32((uint32_t)(a >> 32), c3, k1, 0x96);
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

/* the 16-bit numbers of elements [at, at + 8) of the tensor, two to a word.
 * ALIGNED: at is a multiple of 8, so they are one group. */
template <bool ALIGNED>
__device__ __forceinline__ void draw(uint64_t at, uint64_t tag, uint64_t seed, uint32_t (&o)[4])
{
    philox(at >> 3, tag, seed, o);
    if constexpr (!ALIGNED) {
        uint32_t w[4];
        philox((at >> 3) + 1, tag, seed, w);
        uint32_t x[8] = {o[0], o[1], o[2], o[3], w[0], w[1], w[2], w[3]};
        const unsigned sub = (unsigned)at & 7;
        /* shift the eight words right by sub halves; by masks, since a choice
         * between two of the array's places would put it into scratch memory */
        const uint32_t by2 = 0u - ((sub >> 2) & 1), by1 = 0u - ((sub >> 1) & 1);
#pragma unroll
        for (int k = 0; k < 6; k++) {
            x[k] ^= (x[k] ^ x[k + 2]) & by2;
        }
#pragma unroll
        for (int k = 0; k < 5; k++) {
            x[k] ^= (x[k] ^ x[k + 1]) & by1;
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            o[k] = __builtin_amdgcn_alignbit(x[k + 1], x[k], 16 * (sub & 1));
        }
    }
}

/* An even lane has computed a group of the first of two tiles, its odd neighbour
 * one of the second; both get their half (the lower, the upper) of each. */
__device__ __forceinline__ void share_groups(const uint32_t (&w)[4], bool odd, uint32_t *first,
                                             uint32_t *second)
{
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const uint32_t mine = odd ? w[2 + k] : w[k];
        const uint32_t give = odd ? w[k] : w[2 + k];
        const uint32_t got  = (uint32_t)__builtin_amdgcn_mov_dpp((int)give, 0xB1, 0xf, 0xf, true);
        first[k]  = odd ? got : mine;
        second[k] = odd ? mine : got;
    }
}

/* 16-bit number k of the words */
__device__ __forceinline__ bool kept(const uint32_t *u, int k, uint32_t threshold)
{
    return ((u[k >> 1] >> (16 * (k & 1))) & 0xffffu) >= threshold;
}

/* the sum of N values as the combine associates it */
template <int N>
__device__ __forceinline__ float sum_of(float (&v)[N])
{
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

/* elements of a wave, eight to a lane: one Philox group each */
constexpr int kWaveElems = 512;

/*
 * A wave does 512 neighbouring elements that start at a multiple of eight in
 * the whole tensor, a lane computes one group of eight numbers. With 16-bit
 * operands alone (V = 8) the group is the lane's own vector. With a 32-bit
 * operand a 16-byte vector is four elements: the wave has two tiles of 64
 * vectors, even lanes compute a group of the first tile and odd lanes one of
 * the second, and each hands its neighbour the half that it needs. (Half a
 * group used by each lane instead costs a second Philox: 234 against 216 us for
 * 16384 x 8192 bf16 with an fp32 residual.) N operands (0: nsrc of them, one by
 * one) and the residual are all in flight before the numbers are computed. A
 * block is one wave: 206 us there against 216 with four.
 *
 * HBM bounds it: 16384 x 8192 bf16 with an fp32 residual takes 206 us = 6.5 TB/s
 * (this library's plain copy reaches 6.8), four bf16 sources of 4096 x 4096 33.4
 * us = 6.0 TB/s; without the numbers (p = 0) it takes as long. Fan-ins without
 * an instantiation of their own load their second source on behind the numbers
 * and lose nothing by it (4096 x 4096 bf16: 7 sources 49.1 us = 6.1 TB/s, 8 55.7,
 * 12 77.5, 15 95.6 us). Waves whose parts begin inside a line share it with their
 * neighbours: `map` deals them to the XCDs in runs (8191 x 4097 bf16 43.3 against
 * 46.5 us; on lines the identity is faster, 16384 x 8192 bf16 126.0 against 127.9
 * us). They stay behind calls on lines (8192 x 4096 34.3 us) although HBM reads
 * only 2 % and writes 4 % more than there: each access of a wave touches a line
 * more, and the lines at its ends are written in two pieces.
 *
 * `inv` is 2^64 / cols rounded up (unused for one column): the quotient by
 * cols is its high product, or one less (the rounding adds i * e / 2^64 < 1
 * with e <= 1).
 */
template <typename T, typename R, int N>
__global__ void __launch_bounds__(64)
k_sum_dropout(R *dst, SrcList srcs, unsigned nsrc, const T *bias, const R *residual,
              uint64_t n, uint64_t first, int map, uint64_t cols, uint64_t inv, Rng rng)
{
    constexpr int V = sizeof(T) == 2 && sizeof(R) == 2 ? 8 : 4, TL = 8 / V, NN = N ? N : 1;
    const unsigned phase = (unsigned)(rng.offset % 8);
    const unsigned lane  = threadIdx.x;
    const uint64_t wave  = first + (map ? ucgdev::xcd_tile<ucgdev::kXcdChunk>(blockIdx.x, gridDim.x)
                                        : blockIdx.x);
    const int64_t  begin = (int64_t)(wave * kWaveElems) - phase;     /* the wave's first */
    if (begin >= (int64_t)n) {
        return;
    }
    const int64_t i = begin + (int64_t)lane * V;         /* of the lane's first tile */
    bool whole[TL];                   /* whether a tile's vector lies in the call */
    T x[NN][TL][V];
    R r[TL][V];
#pragma unroll
    for (int j = 0; j < TL; j++) {
        const int64_t at = i + j * 64 * V;
        whole[j] = at >= 0 && at + V <= (int64_t)n;
        if (whole[j]) {
#pragma unroll
            for (int m = 0; m < NN; m++) {
                load_raw<T, V>(static_cast<const T*>(srcs.p[m]) + at, x[m][j]);
            }
            if (residual != nullptr) {
                load_raw<R, V>(residual + at, r[j]);
            }
        }
    }

    uint32_t u[TL][V / 2] = {};
    if (rng.threshold != 0) {
        uint64_t seed, tag;
        rng_state(rng, seed, tag);
        const uint64_t group = (rng.offset - phase) / 8 + wave * (kWaveElems / 8);
        uint32_t w[4];
        if constexpr (V == 8) {
            philox(group + lane, tag, seed, w);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                u[0][k] = w[k];
            }
        } else {
            philox(group + (lane & 1 ? 32 : 0) + lane / 2, tag, seed, w);
            share_groups(w, lane & 1, u[0], u[TL - 1]);
        }
    }

#pragma unroll
    for (int j = 0; j < TL; j++) {
        const int64_t at = i + j * 64 * V;
        uint64_t col = 0;
        if (bias != nullptr) {
            const uint64_t a = at > 0 ? (uint64_t)at : 0;
            col = a - __umul64hi(a, inv) * cols;
            col = cols == 1 ? 0 : (int64_t)col < 0 ? col + cols : col;
        }
        if (whole[j]) {
            float s[V];
#pragma unroll
            for (int k = 0; k < V; k++) {
                float v[NN];
#pragma unroll
                for (int m = 0; m < NN; m++) {
                    v[m] = (float)x[m][j][k];
                }
                s[k] = sum_of<NN>(v);
            }
            if constexpr (N == 0) {
#pragma unroll 4
                for (unsigned m = 1; m < nsrc; m++) {
                    T y[V];
                    load_raw<T, V>(static_cast<const T*>(srcs.p[m]) + at, y);
#pragma unroll
                    for (int k = 0; k < V; k++) {
                        s[k] = (float)y[k] + s[k];
                    }
                }
            }
            if (bias != nullptr) {
                if (col + V <= cols) {
                    T b[V];
                    load_raw<T, V, false>(bias + col, b);  /* temporal: every row's */
#pragma unroll
                    for (int k = 0; k < V; k++) {
                        s[k] += (float)b[k];
                    }
                } else {
                    uint64_t c = col;
#pragma unroll
                    for (int k = 0; k < V; k++) {
                        s[k] += (float)bias[c];
                        c = c + 1 == cols ? 0 : c + 1;
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < V; k++) {
                const float d = kept(u[j], k, rng.threshold) ? s[k] * rng.scale : 0.f;
                s[k] = residual != nullptr ? d + (float)r[j][k] : d;
            }
            store_vec<R, V>(dst + at, s);
            continue;
        }
        for (int k = 0; k < V; k++) {
            const int64_t e = at + k;
            if (e < 0 || e >= (int64_t)n) {
                continue;
            }
            float s;
            if constexpr (N == 0) {
                s = (float)static_cast<const T*>(srcs.p[0])[e];
                for (unsigned m = 1; m < nsrc; m++) {
                    s = (float)static_cast<const T*>(srcs.p[m])[e] + s;
                }
            } else {
                float v[N];
#pragma unroll
                for (int m = 0; m < N; m++) {
                    v[m] = (float)static_cast<const T*>(srcs.p[m])[e];
                }
                s = sum_of<N>(v);
            }
            if (bias != nullptr) {
                s += (float)bias[col];
                col = col + 1 == cols ? 0 : col + 1;
            }
            const float d = kept(u[j], k, rng.threshold) ? s * rng.scale : 0.f;
            dst[e] = (R)(residual != nullptr ? d + (float)residual[e] : d);
        }
    }
}

/*
 * The gradient with the bias' part: a lane keeps eight columns over the rows of
 * its chunk, tx lanes side by side and kThreads / tx rows at once, four rows in
 * flight, and the block's rows are joined in LDS. With 16-bit types the eight
 * are neighbours. A 32-bit operand would take two loads 32 bytes apart in each
 * lane for that, so its lanes have four columns in each of two tiles and share
 * groups as in k_sum_dropout (SPLIT). A row may start anywhere in a group of
 * eight (ALIGNED 0: the columns or the offset are no multiple of eight): then
 * the eight are neighbours whose numbers come from two groups.
 *
 * Sums: a lane's rows in 32 bits, at most kFewRows of them; with more (DEEP) the
 * four of a pass, and passes in 64, for which it needs 12 registers more (8191 x
 * 4097 bf16, 18 rows a lane, 40.9 us without and 41.7 with it; 2^20 x 64 bf16, 128
 * rows, 68.0 and 69.0). Lanes of a column are joined in 64 bits, a part is
 * rounded to 32 (half the join's bytes: 8192 x 4096 bf16 27.7 us, 28.1 in 64),
 * parts are joined in 64.
 *
 * 8192 x 4096 bf16 takes 24.6 us = 5.5 TB/s, and 4.8 for the join of 128 parts
 * (less than half of a launch is its bytes); fp32 54 us with it = 5.0 TB/s. With
 * rows in chunks of neighbours instead of dealt to the parts fp32 took 63, with
 * the eight fp32 columns side by side 74 us. 8191 x 4097 bf16 takes 41 us: twice
 * the Philox rounds, and a block column of one column.
 */
constexpr unsigned kFewRows = 32;

template <typename R, typename T, bool ALIGNED, bool DEEP>
__global__ void __launch_bounds__(kThreads)
k_dropout_grad(T *dsrc, const R *grad, float *dbias, uint64_t rows, uint64_t cols,
               unsigned tx, Rng rng)
{
    constexpr bool SPLIT = ALIGNED && (sizeof(R) == 4 || sizeof(T) == 4);
    constexpr int U = 4, TL = SPLIT ? 2 : 1, V = 8 / TL;
    typedef typename std::conditional<DEEP, double, float>::type S;
    __shared__ S lds[kThreads * 8];
    const unsigned x  = threadIdx.x % tx, y = threadIdx.x / tx, ty = kThreads / tx;
    const uint64_t c0 = (uint64_t)blockIdx.x * tx * 8;          /* the block's first column */
    const uint64_t c  = c0 + x * V, tile = (uint64_t)tx * V;
    /* part b of P takes rows b * ty + y, then P * ty further on: at any time the
     * parts read neighbouring rows, and not rows a power of two apart */
    const uint64_t step = (uint64_t)gridDim.y * ty;
    uint64_t seed, tag;
    rng_state(rng, seed, tag);
    S sum[8] = {};
    bool has[TL];                     /* whether a tile's vector lies in the row */
#pragma unroll
    for (int j = 0; j < TL; j++) {
        has[j] = c + j * tile + V <= cols;
    }
    /* SPLIT: cols is a multiple of eight, so a lane and its neighbour are both
     * in or both out; the lanes of a row take part as long as one tile does */
    if (has[0]) {
        for (uint64_t row = (uint64_t)blockIdx.y * ty + y; row < rows; row += U * step) {
            R g[U][TL][V];
#pragma unroll
            for (int j = 0; j < U; j++) {
                const uint64_t q = row + j * step;
#pragma unroll
                for (int h = 0; h < TL; h++) {
                    load_raw<R, V>(grad + (q < rows ? q : row) * cols + c + (has[h] ? h * tile : 0),
                                   g[j][h]);
                }
            }
            float few[8];             /* the sums that these rows go on with */
#pragma unroll
            for (int k = 0; k < 8; k++) {
                few[k] = DEEP ? 0.f : (float)sum[k];
            }
#pragma unroll
            for (int j = 0; j < U; j++) {
                const uint64_t q = row + j * step;
                if (q < rows) {
                    uint32_t u[8 / 2] = {};
                    const uint64_t at = rng.offset + q * cols;
                    if (rng.threshold != 0) {
                        if constexpr (SPLIT) {
                            uint32_t w[4];
                            philox((at + c0 + (x & 1 ? tile : 0)) / 8 + x / 2, tag, seed, w);
                            share_groups(w, x & 1, u, u + 2);
                        } else {
                            draw<ALIGNED>(at + c, tag, seed, u);
                        }
                    }
#pragma unroll
                    for (int h = 0; h < TL; h++) {
                        float d[V];
#pragma unroll
                        for (int k = 0; k < V; k++) {
                            d[k] = kept(u, h * V + k, rng.threshold)
                                       ? (float)g[j][h][k] * rng.scale : 0.f;
                            few[h * V + k] += d[k];
                        }
                        if (has[h]) {
                            store_vec<T, V>(dsrc + q * cols + c + h * tile, d);
                        }
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < 8; k++) {
                sum[k] = DEEP ? sum[k] + (S)few[k] : (S)few[k];
            }
        }
    } else if (!SPLIT && c < cols) {  /* the row's last columns, fewer than eight: a lane,
                                       * which has the next row's on the way */
        const R *from = grad + ((uint64_t)blockIdx.y * ty + y) * cols;
        R g[8];
        if ((uint64_t)blockIdx.y * ty + y < rows) {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                g[k] = from[c + k < cols ? c + k : cols - 1];
            }
        }
        for (uint64_t q = (uint64_t)blockIdx.y * ty + y; q < rows; q += step) {
            R next[8];
            from = grad + (q + step < rows ? q + step : q) * cols;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                next[k] = from[c + k < cols ? c + k : cols - 1];
            }
            uint32_t u[4] = {};
            if (rng.threshold != 0) {
                draw<ALIGNED>(rng.offset + q * cols + c, tag, seed, u);
            }
            float d[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                d[k] = kept(u, k, rng.threshold) ? (float)g[k] * rng.scale : 0.f;
                sum[k] += (S)d[k];        /* what is past the row is not written */
            }
            store_row<T, 8>(dsrc + q * cols, c, cols, d);
            __builtin_memcpy(g, next, sizeof(g));
        }
    }
#pragma unroll
    for (int k = 0; k < 8; k++) {
        lds[y * tx * 8 + (k / V) * tile + x * V + k % V] = sum[k];
    }
    __syncthreads();
    /* column j of the block's tx * 8: its rows y = 0, 1, .. in order */
    for (unsigned j = threadIdx.x; j < tx * 8; j += kThreads) {
        if (c0 + j < cols) {
            double s = 0;
            for (unsigned q = 0; q < ty; q++) {
                s += (double)lds[q * tx * 8 + j];
            }
            dbias[(uint64_t)blockIdx.y * cols + c0 + j] = (float)s;
        }
    }
}

constexpr unsigned kMaxParts = 256;    /* partials to join */

/* 16 columns by 16 parts of the partials' rows (at most kMaxParts of them, so
 * that a lane's loads are all in flight at once); the sum in every thread of
 * the column */
template <typename X, typename S>
__device__ __forceinline__ S join_columns(const X *part, unsigned nparts, uint64_t stride,
                                          uint64_t col, uint64_t cols, S *lds)
{
    const unsigned x = threadIdx.x & 15, y = threadIdx.x >> 4;
    const X *at = part + (col < cols ? col : cols - 1);
    X v[kMaxParts / 16];
#pragma unroll
    for (unsigned j = 0; j < kMaxParts / 16; j++) {
        const unsigned p = y + j * 16;
        v[j] = at[(p < nparts ? p : nparts - 1) * stride];
    }
    S s = 0;
#pragma unroll
    for (unsigned j = 0; j < kMaxParts / 16; j++) {
        s += y + j * 16 < nparts ? (S)v[j] : (S)0;
    }
    __syncthreads();
    lds[threadIdx.x] = s;
    __syncthreads();
    S t = 0;
#pragma unroll
    for (unsigned q = 0; q < 16; q++) {
        t += lds[q * 16 + x];
    }
    return t;
}

__global__ void __launch_bounds__(kThreads)
k_join_bias(float *dbias, const float *part, unsigned nparts, uint64_t cols)
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

/* the loss' three values from whole counts and sums, by one block of NT */
template <int NT>
__device__ __forceinline__ void balance_loss_block(const int64_t *counts, const float *sums,
                                                   unsigned experts, double balance,
                                                   double z_coef, float *loss, double *lds)
{
    double dot = 0;
    for (unsigned e = threadIdx.x; e < experts; e += NT) {
        dot += (double)counts[e] * (double)sums[e];
    }
    dot = block_sum<NT>(dot, lds);
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

/* columns [c, c + V) of a row of E logits, -inf past its end. EVEN: E is a
 * multiple of V, so that a lane has a whole vector or none. Temporal: a row
 * seldom fills its lines, and its neighbours are other waves' (32768 x 384 fp32
 * statistics 19.9 us, non-temporal 20.8). */
template <typename T, int V, bool EVEN>
__device__ __forceinline__ void load_logits(const T *row, unsigned c, unsigned E, T (&o)[V])
{
    if constexpr (EVEN) {
#pragma unroll
        for (int k = 0; k < V; k++) {
            o[k] = (T)-INFINITY;
        }
        if (c < E) {
            load_raw<T, V, false>(row + c, o);
        }
    } else {
        load_row<T, V>(row, c, E, (T)-INFINITY, o);
    }
}

/* rows of a lane group in flight at once. More (4), and the next rows loaded
 * while these are computed, gained nothing: sixteen waves fill the time. */
template <int NV>
constexpr int rows_at_once()
{
    return NV == 1 ? 2 : 1;
}

constexpr int kBalanceThreads = 1024;  /* 16 waves: one block to a CU */

/* A row lies in G lanes, V neighbouring columns to a lane and vector, so a
 * wave has 64 / G rows at once, U such sets in flight, and a lane keeps the sums
 * of its columns over all rows of the block. A masked row is loaded like the
 * others (the mask is not waited for) and left out afterwards. Counts are
 * integers, so their LDS atomics give the same in any order.
 *
 * Sums: a lane adds up to kFewRows rows in 32 bits; with more (DEEP) it puts
 * them away in 64 and goes on (2^20 tokens of 256 experts, 128 rows a lane, 140.4
 * us without and 142.0 with it; the code alone costs short calls 0.2 us, so they
 * have a kernel without). The rows of a wave and a pair of waves are joined in
 * 32 bits, all else in 64; a block's part is rounded to 32, as the sums are that
 * the group adds up, and the loss is taken from those.
 *
 * 65536 x 256 bf16, top 8: 13.3 us, and 4.8 with the loss for the join. Without the
 * softmax 3.9 less: the exponentials and sums of 16 M probabilities do not hide
 * behind 38 MB here, and 256 blocks start and end together. 512 of them take longer for
 * the join than they save (18.1 against 17.3 us in all). */
template <typename T, typename I, int G, int NV, bool EVEN, bool DEEP>
__global__ void __launch_bounds__(kBalanceThreads)
k_balance(const T *logits, const I *index, const uint8_t *mask, Balance p, BalancePart out,
          int64_t *counts, float *sums, float *loss)
{
    constexpr int V = 16 / sizeof(T), C = NV * V, R = 64 / G, U = rows_at_once<NV>();
    constexpr int W = kBalanceThreads / 64;
    __shared__ float psum[W / 2][G * C + 1];
    __shared__ unsigned hist[G * C + 1];
    __shared__ double join[W];
    const unsigned E    = p.experts;
    const unsigned wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const unsigned l    = lane % G, sub = lane / G;
    const uint64_t r0 = (uint64_t)blockIdx.x * p.chunk;
    const uint64_t r1 = r0 + p.chunk < p.tokens ? r0 + p.chunk : p.tokens;
    T raw[U][NV][V];
    uint8_t on[U];
    I named[U];
    const auto load = [&](uint64_t t) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint64_t q = t + (uint64_t)u * W * R;
            const uint64_t r = q < r1 ? q : r1 - 1;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                load_logits<T, V, EVEN>(logits + r * p.ld, (j * G + l) * V, E, raw[u][j]);
            }
            on[u]    = mask != nullptr ? mask[r] : 1;
            named[u] = l < p.topk ? index[r * p.ld_index + l] : (I)-1;
        }
    };
    const uint64_t t0 = r0 + wave * R + sub;
    if (t0 < r1) {
        load(t0);                     /* in flight while the counts are cleared */
    }
    for (unsigned e = threadIdx.x; e <= G * C; e += kBalanceThreads) {
        hist[e] = 0;
    }
    __syncthreads();
    float acc[C] = {}, zsum = 0.f;
    double far[DEEP ? C : 1] = {}, zfar = 0;   /* of the rows before these */
    unsigned live_rows = 0, held = 0;
    for (uint64_t t = t0; t < r1; t += (uint64_t)U * W * R) {
        if (t != t0) {
            load(t);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint64_t q = t + (uint64_t)u * W * R;
            if (q >= r1 || on[u] == 0) {      /* the same for a row's G lanes */
                continue;
            }
            if ((int64_t)named[u] >= 0 && (int64_t)named[u] < (int64_t)E) {
                atomicAdd(&hist[named[u]], 1u);
            }
            for (unsigned k0 = l + G; k0 < p.topk; k0 += 4 * G) {
                I more[4];
#pragma unroll
                for (unsigned i = 0; i < 4; i++) {
                    const unsigned k = k0 + i * G;
                    more[i] = index[q * p.ld_index + (k < p.topk ? k : k0)];
                }
#pragma unroll
                for (unsigned i = 0; i < 4; i++) {
                    const int64_t e = (int64_t)more[i];
                    if (k0 + i * G < p.topk && e >= 0 && e < (int64_t)E) {
                        atomicAdd(&hist[e], 1u);
                    }
                }
            }
            float x[C], inv, lse;
#pragma unroll
            for (int k = 0; k < C; k++) {
                x[k] = (float)raw[u][k / V][k % V];
            }
            row_softmax<G, C>(x, inv, lse);
#pragma unroll
            for (int k = 0; k < C; k++) {
                acc[k] = __builtin_fmaf(x[k], inv, acc[k]);
            }
            zsum = __builtin_fmaf(lse, lse, zsum);
            live_rows++;
        }
        if constexpr (DEEP) {
            held += U;
            if (held == kFewRows) {
#pragma unroll
                for (int k = 0; k < C; k++) {
                    far[k] += (double)acc[k];
                    acc[k] = 0.f;
                }
                zfar += (double)zsum;
                zsum = 0.f;
                held = 0;
            }
        }
    }
    if constexpr (DEEP) {
#pragma unroll
        for (int k = 0; k < C; k++) {
            acc[k] = (float)(far[k] + (double)acc[k]);
        }
        zsum = (float)(zfar + (double)zsum);
    }
    /* rows of the wave, then waves, in a fixed order */
#pragma unroll
    for (int k = 0; k < C; k++) {
        acc[k] = lanes_all(acc[k], G, 64, Add());
    }
    zsum      = lanes_all(zsum, G, 64, Add());
    live_rows = lanes_all(live_rows, G, 64, Add());
    /* the upper half of the waves hands its sums to the lower: half the LDS */
    for (int half = 1; half >= 0; half--) {
        if ((int)(wave / (W / 2)) == half && sub == 0) {
            float *to = psum[wave % (W / 2)];
#pragma unroll
            for (int k = 0; k < C; k++) {
                const unsigned at = ((k / V) * G + l) * V + k % V;
                to[at] = half ? acc[k] : to[at] + acc[k];
            }
            if (l == 0) {
                to[G * C] = half ? zsum : to[G * C] + zsum;
                atomicAdd(&hist[G * C], live_rows);
            }
        }
        __syncthreads();
    }
    for (unsigned e = threadIdx.x; e <= E; e += kBalanceThreads) {
        const unsigned at = e == E ? G * C : e;
        double s = 0;
#pragma unroll
        for (int w = 0; w < W / 2; w++) {
            s += (double)psum[w][at];
        }
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
            balance_loss_block<kBalanceThreads>(counts, sums, E, p.balance, p.z_coef, loss, join);
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
        balance_loss_block<kThreads>(counts, sums, p.experts, p.balance, p.z_coef, loss, lds);
    }
}

__global__ void __launch_bounds__(kThreads)
k_balance_loss(const int64_t *counts, const float *sums, Balance p, float *loss)
{
    __shared__ double lds[4];
    balance_loss_block<kThreads>(counts, sums, p.experts, p.balance, p.z_coef, loss, lds);
}

/* dx_e = grad * p_e ( a (c_e - sum_j p_j c_j) + 2 b lse ), a = balance / N^2,
 * b = z_coef / N. The counts enter less one of them, which the p (that sum to
 * one) cancel: near balance that keeps the digits that the difference needs,
 * also where choices that name no expert leave all counts far below
 * N topk / experts. It is the middle one of three, so that one expert that is
 * much liked does not set it (their mean, summed in 64 bits over the block, took
 * 0.7 us, in fp32 over a row's lanes 0.2 to 0.5).
 * 49999 x 160 bf16 with a base takes 11.8 us a pass = 4.1 TB/s: the exchanges of
 * each row (a maximum and two sums, five steps each over 32 lanes, of which this
 * layout gives columns to 20) wait for one another, and a wave has two rows in
 * flight beside them (1536 and 2048 blocks, and one row in flight, took longer). */
template <typename T, int G, int NV, bool EVEN>
__global__ void __launch_bounds__(kThreads)
k_balance_grad(const T *logits, const uint8_t *mask, const int64_t *counts, const T *base,
               const float *grad_loss, T *dlogits, Balance p)
{
    constexpr int V = 16 / sizeof(T), C = NV * V, R = 64 / G, U = NV == 1 ? 2 : 1;
    __shared__ float table[G * C];
    const unsigned E    = p.experts;
    const unsigned wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const unsigned l    = lane % G, sub = lane / G;
    const uint64_t step = (uint64_t)gridDim.x * 4 * R;
    struct Set {
        T       raw[U][NV][V], add[U][NV][V];
        uint8_t on[U];
    };
    const auto load = [&](uint64_t t, Set &s) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint64_t q = t + u * step;
            const uint64_t r = q < p.tokens ? q : p.tokens - 1;
#pragma unroll
            for (int j = 0; j < NV; j++) {
                const unsigned c = (j * G + l) * V;
                load_logits<T, V, EVEN>(logits + r * p.ld, c, E, s.raw[u][j]);
                if (base != nullptr) {
                    load_logits<T, V, EVEN>(base + r * p.ld_out, c, E, s.add[u][j]);
                } else {
#pragma unroll
                    for (int k = 0; k < V; k++) {
                        s.add[u][j][k] = (T)0.f;
                    }
                }
            }
            s.on[u] = mask != nullptr ? mask[r] : 1;
        }
    };
    const uint64_t t0 = ((uint64_t)blockIdx.x * 4 + wave) * R + sub;
    Set now;
    if (t0 < p.tokens) {
        load(t0, now);
    }
    /* what a block needs of the counts, once */
    const int64_t tokens = counts[E];
    const int64_t c0 = counts[0], c1 = counts[E / 2], c2 = counts[E - 1];
    const int64_t lo = c0 < c1 ? c0 : c1, hi = c0 < c1 ? c1 : c0;
    const int64_t centre = c2 < lo ? lo : c2 > hi ? hi : c2;
    for (unsigned e = threadIdx.x; e < G * C; e += kThreads) {
        table[e] = e < E ? (float)(counts[e] - centre) : 0.f;
    }
    const double g = grad_loss != nullptr ? (double)*grad_loss : 1.0;
    const float a = tokens > 0 ? (float)(g * p.balance / ((double)tokens * (double)tokens)) : 0.f;
    const float b = tokens > 0 ? (float)(g * 2 * p.z_coef / (double)tokens) : 0.f;
    __syncthreads();
    float c[C];
#pragma unroll
    for (int k = 0; k < C; k++) {
        c[k] = table[((k / V) * G + l) * V + k % V];
    }
    for (uint64_t t = t0; t < p.tokens; t += U * step) {
        Set next;
        if (t + U * step < p.tokens) {
            load(t + U * step, next);
        }
        const auto &raw = now.raw;
        const auto &add = now.add;
        const auto &on = now.on;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint64_t q = t + u * step;
            if (q >= p.tokens) {              /* the same for a row's G lanes */
                continue;
            }
            float x[C], inv, lse;
#pragma unroll
            for (int k = 0; k < C; k++) {
                x[k] = (float)raw[u][k / V][k % V];
            }
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
            for (int j = 0; j < NV; j++) {
                float d[V];
#pragma unroll
                for (int k = 0; k < V; k++) {
                    const float w = (float)add[u][j][k];
                    const float s = __builtin_fmaf(
                        x[j * V + k], __builtin_fmaf(a, c[j * V + k] - dot, z), w);
                    d[k] = on[u] != 0 ? s : w;        /* whatever a masked row holds */
                }
                const unsigned at = (j * G + l) * V;
                if (at < E) {
                    if constexpr (EVEN) {
                        store_vec<T, V>(dlogits + q * p.ld_out + at, d);
                    } else {
                        store_row<T, V>(dlogits + q * p.ld_out, at, E, d);
                    }
                }
            }
        }
        now = next;
    }
}

/* ======================================================================== */
/* policy loss                                                              */
/* ======================================================================== */
struct Policy {
    uint64_t rows, cols, ld;
    int      per_sequence;
    unsigned lanes_log;          /* log2 of the lanes that share a row */
    unsigned steps;              /* vectors of a lane */
    uint64_t chunks;             /* parts of a row */
    uint64_t whole;              /* columns in whole vectors */
    uint64_t tail_chunk;         /* whose lane tail_lane has the others, if any */
    unsigned tail_lane;
    float    up, down;           /* log(1 + clip_high), log(1 - clip_low) */
    float    ratio_up, ratio_down;
    float    kl_coef;
    double   kl_coef64;
};

struct PolicyPart {              /* of one part of a row */
    double   pg, kl;
    unsigned tokens, cut;
};

struct PolicySum {
    double             pg, kl;
    unsigned long long tokens, rows, cut;

    __device__ __forceinline__ void add(const PolicySum &o)
    {
        pg += o.pg;
        kl += o.kl;
        tokens += o.tokens;
        rows += o.rows;
        cut += o.cut;
    }
    /* over `lanes` neighbouring lanes: the five values step by step together,
     * so that their exchanges overlap */
    __device__ __forceinline__ void add_lanes(unsigned lanes)
    {
        for (unsigned o = 1; o < lanes; o <<= 1) {
            const PolicySum x = {__shfl_xor(pg, o, 64), __shfl_xor(kl, o, 64),
                                 __shfl_xor(tokens, o, 64), __shfl_xor(rows, o, 64),
                                 __shfl_xor(cut, o, 64)};
            add(x);
        }
    }
};

/* By the hardware's base-2 exponential (1 ulp), of the rounded product: (1.25 |x|
 * + 2) u of the result, u = 2^-24. A ratio between 1/e and e is off by 3.3 u at
 * most, one of e^20 by 27 u. The product in two parts (2 u for any x) is a choice
 * not made: four to six instructions more for each exponential took 0.1-0.3 us of
 * 27 on 1024 x 8192 fp32 terms, 1.0 of 25.4 on their gradient and 1.9 of 21.3 on
 * 512 x 16384 bf16 terms, for digits of ratios that the clip replaces or that
 * carry no weight. */
__device__ __forceinline__ float exp_of(float x)
{
    return __builtin_amdgcn_exp2f(x * kLog2e);
}

/* (exp(q) - q - 1) / q^2 by its series, for |q| < 1.25, where the subtractions
 * would leave too little (to q^10 / 12!: the rest is below 6e-9 of it there) */
constexpr float kSeries = 1.25f;

__device__ __forceinline__ float exp_series(float q)
{
    float s = 1.f / 479001600.f;
    s = __builtin_fmaf(s, q, 1.f / 39916800.f);
    s = __builtin_fmaf(s, q, 1.f / 3628800.f);
    s = __builtin_fmaf(s, q, 1.f / 362880.f);
    s = __builtin_fmaf(s, q, 1.f / 40320.f);
    s = __builtin_fmaf(s, q, 1.f / 5040.f);
    s = __builtin_fmaf(s, q, 1.f / 720.f);
    s = __builtin_fmaf(s, q, 1.f / 120.f);
    s = __builtin_fmaf(s, q, 1.f / 24.f);
    s = __builtin_fmaf(s, q, 1.f / 6.f);
    return __builtin_fmaf(s, q, 0.5f);
}

constexpr float kExpEnd = 88.f;        /* its exponential is finite */

/* exp(q) - q - 1; both forms are computed: no branch around either */
__device__ __forceinline__ float exp_less(float q)
{
    float s = exp_series(q) * q * q, e = exp_of(q) - q - 1.f;
    asm("" : "+v"(s), "+v"(e));
    return fabsf(q) < kSeries ? s : e;
}

/* exp(q) - 1, to the end of its range (a reference of -inf or of the type's
 * lowest value gives -1) */
__device__ __forceinline__ float exp_minus(float q)
{
    float s = __builtin_fmaf(exp_series(q) * q, q, q), e = exp_of(q) - 1.f;
    asm("" : "+v"(s), "+v"(e));
    return fabsf(q) < kSeries ? s : e;
}

/* What an advantage makes of its tokens: d with A's sign is compared with
 * `limit` (a token is cut goes by d itself, not by its rounded exponential),
 * `cap` is the ratio of a cut token and `count` what it adds to the counts.
 * A = 0 cuts none; its limit keeps ratios that are infinite in 32 bits from
 * its product, which is 0 for any d. */
struct Advantage {
    float    a, limit, cap;
    unsigned count;

    __device__ __forceinline__ Advantage() = default;
    __device__ __forceinline__ Advantage(float x, const Policy &p)
    {
        a     = x + 0.f;              /* -0 as 0 */
        limit = x > 0.f ? p.up : x < 0.f ? -p.down : kExpEnd;
        cap   = x > 0.f ? p.ratio_up : p.ratio_down;
        count = x > 0.f || x < 0.f ? 0x10000u : 0u;
    }
    __device__ __forceinline__ bool cuts(float d) const
    {
        return __uint_as_float(__float_as_uint(d) ^ (__float_as_uint(a) & 0x80000000u)) > limit;
    }
};

/* V neighbouring tokens of a row as they were loaded: converting them would
 * wait for them, and the next loads would not be in flight together */
template <typename T, int V>
struct Tokens {
    T       logp[V], old[V], ref[V];
    float   adv[V];
    uint8_t live[V];
};

/* what a call has of its rows: REF a reference, ROW an advantage for each row
 * (known at compile time, since the branches would be in every token). LINES:
 * rows start on 128-byte lines, and nothing is read twice; elsewhere the lines
 * at the ends of the waves' parts are, and temporal loads find them (513 x 12345
 * bf16 gradient 16.8 against 19.3 us; 1024 x 8192 fp32, on lines, 26.6 against
 * 25.5 us). */
template <typename T, bool REF, bool ROW, bool LINES>
struct PolicyIn {
    const T       *logp, *old, *ref;
    const float   *adv;
    const uint8_t *mask;

    template <int V>
    __device__ __forceinline__ void load(uint64_t at, Tokens<T, V> &t) const
    {
        load_raw<T, V, LINES>(logp + at, t.logp);
        load_raw<T, V, LINES>(old + at, t.old);
        if constexpr (REF) {
            load_raw<T, V, LINES>(ref + at, t.ref);
        }
        if constexpr (!ROW) {
            load_raw<float, V, LINES>(adv + at, t.adv);
        }
        if (mask != nullptr) {
            load_raw<uint8_t, V, LINES>(mask + at, t.live);
        } else {
            __builtin_memset(t.live, 1, V);
        }
    }

    /* one token, for the end of a row that is no whole vector */
    __device__ __forceinline__ void load_one(uint64_t at, Tokens<T, 1> &t) const
    {
        t.logp[0] = logp[at];
        t.old[0]  = old[at];
        t.ref[0]  = REF ? ref[at] : logp[at];
        t.adv[0]  = ROW ? 0.f : adv[at];
        t.live[0] = mask != nullptr ? mask[at] : 1;
    }
};

/* vectors of a lane in flight at once: 16 tokens */
template <typename T>
constexpr int policy_steps()
{
    return (int)sizeof(T);
}

/* Which part of which rows a wave does: the waves of a block lie side by side
 * along a row's parts as far as it has them (wc = 1, 2, 4 .. of them), then
 * along the rows; no division. */
template <int W>
struct PolicyWave {
    unsigned l, per, wc_log;
    uint64_t row_tile, chunk, tile_step, chunk_step;

    __device__ __forceinline__ PolicyWave(const Policy &p)
    {
        const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        l      = lane & ((1u << p.lanes_log) - 1);
        per    = 64u >> p.lanes_log;
        wc_log = 0;
        while ((1u << wc_log) < W && (1u << wc_log) < p.chunks) {
            wc_log++;
        }
        row_tile   = ((uint64_t)blockIdx.x * (W >> wc_log)) + (wave >> wc_log);
        chunk      = ((uint64_t)blockIdx.y << wc_log) + (wave & ((1u << wc_log) - 1));
        tile_step  = (uint64_t)gridDim.x * (W >> wc_log);
        chunk_step = (uint64_t)gridDim.y << wc_log;
    }
    __device__ __forceinline__ uint64_t row(uint64_t tile, const Policy &p) const
    {
        return tile * per + ((threadIdx.x & 63) >> p.lanes_log);
    }
};

/* The sums of a lane over its tokens: those of a vector in 32 bits, of vectors,
 * lanes and parts in 64, since rows of opposite advantages cancel (in 32 the sum
 * was 2.7 times as far off over 85 batches; it costs 0.6 us of 27 for 1024 x 8192
 * fp32). The counts of a wave's part (at most 1024 tokens) share a word. */
struct PolicyAcc {
    double   pg = 0, kl = 0;
    unsigned n = 0;              /* tokens, and cut ones from bit 16 on */

    __device__ __forceinline__ void add_lanes(unsigned lanes)
    {
        for (unsigned o = 1; o < lanes; o <<= 1) {
            const double a = __shfl_xor(pg, o, 64), b = __shfl_xor(kl, o, 64);
            const unsigned c = __shfl_xor(n, o, 64);
            pg += a;
            kl += b;
            n += c;
        }
    }

    template <bool REF, bool ROW, typename T, int V>
    __device__ __forceinline__ void add(const Tokens<T, V> &t, const Advantage &row,
                                        const Policy &p)
    {
        float vpg = 0.f, vkl = 0.f;
#pragma unroll
        for (int k = 0; k < V; k++) {
            const Advantage w = ROW ? row : Advantage(t.adv[k], p);
            const float x = (float)t.logp[k], d = x - (float)t.old[k];
            const bool on = t.live[k] != 0, is = w.cuts(d);
            float r = exp_of(d);
            asm("" : "+v"(r));
            r = (is ? w.cap : r) * -w.a;
            vpg += on ? r : 0.f;
            n += on;
            n += (on & is) ? w.count : 0u;
            if constexpr (REF) {
                float e = exp_less((float)t.ref[k] - x);
                asm("" : "+v"(e));
                vkl += on ? e : 0.f;
            }
        }
        pg += (double)vpg;
        kl += (double)vkl;
    }
};

/* The join of a row's parts by `lanes` lanes, eight parts of each in flight at
 * once, and the thread's sum over its rows; block b of the grid takes rows
 * b * NT / lanes, .. */
template <int NT>
__device__ __forceinline__ PolicySum policy_rows(const PolicyPart *part, const Policy &p,
                                                 int32_t *row_tokens, unsigned lanes)
{
    constexpr int U = 8;
    PolicySum sum = {};
    const unsigned l = threadIdx.x % lanes, per = NT / lanes;
    for (uint64_t r = (uint64_t)blockIdx.x * per + threadIdx.x / lanes; r < p.rows;
         r += (uint64_t)gridDim.x * per) {
        PolicySum one = {};
        for (uint64_t w = l; w < p.chunks; w += (uint64_t)U * lanes) {
            PolicyPart x[U];
#pragma unroll
            for (int j = 0; j < U; j++) {
                const uint64_t q = w + (uint64_t)j * lanes;
                x[j] = part[r * p.chunks + (q < p.chunks ? q : w)];
            }
#pragma unroll
            for (int j = 0; j < U; j++) {
                if (w + (uint64_t)j * lanes < p.chunks) {
                    one.add({x[j].pg, x[j].kl, x[j].tokens, 0, x[j].cut});
                }
            }
        }
        one.add_lanes(lanes);
        if (l == 0) {
            if (p.per_sequence && one.tokens != 0) {
                one.pg /= (double)one.tokens;
                one.kl /= (double)one.tokens;
            }
            one.rows = one.tokens != 0;
            sum.add(one);
            if (row_tokens != nullptr) {
                row_tokens[r] = (int32_t)one.tokens;
            }
        }
    }
    return sum;
}

/* over the block's threads; lds holds NT / 64 of them */
template <int NT>
__device__ __forceinline__ PolicySum policy_block(PolicySum s, PolicySum *lds)
{
    s.add_lanes(64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        lds[threadIdx.x >> 6] = s;
    }
    __syncthreads();
    s = lds[0];
#pragma unroll
    for (int w = 1; w < NT / 64; w++) {
        s.add(lds[w]);
    }
    return s;
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

/* 1024 x 8192 fp32 with a reference takes 20.7 us = 5.3 TB/s and 6.4 for the join
 * of 8192 parts: 37 vector instructions a token, two exponentials among them, leave
 * HBM about the bound. Twice the tokens in flight took 29.2 us in all against
 * 27.5, half of them as long as these.
 *
 * A wave does one part of 64 / lanes rows at a time: `steps` vectors of each
 * of the lanes that share the row, all in flight at once. The tokens behind the
 * last whole vector are one lane's, one after the other: 2048 rows of 1023 bf16
 * take 14.3 us in all where 1024 take 11.9, of 7 9.4 where 8 take 8.0. NT =
 * kSingle: the only block, which has the parts in LDS and joins them too. */
constexpr int kSingle      = 512;
constexpr int kSingleParts = 1024;

template <typename T, bool REF, bool ROW, bool LINES, int NT>
__global__ void __launch_bounds__(NT)
k_policy(PolicyIn<T, REF, ROW, LINES> in, Policy p, PolicyPart *part, unsigned *done,
         float *sums, int64_t *counts, int32_t *row_tokens, float *loss)
{
    constexpr int V = 16 / sizeof(T), S = policy_steps<T>(), W = NT / 64;
    constexpr bool single = NT == kSingle;
    __shared__ PolicySum lds[W];
    __shared__ PolicyPart own[single ? kSingleParts : 1];
    if constexpr (single) {
        part = own;
    }
    const PolicyWave<W> w(p);
    const unsigned lanes = 1u << p.lanes_log, l = w.l, cs = lanes * V;
    for (uint64_t tile = w.row_tile; tile * w.per < p.rows; tile += w.tile_step)
    for (uint64_t chunk = w.chunk; chunk < p.chunks; chunk += w.chunk_step) {
        const uint64_t row   = w.row(tile, p);
        const uint64_t c0    = chunk * p.steps * cs + l * V;
        const uint64_t end   = row < p.rows ? p.whole : 0;
        const uint64_t at    = row * p.ld + c0;
        Tokens<T, V> t[S];
        Advantage a;
        a.a = row < p.rows && ROW ? in.adv[row] : 0.f;
#pragma unroll
        for (unsigned j = 0; j < S; j++) {
            if (j < p.steps && c0 + j * cs < end) {
                in.load(at + j * cs, t[j]);
            }
        }
        a = Advantage(a.a, p);
        PolicyAcc acc;
#pragma unroll
        for (unsigned j = 0; j < S; j++) {
            if (j < p.steps && c0 + j * cs < end) {
                acc.template add<REF, ROW>(t[j], a, p);
            }
        }
        /* the rest of the row, by the lane whose turn it would be */
        if (row < p.rows && chunk == p.tail_chunk && l == p.tail_lane) {
#pragma unroll 1
            for (uint64_t c = p.whole; c < p.cols; c++) {
                Tokens<T, 1> one;
                in.load_one(row * p.ld + c, one);
                acc.template add<REF, ROW>(one, a, p);
            }
        }
        acc.add_lanes(lanes);
        if (l == 0 && row < p.rows) {
            part[row * p.chunks + chunk] = {acc.pg, acc.kl, acc.n & 0xffff, acc.n >> 16};
        }
    }
    if constexpr (single) {
        __syncthreads();
        const PolicySum s = policy_block<NT>(policy_rows<NT>(part, p, row_tokens, 1), lds);
        if (threadIdx.x == 0) {
            policy_write(s, p, sums, counts, loss);
        }
    } else if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
        *done = 0;
    }
}

__global__ void __launch_bounds__(kThreads)
k_policy_join(const PolicyPart *part, PolicySum *block, unsigned *done, Policy p, unsigned lanes,
              float *sums, int64_t *counts, int32_t *row_tokens, float *loss)
{
    __shared__ PolicySum lds[kThreads / 64];
    __shared__ unsigned arrived;
    PolicySum s = policy_block<kThreads>(policy_rows<kThreads>(part, p, row_tokens, lanes), lds);
    if (threadIdx.x == 0) {
        block[blockIdx.x] = s;
    }
    if (last_block(done, &arrived)) {
        PolicySum t = {};
        if (threadIdx.x < gridDim.x) {
            t = block[threadIdx.x];
        }
        t = policy_block<kThreads>(t, lds);
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

/* the gradient of V tokens, each times its weight */
template <bool REF, bool ROW, typename T, int V>
__device__ __forceinline__ void policy_slope(const Tokens<T, V> &t, const Advantage &row, float w,
                                             const Policy &p, float (&o)[V])
{
#pragma unroll
    for (int k = 0; k < V; k++) {
        const Advantage a = ROW ? row : Advantage(t.adv[k], p);
        const float x = (float)t.logp[k], d = x - (float)t.old[k];
        float r = exp_of(d);
        asm("" : "+v"(r));
        float g = (a.cuts(d) ? 0.f : r) * -a.a;
        if constexpr (REF) {
            const float q = (float)t.ref[k] - x;
            g = __builtin_fmaf(-p.kl_coef, exp_minus(q), g);
        }
        asm("" : "+v"(g));
        o[k] = t.live[k] != 0 ? g * w : 0.f;
    }
}

/* 513 x 12345 bf16 with a reference and advantages by tokens takes 15.9 us = 5.2
 * TB/s, 1024 x 8192 fp32 25.5 us = 5.6 TB/s. A row's last tokens as in k_policy:
 * 2048 x 1023 bf16 9.6 us, 1024 6.6. */
template <typename T, bool REF, bool ROW, bool LINES>
__global__ void __launch_bounds__(kThreads)
k_policy_grad(PolicyIn<T, REF, ROW, LINES> in, const int32_t *row_tokens, const int64_t *counts,
              const float *grad_loss, T *dlogp, Policy p)
{
    constexpr int V = 16 / sizeof(T), S = policy_steps<T>();
    const PolicyWave<kThreads / 64> w(p);
    const unsigned l = w.l, cs = V << p.lanes_log;
    const uint64_t end = p.whole;
    for (uint64_t tile = w.row_tile; tile * w.per < p.rows; tile += w.tile_step)
    for (uint64_t chunk = w.chunk; chunk < p.chunks; chunk += w.chunk_step) {
        const uint64_t row = w.row(tile, p);
        if (row >= p.rows) {
            continue;
        }
        const uint64_t c0  = chunk * p.steps * cs + l * V;
        const uint64_t at  = row * p.ld + c0;
        Tokens<T, V> t[S];
#pragma unroll
        for (unsigned j = 0; j < S; j++) {
            if (j < p.steps && c0 + j * cs < end) {
                in.load(at + j * cs, t[j]);
            }
        }
        const Advantage a(ROW ? in.adv[row] : 0.f, p);
        const int64_t n = p.per_sequence ? counts[1] : counts[0];
        const double g  = grad_loss != nullptr ? (double)*grad_loss : 1.0;
        const int m     = p.per_sequence ? row_tokens[row] : 1;
        const float weight = n > 0 && m > 0 ? (float)(g / ((double)n * m)) : 0.f;
#pragma unroll
        for (unsigned j = 0; j < S; j++) {
            if (j < p.steps && c0 + j * cs < end) {
                float o[V];
                policy_slope<REF, ROW>(t[j], a, weight, p, o);
                store_vec<T, V>(dlogp + at + j * cs, o);
            }
        }
        /* the rest of the row, by the lane whose turn it would be */
        if (chunk == p.tail_chunk && l == p.tail_lane) {
#pragma unroll 1
            for (uint64_t c = end; c < p.cols; c++) {
                Tokens<T, 1> one;
                float o[1];
                in.load_one(row * p.ld + c, one);
                policy_slope<REF, ROW>(one, a, weight, p, o);
                dlogp[row * p.ld + c] = (T)o[0];
            }
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

struct Range {
    const void *p;
    size_t      bytes;
};

/* whether an output shares bytes with another output or with an input (NULL
 * ranges share none) */
bool clash(std::initializer_list<Range> outs, std::initializer_list<Range> ins)
{
    for (const Range *a = outs.begin(); a != outs.end(); a++) {
        if (a->p == nullptr) {
            continue;
        }
        for (const Range *b = a + 1; b != outs.end(); b++) {
            if (b->p != nullptr && overlap(a->p, a->bytes, b->p, b->bytes)) {
                return true;
            }
        }
        for (const Range &b : ins) {
            if (b.p != nullptr && overlap(a->p, a->bytes, b.p, b.bytes)) {
                return true;
            }
        }
    }
    return false;
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

/* f(T, whether there is a reference, whether advantages are by rows, whether
 * rows start on lines) */
template <typename F>
void with_policy(int dt, bool ref, bool row, bool lines, F f)
{
    const auto choose = [&](auto t, auto rf, auto rw) {
        if (lines) {
            f(t, rf, rw, std::true_type());
        } else {
            f(t, rf, rw, std::false_type());
        }
    };
    with_float(dt, [&](auto t) {
        if (ref && row) {
            choose(t, std::true_type(), std::true_type());
        } else if (ref) {
            choose(t, std::true_type(), std::false_type());
        } else if (row) {
            choose(t, std::false_type(), std::true_type());
        } else {
            choose(t, std::false_type(), std::false_type());
        }
    });
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
/* work-items of one launch (a dispatch counts them in 32 bits) */
constexpr uint64_t kMaxItems = (uint64_t)1 << 31;
/* columns of a bias whose gradient one launch can join (16 to a block) */
constexpr uint64_t kMaxBias = (uint64_t)1 << 27;

/* whether the waves' parts of an operand begin inside a 128-byte line */
template <typename T>
bool off_line(const void *p, uint64_t phase)
{
    return ((uintptr_t)p - phase * sizeof(T)) % 128 != 0;
}

template <typename T, typename R, int N>
void launch_sum(hipStream_t st, R *dst, const SrcList &srcs, unsigned nsrc, const T *bias,
                const R *residual, uint64_t n, uint64_t cols, const Rng &rng)
{
    constexpr uint64_t kMost = kMaxItems / 64;      /* waves of a launch */
    const uint64_t inv   = cols == 1 ? 0 : UINT64_MAX / cols + 1;
    const uint64_t waves = div_up(n + rng.offset % 8, kWaveElems);
    const uint64_t phase = rng.offset % 8;
    bool map = off_line<R>(dst, phase) || (residual != nullptr && off_line<R>(residual, phase));
    for (unsigned m = 0; m < nsrc; m++) {
        map = map || off_line<T>(srcs.p[m], phase);
    }
    for (uint64_t first = 0; first < waves; first += kMost) {
        const uint64_t left = waves - first < kMost ? waves - first : kMost;
        hipLaunchKernelGGL((k_sum_dropout<T, R, N>), dim3((unsigned)left), dim3(64), 0, st, dst,
                           srcs, nsrc, bias, residual, n, first, (int)map, cols, inv, rng);
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

/* how the gradient with the bias' part cuts its rows */
struct GradPlan {
    unsigned tx;                 /* lanes side by side */
    unsigned parts;
    uint64_t blocks_x;
    bool     deep;               /* a lane has more than kFewRows rows */
};

GradPlan grad_plan(uint64_t rows, uint64_t cols)
{
    GradPlan g;
    const uint64_t groups = div_up(cols, 8);
    g.tx = 2;                    /* neighbours share groups */
    while (g.tx < 64 && g.tx < groups) {
        g.tx *= 2;
    }
    g.blocks_x        = div_up(groups, g.tx);
    const uint64_t ty = kThreads / g.tx;
    /* 1024 blocks (2048 write twice the partials: 28.9 against 27.2 us for
     * 8192 x 4096 bf16), few enough parts to join at once, four rows a lane at
     * least */
    uint64_t parts = div_up(1024, g.blocks_x);
    parts   = parts < kMaxParts ? parts : kMaxParts;
    const uint64_t most = div_up(rows, ty * 4);
    parts   = parts < most ? parts : most;
    g.parts = parts > 0 ? (unsigned)parts : 1;
    g.deep  = div_up(rows, g.parts * ty) > kFewRows;
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

/* Blocks of k_balance: one to a CU at most, and to be joined at once. One block
 * does up to 32768 logits by itself, which takes less than a second launch (200
 * tokens of 8 experts 4.5 against 8.5 us, 300 of 64 6.2 against 7.7); beyond, a
 * block has 2048 logits at least, in 16 to 128 rows (1000 tokens of 256 experts
 * 8.6 us at 16 rows, 11.4 at 128; 3000 of 16 7.8 at 16 rows, 7.5 at 128). */
void balance_plan(uint64_t tokens, uint64_t experts, uint64_t *blocks, uint64_t *chunk)
{
    constexpr uint64_t kAlone = 32768;
    if (tokens <= kAlone / experts) {
        *chunk  = tokens;
        *blocks = 1;
        return;
    }
    const uint64_t c = div_up(tokens, kMaxParts), few = 2048 / experts;
    const uint64_t least = few < 16 ? 16 : few > 128 ? 128 : few;
    *chunk  = c < least ? least : c;
    *blocks = div_up(tokens, *chunk);
}

/* f(G lanes to a row, NV vectors to a lane, whether the row is whole vectors)
 * for `experts` columns */
template <typename T, typename F>
void with_layout(unsigned experts, F f)
{
    constexpr unsigned V = 16 / sizeof(T);
    const unsigned groups = (unsigned)div_up(experts, V);
    const auto even = [&](auto g, auto nv) {
        if (experts % V == 0) {
            f(g, nv, std::true_type());
        } else {
            f(g, nv, std::false_type());
        }
    };
    typedef std::integral_constant<int, 1> one;
    if (groups <= 1) {
        even(one(), one());
    } else if (groups <= 2) {
        even(std::integral_constant<int, 2>(), one());
    } else if (groups <= 4) {
        even(std::integral_constant<int, 4>(), one());
    } else if (groups <= 8) {
        even(std::integral_constant<int, 8>(), one());
    } else if (groups <= 16) {
        even(std::integral_constant<int, 16>(), one());
    } else if (groups <= 32) {
        even(std::integral_constant<int, 32>(), one());
    } else if (groups <= 64) {
        even(std::integral_constant<int, 64>(), one());
    } else if (groups <= 128) {
        even(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
    } else if constexpr (V == 4) {
        even(std::integral_constant<int, 64>(), std::integral_constant<int, 4>());
    }
}

/* ---- policy ---- */
constexpr unsigned kPolicyJoin = 64;      /* joining blocks at most */

void policy_split(uint64_t cols, int size, Policy *p)
{
    const unsigned V = 16 / size, most = size;     /* policy_steps() */
    const uint64_t groups = div_up(cols, V);
    p->lanes_log = 0;
    while (p->lanes_log < 6 && (1u << p->lanes_log) < groups) {
        p->lanes_log++;
    }
    const uint64_t lanes = (uint64_t)1 << p->lanes_log, vecs = div_up(groups, lanes);
    p->steps  = (unsigned)(vecs < most ? (vecs ? vecs : 1) : most);
    p->chunks = vecs ? div_up(vecs, p->steps) : 1;
    p->whole  = cols / V * V;
    const uint64_t step = p->whole / (lanes * V);       /* the last vector's */
    p->tail_chunk = p->whole < cols ? step / p->steps : UINT64_MAX;
    p->tail_lane  = (unsigned)(p->whole / V % lanes);
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
    p->per_sequence = q->per_sequence;
    p->up           = (float)log1p(q->clip_high);
    p->down         = (float)log1p(-q->clip_low);
    p->ratio_up     = (float)(1 + q->clip_high);
    p->ratio_down   = (float)(1 - q->clip_low);
    p->kl_coef      = (float)q->kl_coef;
    p->kl_coef64    = q->kl_coef;
    policy_split(q->cols, (int)size_of(q->dt), p);
    return UCS_OK;
}

/* blocks of W waves as PolicyWave lays them out */
dim3 policy_grid(const Policy &p, uint64_t W)
{
    uint64_t wc = 1;
    while (wc < W && wc < p.chunks) {
        wc *= 2;
    }
    const uint64_t x = div_up(div_up(p.rows, (uint64_t)64 >> p.lanes_log), W / wc);
    const uint64_t y = div_up(p.chunks, wc);
    const uint64_t most = 1u << 20;    /* the kernels go on from there in a loop */
    const uint64_t gy = y < 1024 ? y : 1024, gx = x ? x : 1;
    return dim3((unsigned)(gx < most / gy ? gx : most / gy), (unsigned)gy);
}

bool on_lines(const Policy &p, size_t size, const void *logp, const void *old, const void *ref)
{
    return (((uintptr_t)logp | (uintptr_t)old | (uintptr_t)ref | p.ld * size) & 127) == 0;
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
        if (clash({{dst, n * rs}}, {{residual != dst ? residual : nullptr, n * rs},
                                    {bias, params->cols * ts}, {params->rng, 16}})) {
            return invalid(what, "dst overlaps the residual, the bias or rng");
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
    if (cols == 0 || cols > kMaxBias) {
        return 0;
    }
    const GradPlan g = grad_plan(rows, cols);
    return g.parts > 1 ? round16(g.parts * cols * sizeof(float)) : 0;
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
        clash({{dsrc, n * ts}, {dbias, cols * 4}, {need ? workspace : nullptr, need}},
              {{params->rng, 16}}) ||
        clash({{dbias, cols * 4}, {need ? workspace : nullptr, need}}, {{grad, n * rs}})) {
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
        const GradPlan plan = grad_plan(rows, cols);
        float *out          = plan.parts > 1 ? static_cast<float*>(workspace) : dbias;
        const dim3 grid((unsigned)plan.blocks_x, plan.parts);
        const auto launch = [&](auto aligned, auto deep) {
            hipLaunchKernelGGL((k_dropout_grad<R, T, decltype(aligned)::value, decltype(deep)::value>),
                               grid, dim3(kThreads), 0, stream, d, g, out, rows, cols, plan.tx, rng);
        };
        const auto launch_deep = [&](auto aligned) {
            if (plan.deep) {
                launch(aligned, std::true_type());
            } else {
                launch(aligned, std::false_type());
            }
        };
        if (cols % 8 == 0 && rng.offset % 8 == 0) {
            launch_deep(std::true_type());
        } else {
            launch_deep(std::false_type());
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
    if (experts == 0) {
        return 0;
    }
    balance_plan(tokens, experts, &blocks, &chunk);
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
    if (clash({{counts, (b.experts + 1) * sizeof(int64_t)}, {sums, (b.experts + 1) * sizeof(float)},
               {loss, 3 * sizeof(float)}, {need ? workspace : nullptr, need}},
              {{logits, bytes}, {index, index_bytes}, {mask, b.tokens}})) {
        return invalid(what, "overlapping buffers");
    }
    if (ctx == nullptr) {
        return invalid(what, "ctx is NULL");
    }
    uint64_t blocks;
    balance_plan(b.tokens, b.experts, &blocks, &b.chunk);
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
        with_layout<T>(b.experts, [&](auto g, auto nv, auto even) {
            constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
            constexpr bool EVEN = decltype(even)::value;
            /* a wave has 64 / G rows at once */
            const bool deep = div_up(b.chunk, kBalanceThreads / G) > kFewRows;
            const auto launch = [&](auto i, auto dp) {
                typedef decltype(i) I;
                hipLaunchKernelGGL((k_balance<T, I, G, NV, EVEN, decltype(dp)::value>),
                                   dim3((unsigned)blocks), dim3(kBalanceThreads), 0, stream,
                                   static_cast<const T*>(logits), static_cast<const I*>(index),
                                   mask, b, part, direct, sums, loss);
            };
            const auto launch_index = [&](auto dp) {
                if (is == 4) {
                    launch(int32_t(), dp);
                } else {
                    launch(int64_t(), dp);
                }
            };
            if (deep) {
                launch_index(std::true_type());
            } else {
                launch_index(std::false_type());
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
    if (clash({{loss, 3 * sizeof(float)}}, {{counts, (b.experts + 1) * sizeof(int64_t)},
                                            {sums, (b.experts + 1) * sizeof(float)}})) {
        return invalid(what, "overlapping buffers");
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
        clash({{dlogits, out_bytes}}, {{base != dlogits ? base : nullptr, out_bytes},
                                       {mask, b.tokens},
                                       {counts, (b.experts + 1) * sizeof(int64_t)},
                                       {grad_loss, sizeof(float)}})) {
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
        with_layout<T>(b.experts, [&](auto g, auto nv, auto even) {
            constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
            constexpr bool EVEN = decltype(even)::value;
            const uint64_t want = div_up(b.tokens, 4 * (64 / G) * (NV == 1 ? 2 : 1));
            const unsigned grid = (unsigned)(want < 1024 ? want : 1024);
            hipLaunchKernelGGL((k_balance_grad<T, G, NV, EVEN>), dim3(grid), dim3(kThreads), 0, stream,
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
    for (int size : {2, 4}) {
        Policy p;
        policy_split(cols, size, &p);
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
    const size_t nb = bytes / 4 * ts;
    if (clash({{sums, 2 * sizeof(float)}, {counts, 3 * sizeof(int64_t)}, {row_tokens, p.rows * 4},
               {loss, 3 * sizeof(float)}, {workspace, need}},
              {{logp, nb}, {old, nb}, {ref, nb}, {mask, bytes / 4},
               {adv, params->adv_per_row ? p.rows * 4 : bytes}})) {
        return invalid(what, "overlapping buffers");
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
    const dim3 grid    = policy_grid(p, kThreads / 64);
    /* one block does a few parts by itself: a second launch costs more. Without
     * rows it has none, however many a row would have, and writes the zeros. */
    const bool single = p.rows == 0 || (grid.x * grid.y <= 4 &&
                                        p.rows * p.chunks <= (uint64_t)kSingleParts);
    const bool lines = on_lines(p, ts, logp, old, ref);
    /* rows without columns: adv may be NULL, and is not read by rows either */
    const bool by_row = params->adv_per_row != 0 && bytes != 0;
    with_policy(params->dt, ref != nullptr, by_row, lines && !single,
                [&](auto t, auto rf, auto rw, auto ln) {
        typedef decltype(t) T;
        constexpr bool REF = decltype(rf)::value, ROW = decltype(rw)::value;
        constexpr bool LINES = decltype(ln)::value;
        const PolicyIn<T, REF, ROW, LINES> in = {static_cast<const T*>(logp),
                                                 static_cast<const T*>(old),
                                                 static_cast<const T*>(ref), adv, mask};
        if constexpr (!LINES) {
            if (single) {
                hipLaunchKernelGGL((k_policy<T, REF, ROW, false, kSingle>), dim3(1),
                                   dim3(kSingle), 0, stream, in, p, part, done, sums, counts,
                                   row_tokens, loss);
                return;
            }
        }
        hipLaunchKernelGGL((k_policy<T, REF, ROW, LINES, kThreads>), grid, dim3(kThreads), 0,
                           stream, in, p, part, done, sums, counts, row_tokens, loss);
    });
    if (!single) {
        unsigned lanes = 1;               /* with eight parts each */
        while (lanes < 64 && lanes * 8 < p.chunks) {
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
    if (clash({{loss, 3 * sizeof(float)}}, {{counts, 3 * sizeof(int64_t)},
                                            {sums, 2 * sizeof(float)}})) {
        return invalid(what, "overlapping buffers");
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
    if (clash({{dlogp, nb}}, {{logp != dlogp ? logp : nullptr, nb}, {old != dlogp ? old : nullptr, nb},
                              {ref != dlogp ? ref : nullptr, nb}, {mask, bytes / 4},
                              {adv, params->adv_per_row ? p.rows * 4 : bytes},
                              {row_tokens, p.rows * 4}, {counts, 3 * sizeof(int64_t)},
                              {grad_loss, sizeof(float)}})) {
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
    const bool lines = on_lines(p, ts, logp, old, ref);
    with_policy(params->dt, ref != nullptr, params->adv_per_row != 0, lines,
                [&](auto t, auto rf, auto rw, auto ln) {
        typedef decltype(t) T;
        constexpr bool REF = decltype(rf)::value, ROW = decltype(rw)::value;
        constexpr bool LINES = decltype(ln)::value;
        const PolicyIn<T, REF, ROW, LINES> in = {static_cast<const T*>(logp),
                                                 static_cast<const T*>(old),
                                                 static_cast<const T*>(ref), adv, mask};
        hipLaunchKernelGGL((k_policy_grad<T, REF, ROW, LINES>), policy_grid(p, kThreads / 64),
                           dim3(kThreads), 0, stream_of(ctx), in, row_tokens, counts, grad_loss,
                           static_cast<T*>(dlogp), p);
    });
    HIP_TRY(hipGetLastError());
    dev_ctx_count(ctx, 1, 0);
    return UCS_OK;
}

}  /* extern "C" */
