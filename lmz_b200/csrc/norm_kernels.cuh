// Root-mean-square norms with the residual's addition, their output as it is or in 8 bits, and their gradients.
//
//   s[t] = x[t] + r[t], rounded to the tensors' type (it is the residual stream that goes on);  n[t] = s[t] / sqrt(mean(s[t]^2) + eps)
//   y[t] = n[t] w;  in 8 bits: q[t] = y[t] / scale[t], scale[t] = max |y[t]| / 448
//   ds[t] += rstd[t] (dy[t] w - n[t] mean(dy[t] w n[t])),  dw = sum of dy[t] n[t]
#pragma once
#include <cuda_fp8.h>

#include "tcgen.cuh"
#include "vectors.cuh"

namespace lmz {

constexpr uint32_t NORM_THREADS = 256, NORM_MOST = 1024;
// Elements that a thread has of a row in registers.  Where vectors are narrow, half as many: a thread has more loads to wait for then (one B200, gradients
// of 3001x997 FP32, rows that start on 4 bytes: 31 us by sixteen, 9 by eight).
__host__ __device__ constexpr uint32_t norm_each(uint32_t vector_bytes) { return vector_bytes == 16 ? 16 : 8; }

struct NormArgs {
    const void *x, *residual, *weight;           // residual: or NULL; weight: NULL for rows that only go to 8 bits
    void *y, *stream;                            // y or q
    uint8_t *q;
    float *scale, *rstd;                         // rstd: kept for the gradients, or NULL
    uint64_t tokens, dim, x_stride, residual_stride;
    uint32_t vectors;                            // of a row
    uint32_t lane_log;                           // 2^lane_log threads share a row
    float eps;
};

// A row's sum over the 2^log threads that share it; `room`: a word per warp of the block.  All threads of a block call it together.
__device__ __forceinline__ float row_sum(float v, uint32_t log, float *room)
{
    for (uint32_t o = 1; o < 32 && o >> log == 0; o <<= 1) v += __shfl_xor_sync(~0u, v, o);
    if (log <= 5) return v;
    const uint32_t warps = 1u << (log - 5), warp = threadIdx.x >> 5, first = warp & ~(warps - 1);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) room[warp] = v;
    __syncthreads();
    v = room[first + (threadIdx.x & (warps - 1))];
    for (uint32_t o = 1; o < warps; o <<= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

// And its largest magnitude, by its bits: those of a NaN are above those of infinity, so that it stays.
__device__ __forceinline__ float row_most(uint32_t v, uint32_t log, float *room)
{
    if (log < 5) {
        for (uint32_t o = 1; o >> log == 0; o <<= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
        return __uint_as_float(v);
    }
    v = __reduce_max_sync(~0u, v);
    if (log == 5) return __uint_as_float(v);
    const uint32_t warps = 1u << (log - 5), warp = threadIdx.x >> 5, first = warp & ~(warps - 1);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) room[warp] = __uint_as_float(v);
    __syncthreads();
    return __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(room[first + (threadIdx.x & (warps - 1))])));
}

template <class W, int N>
__device__ __forceinline__ void load_weights(const W *from, float *to)
{
    constexpr int B = N * sizeof(W) < 16 ? N * sizeof(W) : 16;
    using V = Vec<W, B>;
#pragma unroll
    for (int i = 0; i < N / V::N; i++) {
        V v;
        v.raw = reinterpret_cast<const typename Raw<B>::type *>(from)[i];
        widen_all(v, to + i * V::N);
    }
}

__device__ __forceinline__ float rms_of(float squares, uint64_t dim, float eps) { return 1.0f / sqrtf(squares / static_cast<float>(dim) + eps); }

// 448 is the largest number that 8 bits with 4 of exponent and 3 of mantissa hold.  A row of zeros gets the smallest scale there is, below which
// the quotient would lose bits.
__device__ __forceinline__ float scale_of_most(float most)
{
    const float s = most / 448.0f;
    return s < 1.17549435e-38f ? 1.17549435e-38f : s;            // (a NaN stays)
}

// u / v for rounding to 8 bits, by v's correctly rounded reciprocal: the first product is at most one and a half units in the last place off, and its remainder, which a
// multiply-add has to one unit, brings it to within 2^-22 of a unit before it is rounded.  Whether that is on the same side of the middle between two numbers of 8 bits as
// the quotient in 32 bits can go wrong only next to that middle's neighbours: where v's 24 bits are within eight of a multiple of 2^20.  All of those, and 64 on either
// side, with every such middle, are right but one, 2^24 - 1, which is left to division.  (Remainders of quotients that 8 bits tell from zero, 2^-10 and more, have to be
// numbers of 32 bits.)  A third of a division's instructions; a second step of the same kind would cost 8192x8192 5 us of 83.
__device__ __forceinline__ bool divides(float v) { return v > 0x1p-60f && v < 0x1p60f && (~__float_as_uint(v) & 0x7FFFFF); }
__device__ __forceinline__ float divided(float u, float v, float reciprocal)
{
    const float q = u * reciprocal;
    return fmaf(fmaf(-q, v, u), reciprocal, q);
}

// N numbers of 8 bits, as one store.
template <int N>
__device__ __forceinline__ void store_8bit(uint8_t *to, const float *v)
{
    if constexpr (N == 1) {
        *to = __nv_cvt_float_to_fp8(v[0], __NV_SATFINITE, __NV_E4M3);
    } else {
        auto two = [&](int e) -> uint32_t { return __nv_cvt_float2_to_fp8x2(make_float2(v[e], v[e + 1]), __NV_SATFINITE, __NV_E4M3); };
        if constexpr (N == 2) {
            *reinterpret_cast<uint16_t *>(to) = static_cast<uint16_t>(two(0));
        } else {
            union { uint32_t word[N / 4]; typename Raw<N>::type raw; } all;
#pragma unroll
            for (int e = 0; e < N; e += 4) all.word[e / 4] = two(e) | two(e + 2) << 16;
            *reinterpret_cast<typename Raw<N>::type *>(to) = all.raw;
        }
    }
}

// A row's 2^lane_log threads take its vectors of VB bytes in turn.  What a thread has of a row stays in registers, so that a row is read once;
// LONG: rows of more elements than NORM_MOST threads hold are read again for each pass, out of L2.  Sums in 32 bits.
//
// WHOLE: every thread has a whole share of a row, and nothing is asked for each vector.
//
// Bound by HBM (x and the residual read, the stream and y written), in 8 bits nearly by the instructions, too.  A row is a block's or less: 16 elements
// a thread (of a row of 8192, by 8 elements 125 us, by 16 95, by 32 103, before loads went ahead).  One B200, BF16 with a residual: 16384x4096 80 us
// (6.7 TB/s), 8192x8192 to 8 bits 83 (5.7 TB/s), 1x4096 2.4.  32 registers, so that two blocks of 1024 threads have room: FP32 rows, and odd 16-bit ones, put some of
// theirs away for that (16384x4096 FP32 197 us, 5.4 TB/s).
template <class T, class W, int VB, bool BITS8, bool LONG, bool WHOLE>
__global__ void __launch_bounds__(NORM_MOST, 2) k_norm(const NormArgs a)
{
    using V = Vec<T, VB>;
    using R = typename Raw<VB>::type;
    constexpr int NV = LONG ? 1 : norm_each(VB) / V::N;
    __shared__ float room[2][32];
    const uint32_t lanes = 1u << a.lane_log, lane = threadIdx.x & (lanes - 1);
    const uint64_t t = static_cast<uint64_t>(blockIdx.x) * (blockDim.x >> a.lane_log) + (threadIdx.x >> a.lane_log);
    const bool on = WHOLE || t < a.tokens;
    auto has = [&](int i) { return WHOLE || (on && lane + i * lanes < a.vectors); };
    const R *x = reinterpret_cast<const R *>(static_cast<const T *>(a.x) + (on ? t : 0) * a.x_stride);
    const R *res = reinterpret_cast<const R *>(static_cast<const T *>(a.residual) + (on ? t : 0) * a.residual_stride);
    R *stream = reinterpret_cast<R *>(static_cast<T *>(a.stream) + t * a.dim);
    const W *weight = static_cast<const W *>(a.weight);
    wait_for_previous();
    let_next_start();

    auto take = [&](uint32_t v, V p, V q, float *to, bool write) {               // s
        if (a.residual) {
            float both[V::N], other[V::N];
            widen_all(p, both), widen_all(q, other);
#pragma unroll
            for (int e = 0; e < V::N; e++) both[e] += other[e];
            narrow_all(both, p);
            if (write && a.stream) stream[v] = p.raw;
        }
        widen_all(p, to);
    };
    auto load = [&](uint32_t v, float *to, bool write) {
        V p, q;
        p.raw = x[v];
        if (a.residual) q.raw = res[v];
        take(v, p, q, to, write);
    };
    float s[NV][V::N];
    float squares = 0;
    if constexpr (LONG) {
        if (on)
            for (uint32_t v = lane; v < a.vectors; v += lanes) {
                load(v, s[0], true);
#pragma unroll
                for (int e = 0; e < V::N; e++) squares += s[0][e] * s[0][e];
            }
    } else {
        V p[NV], q[NV];                                          // (all on their way before the first is waited for)
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (has(i)) p[i].raw = x[lane + i * lanes];
        if (a.residual) {
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (has(i)) q[i].raw = res[lane + i * lanes];
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            if (!has(i)) continue;
            take(lane + i * lanes, p[i], q[i], s[i], true);
#pragma unroll
            for (int e = 0; e < V::N; e++) squares += s[i][e] * s[i][e];
        }
    }
    float rstd = 1;
    if (weight) {
        rstd = rms_of(row_sum(squares, a.lane_log, room[0]), a.dim, a.eps);
        if (a.rstd && on && lane == 0) a.rstd[t] = rstd;
    }
    auto normed = [&](uint32_t v, float *u) {                    // s -> y, in 32 bits
        if (!weight) return;
        float w[V::N];
        load_weights<W, V::N>(weight + v * V::N, w);
#pragma unroll
        for (int e = 0; e < V::N; e++) u[e] = u[e] * rstd * w[e];
    };
    auto each = [&](auto f) {                                    // every vector's y
        if (!on) return;
        if constexpr (LONG) {
            for (uint32_t v = lane; v < a.vectors; v += lanes) {
                load(v, s[0], false);
                normed(v, s[0]);
                f(v, s[0]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (has(i)) f(lane + i * lanes, s[i]);
        }
    };
    if constexpr (!LONG) {
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (has(i)) normed(lane + i * lanes, s[i]);
    }
    if constexpr (BITS8) {
        uint32_t most = 0;
        each([&](uint32_t, const float *u) {
#pragma unroll
            for (int e = 0; e < V::N; e++) most = max(most, __float_as_uint(u[e]) & 0x7FFFFFFF);
        });
        const float scale = scale_of_most(row_most(most, a.lane_log, room[1])), inverse = 1.0f / scale;
        if (on && lane == 0) a.scale[t] = scale;
        const bool quick = divides(scale);
        auto write = [&](auto quotient) {
            each([&](uint32_t v, const float *u) {
                float d[V::N];
#pragma unroll
                for (int e = 0; e < V::N; e++) d[e] = quotient(u[e]);
                store_8bit<V::N>(a.q + t * a.dim + static_cast<uint64_t>(v) * V::N, d);
            });
        };
        if (quick) write([&](float u) { return divided(u, scale, inverse); });
        else write([&](float u) { return u / scale; });
    } else {
        each([&](uint32_t v, const float *u) {
            V p;
            narrow_all(u, p);
            reinterpret_cast<R *>(static_cast<T *>(a.y) + t * a.dim)[v] = p.raw;
        });
    }
}

struct NormGradArgs {
    const void *s, *weight, *dy, *ds;            // s: what was normed (rows s_stride apart); ds: the stream's own gradient, or NULL
    const float *rstd;
    void *dx;                                    // or NULL
    float *partial;                              // [block][dim]: its sum of dy n; or NULL
    uint64_t tokens, dim, s_stride;
    uint32_t vectors, lane_log;
};

// The gradient of s, and each block's share of the weight's: a row of threads takes every (rows of threads)-th token, and a block's rows of
// threads add up in their order, so that sums have one order.  LONG: the shares lie in global memory, where a thread finds its own columns again.
//
// MOST: threads of a block.  WHOLE: every thread has a whole share of a row.
//
// Bound by HBM: dy, s and ds read, dx written.  One B200, 16384x4096 BF16: 91 us without the weight's gradient (5.9 TB/s), 102 with it and k_join (130 before words
// were taken apart two elements at a time).  Going by n costs 3 us of that: the same by s times rstd^3 left 32 bits' range on the way.
template <class T, class W, int VB, bool LONG, uint32_t MOST, bool WHOLE>
__global__ void __launch_bounds__(MOST, NORM_MOST / MOST) k_norm_grad(const NormGradArgs a)
{
    using V = Vec<T, VB>;
    using R = typename Raw<VB>::type;
    constexpr int NV = LONG ? 1 : norm_each(VB) / V::N;
    constexpr bool SEVERAL = MOST == NORM_THREADS;               // rows of threads in a block, at times
    __shared__ float room[2][32];
    __shared__ float shares[SEVERAL ? NORM_THREADS * norm_each(VB) / 2 : 1];
    const uint32_t lanes = 1u << a.lane_log, lane = threadIdx.x & (lanes - 1), per = blockDim.x >> a.lane_log, sub = threadIdx.x >> a.lane_log;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * per;
    const W *weight = static_cast<const W *>(a.weight);
    float *share = a.partial + blockIdx.x * a.dim;
    wait_for_previous();
    let_next_start();
    float sum[NV][V::N];
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int e = 0; e < V::N; e++) sum[i][e] = 0;
    auto has = [&](int i) { return WHOLE || lane + i * lanes < a.vectors; };
    uint32_t turn = 0;
    // (a block's rows of threads make as many turns as its first one, whose tokens are the lowest: they meet at barriers)
    for (uint64_t t0 = static_cast<uint64_t>(blockIdx.x) * per; t0 < a.tokens; t0 += step, turn++) {
        const uint64_t t = t0 + sub;
        const bool on = t < a.tokens;
        const R *s = reinterpret_cast<const R *>(static_cast<const T *>(a.s) + (on ? t : 0) * a.s_stride);
        const R *dy = reinterpret_cast<const R *>(static_cast<const T *>(a.dy) + (on ? t : 0) * a.dim);
        const R *ds = reinterpret_cast<const R *>(static_cast<const T *>(a.ds) + (on ? t : 0) * a.dim);
        R *dx = reinterpret_cast<R *>(static_cast<T *>(a.dx) + t * a.dim);
        const float rstd = on ? a.rstd[t] : 0;
        V n[NV], g[NV], d[NV];
        float along = 0;                                         // the sum of dy w n
        auto load = [&](uint32_t v, V &p, V &q, V &r) {
            p.raw = s[v], q.raw = dy[v];
            if (a.ds) r.raw = ds[v];
        };
        auto add = [&](uint32_t v, const V &p, const V &q) {
            float w[V::N], x[V::N], y[V::N];
            load_weights<W, V::N>(weight + v * V::N, w);
            widen_all(p, x), widen_all(q, y);
#pragma unroll
            for (int e = 0; e < V::N; e++) along += y[e] * w[e] * (x[e] * rstd);
        };
        auto finish = [&](uint32_t v, const V &p, const V &q, V r, float toward, float *sums) {
            float w[V::N], x[V::N], y[V::N], u[V::N];
            load_weights<W, V::N>(weight + v * V::N, w);
            widen_all(p, x), widen_all(q, y);
#pragma unroll
            for (int e = 0; e < V::N; e++) {
                x[e] *= rstd;
                sums[e] += y[e] * x[e];
                u[e] = (y[e] * w[e] - x[e] * toward) * rstd;
            }
            if (!a.dx) return;
            if (a.ds) {
                widen_all(r, w);
#pragma unroll
                for (int e = 0; e < V::N; e++) u[e] += w[e];
            }
            narrow_all(u, r);
            dx[v] = r.raw;
        };
        if constexpr (LONG) {
            if (on)
                for (uint32_t v = lane; v < a.vectors; v += lanes) {
                    load(v, n[0], g[0], d[0]);
                    add(v, n[0], g[0]);
                }
        } else {
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (on && has(i)) load(lane + i * lanes, n[i], g[i], d[i]);
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (on && has(i)) add(lane + i * lanes, n[i], g[i]);
        }
        // (by n, and not by s rstd^3: neither rstd's powers nor products with s stay within 32 bits wherever the squares do)
        const float toward = row_sum(along, a.lane_log, room[turn & 1]) / static_cast<float>(a.dim);
        if (!on) continue;
        if constexpr (LONG) {
            for (uint32_t v = lane; v < a.vectors; v += lanes) {
                float *mine = share + static_cast<uint64_t>(v) * V::N;
                load(v, n[0], g[0], d[0]);
#pragma unroll
                for (int e = 0; e < V::N; e++) sum[0][e] = turn && a.partial ? mine[e] : 0;
                finish(v, n[0], g[0], d[0], toward, sum[0]);
#pragma unroll
                for (int e = 0; e < V::N; e++)
                    if (a.partial) mine[e] = sum[0][e];
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (has(i)) finish(lane + i * lanes, n[i], g[i], d[i], toward, sum[i]);
        }
    }
    if (LONG || !a.partial) return;
    auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (has(i))
#pragma unroll
                for (int e = 0; e < V::N; e++) f((lane + i * lanes) * V::N + e, sum[i][e]);
    };
    if constexpr (SEVERAL) {                                     // (of at most half of the columns that NORM_THREADS have)
        for (uint32_t k = 0; k + 1 < per; k++) {
            if (sub == k) each([&](uint32_t c, float v) { shares[c] = k ? shares[c] + v : v; });
            __syncthreads();
        }
        if (sub + 1 != per) return;
        if (per > 1) each([&](uint32_t c, float &v) { v += shares[c]; });
    }
    each([&](uint32_t c, float v) { share[c] = v; });
}

// out[d] = the sum of `rows` shares.  A block has 32 columns; its warps take the shares in turn, and their sums meet in their order.  Bound by latency: 592
// shares of 4096 (in L2) 6 us, by half the warps and without loads ahead 10.
constexpr uint32_t JOIN_WARPS = 32, JOIN_AHEAD = 10;
template <class W>
__global__ void __launch_bounds__(32 * JOIN_WARPS) k_join(const float *partial, uint64_t rows, uint64_t dim, W *out)
{
    __shared__ float sums[JOIN_WARPS][32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t d = blockIdx.x * 32ull + lane;
    wait_for_previous();
    let_next_start();
    float sum = 0;
    if (d < dim)
        for (uint64_t r = warp; r < rows; r += JOIN_WARPS * JOIN_AHEAD) {
            float v[JOIN_AHEAD];
#pragma unroll
            for (uint32_t i = 0; i < JOIN_AHEAD; i++) v[i] = r + i * JOIN_WARPS < rows ? partial[(r + i * JOIN_WARPS) * dim + d] : 0;
#pragma unroll
            for (uint32_t i = 0; i < JOIN_AHEAD; i++) sum += v[i];
        }
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp || d >= dim) return;
    for (uint32_t w = 1; w < JOIN_WARPS; w++) sum += sums[w][lane];
    out[d] = narrow<W>(sum);
}

}  // namespace lmz
