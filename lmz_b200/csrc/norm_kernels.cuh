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

constexpr uint32_t NORM_THREADS = 256, NORM_MOST = 1024, NORM_EACH = 16;     // elements that a thread has of a row in registers

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

// Sums and largest values over the 2^log threads that share a row; `room`: a word per warp of the block.  All threads of a block call it
// together, and once per pass over rows with a room of its own.
template <class F>
__device__ __forceinline__ float row_join(float v, uint32_t log, float *room, F both)
{
    for (uint32_t o = 1; o < 32 && o >> log == 0; o <<= 1) v = both(v, __shfl_xor_sync(~0u, v, o));
    if (log <= 5) return v;
    const uint32_t warps = 1u << (log - 5), warp = threadIdx.x >> 5, first = warp & ~(warps - 1);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) room[warp] = v;
    __syncthreads();
    v = room[first + (threadIdx.x & (warps - 1))];
    for (uint32_t o = 1; o < warps; o <<= 1) v = both(v, __shfl_xor_sync(~0u, v, o));
    return v;
}
__device__ __forceinline__ float row_sum(float v, uint32_t log, float *room)
{
    return row_join(v, log, room, [](float a, float b) { return a + b; });
}
// (By their bits: those of a NaN are above those of infinity, so that it stays.)
__device__ __forceinline__ float row_most(float v, uint32_t log, float *room)
{
    return row_join(v, log, room, [](float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); });
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
#pragma unroll
        for (int e = 0; e < V::N; e++) to[i * V::N + e] = widen(v.e[e]);
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

// u / v rounded once, by v's reciprocal: the quotient's remainder, which one multiply-add has exactly, corrects it (Markstein's theorem: a
// correctly rounded reciprocal and this step give the correctly rounded quotient).  A third of a division's instructions.
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
        union { uint16_t part[N / 2]; typename Raw<N>::type raw; } all;
#pragma unroll
        for (int e = 0; e < N; e += 2) all.part[e / 2] = __nv_cvt_float2_to_fp8x2(make_float2(v[e], v[e + 1]), __NV_SATFINITE, __NV_E4M3);
        *reinterpret_cast<typename Raw<N>::type *>(to) = all.raw;
    }
}

// A row's 2^lane_log threads take its vectors of VB bytes in turn.  What a thread has of a row stays in registers, so that a row is read once;
// LONG: rows of more elements than NORM_MOST threads hold are read again for each pass, out of L2.  Sums in 32 bits.
//
// Bound by HBM: x and the residual read, the stream and y written.
template <class T, class W, int VB, bool BITS8, bool LONG>
__global__ void __launch_bounds__(NORM_MOST) k_norm(const NormArgs a)
{
    using V = Vec<T, VB>;
    using R = typename Raw<VB>::type;
    constexpr int NV = LONG ? 1 : NORM_EACH / V::N;
    __shared__ float room[2][32];
    const uint32_t lanes = 1u << a.lane_log, lane = threadIdx.x & (lanes - 1);
    const uint64_t t = static_cast<uint64_t>(blockIdx.x) * (blockDim.x >> a.lane_log) + (threadIdx.x >> a.lane_log);
    const bool on = t < a.tokens;
    const R *x = reinterpret_cast<const R *>(static_cast<const T *>(a.x) + (on ? t : 0) * a.x_stride);
    const R *res = reinterpret_cast<const R *>(static_cast<const T *>(a.residual) + (on ? t : 0) * a.residual_stride);
    R *stream = reinterpret_cast<R *>(static_cast<T *>(a.stream) + t * a.dim);
    const W *weight = static_cast<const W *>(a.weight);
    wait_for_previous();
    let_next_start();

    auto load = [&](uint32_t v, float *to, bool write) {         // s
        V p;
        p.raw = x[v];
        if (a.residual) {
            V q;
            q.raw = res[v];
#pragma unroll
            for (int e = 0; e < V::N; e++) p.e[e] = narrow<T>(widen(p.e[e]) + widen(q.e[e]));
            if (write && a.stream) stream[v] = p.raw;
        }
#pragma unroll
        for (int e = 0; e < V::N; e++) to[e] = widen(p.e[e]);
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
#pragma unroll
        for (int i = 0; i < NV; i++) {
#pragma unroll
            for (int e = 0; e < V::N; e++) s[i][e] = 0;
            if (on && lane + i * lanes < a.vectors) load(lane + i * lanes, s[i], true);
        }
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int e = 0; e < V::N; e++) squares += s[i][e] * s[i][e];
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
                if (lane + i * lanes < a.vectors) f(lane + i * lanes, s[i]);
        }
    };
    if constexpr (!LONG) {
#pragma unroll
        for (int i = 0; i < NV; i++)
            if (on && lane + i * lanes < a.vectors) normed(lane + i * lanes, s[i]);
    }
    if constexpr (BITS8) {
        float most = 0;
        each([&](uint32_t, const float *u) {
#pragma unroll
            for (int e = 0; e < V::N; e++) most = __uint_as_float(max(__float_as_uint(most), __float_as_uint(u[e]) & 0x7FFFFFFF));
        });
        const float scale = scale_of_most(row_most(most, a.lane_log, room[1])), inverse = 1.0f / scale;
        if (on && lane == 0) a.scale[t] = scale;
        const bool quick = scale > 1e-30f && scale < 1e30f;      // (neither NaN nor infinite, and no remainder below the smallest number)
        each([&](uint32_t v, const float *u) {
            float d[V::N];
#pragma unroll
            for (int e = 0; e < V::N; e++) d[e] = quick ? divided(u[e], scale, inverse) : u[e] / scale;
            store_8bit<V::N>(a.q + t * a.dim + static_cast<uint64_t>(v) * V::N, d);
        });
    } else {
        each([&](uint32_t v, const float *u) {
            V p;
#pragma unroll
            for (int e = 0; e < V::N; e++) p.e[e] = narrow<T>(u[e]);
            reinterpret_cast<R *>(static_cast<T *>(a.y) + t * a.dim)[v] = p.raw;
        });
    }
}

struct NormGradArgs {
    const void *s, *weight, *dy, *ds;            // s: what was normed (rows s_stride apart); ds: the stream's own gradient, or NULL
    const float *rstd;
    void *dx;                                    // or NULL
    float *partial;                              // [row of threads][dim]: each one's sum of dy n; or NULL
    uint64_t tokens, dim, s_stride;
    uint32_t vectors, lane_log;
};

// The gradient of s, and each row of threads' share of the weight's: a row of threads takes every (rows of threads)-th token, so that
// its sums have one order.  LONG: the shares lie in global memory, where a thread finds its own columns again.
//
// Bound by HBM: dy, s and ds read, dx written.
template <class T, class W, int VB, bool LONG>
__global__ void __launch_bounds__(NORM_MOST) k_norm_grad(const NormGradArgs a)
{
    using V = Vec<T, VB>;
    using R = typename Raw<VB>::type;
    constexpr int NV = LONG ? 1 : NORM_EACH / V::N;
    __shared__ float room[2][32];
    const uint32_t lanes = 1u << a.lane_log, lane = threadIdx.x & (lanes - 1), per = blockDim.x >> a.lane_log;
    const uint64_t me = static_cast<uint64_t>(blockIdx.x) * per + (threadIdx.x >> a.lane_log), step = static_cast<uint64_t>(gridDim.x) * per;
    const W *weight = static_cast<const W *>(a.weight);
    float *share = a.partial + me * a.dim;
    wait_for_previous();
    let_next_start();
    float sum[NV][V::N];
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int e = 0; e < V::N; e++) sum[i][e] = 0;
    uint32_t turn = 0;
    // (a block's rows of threads make as many turns as its first one, whose tokens are the lowest: they meet at barriers)
    for (uint64_t t0 = static_cast<uint64_t>(blockIdx.x) * per; t0 < a.tokens; t0 += step, turn++) {
        const uint64_t t = t0 + (threadIdx.x >> a.lane_log);
        const bool on = t < a.tokens;
        const R *s = reinterpret_cast<const R *>(static_cast<const T *>(a.s) + (on ? t : 0) * a.s_stride);
        const R *dy = reinterpret_cast<const R *>(static_cast<const T *>(a.dy) + (on ? t : 0) * a.dim);
        const float rstd = on ? a.rstd[t] : 0;
        V n[NV], g[NV];
        float along = 0;
        auto load = [&](uint32_t v, V &p, V &q) { p.raw = s[v], q.raw = dy[v]; };
        auto add = [&](uint32_t v, const V &p, const V &q) {
            float w[V::N];
            load_weights<W, V::N>(weight + v * V::N, w);
#pragma unroll
            for (int e = 0; e < V::N; e++) along += widen(q.e[e]) * w[e] * (widen(p.e[e]) * rstd);
        };
        auto finish = [&](uint32_t v, const V &p, const V &q, float mean, float *sums) {
            float w[V::N];
            V d;
            load_weights<W, V::N>(weight + v * V::N, w);
            d.raw = {};
            if (a.ds) d.raw = reinterpret_cast<const R *>(static_cast<const T *>(a.ds) + t * a.dim)[v];
#pragma unroll
            for (int e = 0; e < V::N; e++) {
                const float ne = widen(p.e[e]) * rstd, ge = widen(q.e[e]);
                sums[e] += ge * ne;
                const float u = rstd * (ge * w[e] - ne * mean);
                d.e[e] = narrow<T>(a.ds ? u + widen(d.e[e]) : u);
            }
            if (a.dx) reinterpret_cast<R *>(static_cast<T *>(a.dx) + t * a.dim)[v] = d.raw;
        };
        if constexpr (LONG) {
            if (on)
                for (uint32_t v = lane; v < a.vectors; v += lanes) {
                    load(v, n[0], g[0]);
                    add(v, n[0], g[0]);
                }
        } else {
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (on && lane + i * lanes < a.vectors) load(lane + i * lanes, n[i], g[i]);
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (on && lane + i * lanes < a.vectors) add(lane + i * lanes, n[i], g[i]);
        }
        const float mean = row_sum(along, a.lane_log, room[turn & 1]) / static_cast<float>(a.dim);
        if (!on) continue;
        if constexpr (LONG) {
            for (uint32_t v = lane; v < a.vectors; v += lanes) {
                float *mine = share + static_cast<uint64_t>(v) * V::N;
                load(v, n[0], g[0]);
#pragma unroll
                for (int e = 0; e < V::N; e++) sum[0][e] = turn && a.partial ? mine[e] : 0;
                finish(v, n[0], g[0], mean, sum[0]);
#pragma unroll
                for (int e = 0; e < V::N; e++)
                    if (a.partial) mine[e] = sum[0][e];
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; i++)
                if (lane + i * lanes < a.vectors) finish(lane + i * lanes, n[i], g[i], mean, sum[i]);
        }
    }
    if (LONG || !a.partial) return;
#pragma unroll
    for (int i = 0; i < NV; i++)
        if (lane + i * lanes < a.vectors)
#pragma unroll
            for (int e = 0; e < V::N; e++) share[(lane + i * lanes) * V::N + e] = sum[i][e];
}

// out[d] = the sum of `rows` shares.  A block has 32 columns; its warps take the shares in turn, and their sums meet in their order.
constexpr uint32_t JOIN_WARPS = 16;
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
        for (uint64_t r = warp; r < rows; r += JOIN_WARPS) sum += partial[r * dim + d];
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp || d >= dim) return;
    for (uint32_t w = 1; w < JOIN_WARPS; w++) sum += sums[w][lane];
    out[d] = narrow<W>(sum);
}

}  // namespace lmz
