// What stands behind a product's sums, forwards and backwards:  z = sums + bias,  y = act(z) times + residual.
#pragma once
#include <type_traits>

#include "tcgen.cuh"
#include "vectors.cuh"

namespace lmz {

enum Activation : uint32_t { ACT_NONE, ACT_RELU, ACT_SILU, ACT_GELU, ACT_GELU_TANH, ACT_COUNT };

constexpr float ROOT_1_2PI = 0.39894228f, LOG2_E = 1.44269504f, TANH_CUBE = 0.044715f, TANH_TWICE = 1.59576912f;     // (the last: twice the root of 2 / pi)

// The tensor pipe's neighbours: powers of two and reciprocals as the special function unit has them, some 2^-22 of their result off; what is below 2^-126 is zero.
__device__ __forceinline__ float power_of_two(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float reciprocal(float v) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }

// The exponential goes by its root and its square is taken, so that it reaches as far as results of 16 bits do, whose smallest are e^-97: it is off by some 2^-21
// of itself and two to five times 2^-24 for each unit of its argument, under 2^-15 everywhere, where half a step of F16 is 2^-11.
//
// 1 / (1 + exp(-v)), good to its own size on both sides (numerator and denominator 2^-64 times what they are: the exponential has room).
__device__ __forceinline__ float sigmoid(float v)
{
    const float h = power_of_two(v * (-0.5f * LOG2_E)) * 0x1p-32f;
    return reciprocal(fmaf(h, h, 0x1p-64f)) * 0x1p-64f;
}

// The normal distribution's integral up to v, good to its own size (1 + erf cancels below zero: at -5 it is off by 4 %), and its density's exponential. For v < 0 it
// is exp(-v^2 / 2) P(-v), where P falls slowly from 1/2 like 0.4 / t: a polynomial in s = 1 / (1 + 0.3 t) without a constant, of the least relative error on
// [0, 14.6] (2^-22.5; 2^-21 with its roundings; found by reweighted least squares), behind which the exponential is zero.
__device__ __forceinline__ float normal_below(float v, float &bell)
{
    const float t = fabsf(v), s = reciprocal(fmaf(0.3f, t, 1)), h = power_of_two(t * (t * (-0.25f * LOG2_E)));
    float p = 0.0353742f;
    p = fmaf(p, s, -0.15595277f), p = fmaf(p, s, 0.20420392f), p = fmaf(p, s, -0.05171105f), p = fmaf(p, s, 0.12752213f);
    p = fmaf(p, s, 0.100226894f), p = fmaf(p, s, 0.12070406f), p = fmaf(p, s, 0.11963253f);
    const float tail = h * (p * s) * h;
    bell = h * h;
    return v < 0 ? tail : 1 - tail;
}

__device__ __forceinline__ float act(uint32_t kind, float z)
{
    float bell;
    switch (kind) {
    case ACT_RELU: return z < 0 ? 0.0f : z;                      // (a NaN stays)
    case ACT_SILU: return z * sigmoid(z);
    case ACT_GELU: return z * normal_below(z, bell);
    case ACT_GELU_TANH: return z * sigmoid(TANH_TWICE * (z + TANH_CUBE * z * z * z));     // ((1 + tanh u) / 2 is the sigmoid of 2 u)
    default: return z;
    }
}

// N of them: the kind is asked for once.
template <int N>
__device__ __forceinline__ void act_all(uint32_t kind, float *v)
{
    auto each = [&](auto k) {
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = act(decltype(k)::value, v[e]);
    };
    switch (kind) {
    case ACT_RELU: return each(std::integral_constant<uint32_t, ACT_RELU>{});
    case ACT_SILU: return each(std::integral_constant<uint32_t, ACT_SILU>{});
    case ACT_GELU: return each(std::integral_constant<uint32_t, ACT_GELU>{});
    case ACT_GELU_TANH: return each(std::integral_constant<uint32_t, ACT_GELU_TANH>{});
    }
}

// N activations and their derivatives.
template <int N>
__device__ __forceinline__ void act_and_slope(uint32_t kind, const float *z, float *y, float *slope)
{
    auto each = [&](auto f) {
#pragma unroll
        for (int e = 0; e < N; e++) f(z[e], y[e], slope[e]);
    };
    switch (kind) {
    case ACT_RELU: return each([](float z, float &y, float &slope) { y = z < 0 ? 0.0f : z, slope = z > 0 ? 1.0f : 0.0f; });
    case ACT_SILU:
        return each([](float z, float &y, float &slope) {
            const float below = sigmoid(z);
            y = z * below, slope = fmaf(y, 1 - below, below);
        });
    case ACT_GELU:
        return each([](float z, float &y, float &slope) {
            float bell;
            const float below = normal_below(z, bell);
            y = z * below, slope = fmaf(z * ROOT_1_2PI, bell, below);
        });
    case ACT_GELU_TANH:
        return each([](float z, float &y, float &slope) {
            const float below = sigmoid(TANH_TWICE * (z + TANH_CUBE * z * z * z));
            y = z * below;
            const float near = fminf(fmaxf(z, -16.0f), 16.0f);   // (beyond, below or 1 - below is zero, and z or its square may be infinite)
            slope = fmaf(near * below * (1 - below), TANH_TWICE * (1 + 3 * TANH_CUBE * near * near), below);
        });
    default: return each([](float z, float &y, float &slope) { y = z, slope = 1; });
    }
}

// Which rows an expert has: offsets that ascend, 32 or 64 bits each, kept within the rows there are.
struct Groups {
    const void *offsets;                         // NULL: one, of all rows
    uint32_t count;
    bool wide;
    uint64_t rows;
    __device__ __forceinline__ uint64_t at(uint32_t i) const
    {
        if (!offsets) return i ? rows : 0;
        const int64_t v = wide ? static_cast<const int64_t *>(offsets)[i] : static_cast<const int32_t *>(offsets)[i];
        return v < 0 ? 0 : static_cast<uint64_t>(v) < rows ? static_cast<uint64_t>(v) : rows;
    }
};

// Where each group's rows begin, count + 1 of them in shared memory: the offsets, none below one before it (so that no row has two groups
// whatever they are).  By the block's first warp; the caller's barrier follows.
__device__ __forceinline__ void group_starts(const Groups &g, uint32_t *starts)
{
    if (threadIdx.x >= 32) return;
    uint32_t most = 0;
    for (uint32_t i0 = 0; i0 <= g.count; i0 += 32) {
        const uint32_t i = i0 + threadIdx.x;
        uint32_t v = i <= g.count ? static_cast<uint32_t>(g.at(i)) : 0;
#pragma unroll
        for (uint32_t o = 1; o < 32; o <<= 1) {
            const uint32_t below = __shfl_up_sync(~0u, v, o);
            if (threadIdx.x >= o) v = max(v, below);
        }
        v = max(v, most);
        if (i <= g.count) starts[i] = v;
        most = __shfl_sync(~0u, v, 31);
    }
}

// Of count + 1 ascending starts the last group whose start is not above `row` (empty groups before it are passed over).
__device__ __forceinline__ uint32_t group_of(const uint32_t *starts, uint32_t count, uint32_t row)
{
    uint32_t lo = 0, hi = count;                                 // starts[lo] <= row < starts[hi], or an end
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (starts[mid] <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

constexpr uint32_t MAX_EXPERTS = 1024;
constexpr uint32_t EG_THREADS = 128, EG_MOST_ROWS = 32, EG_LEAST_ROWS = 4, EG_STEP = 2;     // rows of a chunk, and of those under way together

// F16 has few powers of two: dz may leave it where dx and dW do not.  So dz is written times a power of two, its group's own, which the products' sums are divided by.
// USUAL_POWER is right where the group's largest (finite) element is between 4 and 255, so that an element that is less than half a step of F16 is under 2^-34 of that;
// other groups are written once more, their largest brought to 2^14 and more.
constexpr int USUAL_POWER = 8;
__device__ __forceinline__ int dz_power(uint32_t most)           // `most`: its bits
{
    if (most == 0 || (most >= 0x40800000u && most <= 0x437FE000u)) return USUAL_POWER;
    const int power = 14 - (static_cast<int>(most >> 23) - 127);
    return power < 100 ? power : 100;
}
__device__ __forceinline__ float two_to(int power) { return __int_as_float((127 + power) << 23); }

struct EpilogueGradArgs {
    const void *dy, *times;                      // times: or NULL, rows times_stride apart
    const float *z;                              // NULL where neither the slope nor dtimes goes by it
    void *dz, *dtimes;                           // or NULL
    float *partial;                              // [chunk of rows + group][out]: sums of dz, or NULL
    uint32_t *most;                              // [group]: bits of the largest finite dz, zeros before; or NULL: dz is written as it is
    Groups groups;
    uint64_t rows, out, times_stride, dz_stride;
    uint32_t vectors, activation, chunk;         // chunk: rows
};

template <int N>
__device__ __forceinline__ void load_floats(const float *from, float *to)
{
    constexpr int B = N * 4 < 16 ? N * 4 : 16;
#pragma unroll
    for (int i = 0; i < N * 4 / B; i++) reinterpret_cast<typename Raw<B>::type *>(to)[i] = reinterpret_cast<const typename Raw<B>::type *>(from)[i];
}

// dz = dy times act'(z), dtimes = dy act(z), and what each chunk of rows adds to the gradient of its groups' bias: a chunk and a group that
// meet have the place chunk + group, which no other two have.  Rows of no group get zeros.
//
// dz is rounded to the tensors' type: the tensor core's operands are of one type, and a second part for what is cut off would double the products that dominate a step. It
// costs the gradients of x and W a third more error than a dz in 32 bits (BF16 2.3e-3 for 1.7e-3, F16 2.9e-4 for 2.1e-4); the bias's and the factor's do without it.
// z comes in 32 bits: a factor's gradient is z or its activation times dy, rounded once.
// Bound by HBM.  A thread has a vector of columns and goes down a chunk's rows, EG_STEP under way at a time (four cost the threads that an SM has: 380 us and
// not 228).  One B200, 8192x14336 BF16, silu and a factor: 215 to 228 us (6.2 TB/s and more), the
// factor's gradient alone 187.
template <class T, int VB>
__global__ void __launch_bounds__(EG_THREADS) k_epilogue_grad(const EpilogueGradArgs a)
{
    using V = Vec<T, VB>;
    using R = typename Raw<VB>::type;
    __shared__ uint32_t starts[MAX_EXPERTS + 1];
    wait_for_previous();
    let_next_start();
    group_starts(a.groups, starts);
    __syncthreads();
    const uint64_t v = blockIdx.y * static_cast<uint64_t>(EG_THREADS) + threadIdx.x;
    const uint32_t together = __ballot_sync(~0u, v < a.vectors);
    const uint32_t chunk = blockIdx.x, begin = chunk * a.chunk, end = begin + a.chunk < a.rows ? begin + a.chunk : static_cast<uint32_t>(a.rows);
    if (v >= a.vectors) return;
    const uint32_t first = starts[0], last = starts[a.groups.count];
    uint32_t group = group_of(starts, a.groups.count, begin < first ? first : begin);
    float sum[V::N];
#pragma unroll
    for (int e = 0; e < V::N; e++) sum[e] = 0;
    bool any = false;
    constexpr bool HALF = __is_same(T, __half);
    uint32_t most = 0;
    auto flush = [&] {
        if (HALF && a.most) {                                    // (the same groups for all of a warp)
            most = __reduce_max_sync(together, most);
            if ((threadIdx.x & 31) == 0 && most > *const_cast<volatile uint32_t *>(a.most + group)) atomicMax(a.most + group, most);
            most = 0;
        }
        if (a.partial && any) {
            float *to = a.partial + (static_cast<uint64_t>(chunk) + group) * a.out + v * V::N;
#pragma unroll
            for (int e = 0; e < V::N; e++) to[e] = sum[e];
        }
#pragma unroll
        for (int e = 0; e < V::N; e++) sum[e] = 0;
        any = false;
    };
    for (uint32_t t0 = begin; t0 < end; t0 += EG_STEP) {
        V d[EG_STEP], m[EG_STEP];
        alignas(16) float z[EG_STEP][V::N];
#pragma unroll
        for (uint32_t i = 0; i < EG_STEP; i++) {
            const uint32_t t = t0 + i;
            d[i].raw = m[i].raw = {};
#pragma unroll
            for (int e = 0; e < V::N; e++) z[i][e] = 0;
            if (t >= end || t < first || t >= last) continue;
            d[i].raw = reinterpret_cast<const R *>(static_cast<const T *>(a.dy) + t * a.out)[v];
            if (a.z) load_floats<V::N>(a.z + t * a.out + v * V::N, z[i]);
            if (a.times) m[i].raw = reinterpret_cast<const R *>(static_cast<const T *>(a.times) + t * a.times_stride)[v];
        }
#pragma unroll
        for (uint32_t i = 0; i < EG_STEP; i++) {
            const uint32_t t = t0 + i;
            if (t >= end) break;
            V dz, dm;
            dz.raw = dm.raw = {};
            if (t >= first && t < last) {
                if (t >= starts[group + 1]) {
                    flush();
                    group = group_of(starts, a.groups.count, t);
                }
                float y[V::N], u[V::N];
                act_and_slope<V::N>(a.activation, z[i], y, u);
                float g[V::N];
                widen_all(d[i], g);
#pragma unroll
                for (int e = 0; e < V::N; e++) y[e] *= g[e], u[e] *= g[e];
                narrow_all(y, dm);
                if (a.times) {
                    widen_all(m[i], g);
#pragma unroll
                    for (int e = 0; e < V::N; e++) u[e] *= g[e];
                }
#pragma unroll
                for (int e = 0; e < V::N; e++) sum[e] += u[e];
                if (HALF && a.most) {
#pragma unroll
                    for (int e = 0; e < V::N; e++) {
                        const uint32_t size = __float_as_uint(u[e]) & 0x7FFFFFFF;
                        if (size < 0x7F800000) most = max(most, size);
                        u[e] *= two_to(USUAL_POWER);
                    }
                }
                narrow_all(u, dz);
                any = true;
            }
            if (a.dz) reinterpret_cast<R *>(static_cast<T *>(a.dz) + t * a.dz_stride)[v] = dz.raw;
            if (a.dtimes) reinterpret_cast<R *>(static_cast<T *>(a.dtimes) + t * a.out)[v] = dm.raw;
        }
    }
    flush();
}

// dz again, of the groups whose power is not the usual one.  Bound by HBM as the first time, where there are such; else by the launch.
template <class T, int VB>
__global__ void __launch_bounds__(EG_THREADS) k_dz_again(const EpilogueGradArgs a)
{
    using V = Vec<T, VB>;
    using R = typename Raw<VB>::type;
    __shared__ uint32_t starts[MAX_EXPERTS + 1];
    wait_for_previous();
    let_next_start();
    group_starts(a.groups, starts);
    __syncthreads();
    const uint64_t v = blockIdx.y * static_cast<uint64_t>(EG_THREADS) + threadIdx.x;
    if (v >= a.vectors) return;
    const uint32_t begin = blockIdx.x * a.chunk, last = starts[a.groups.count];
    const uint32_t end = begin + a.chunk < last ? begin + a.chunk : last;
    for (uint32_t t = begin < starts[0] ? starts[0] : begin; t < end;) {
        const uint32_t group = group_of(starts, a.groups.count, t), stop = starts[group + 1] < end ? starts[group + 1] : end;
        const int power = dz_power(a.most[group]);
        for (; power != USUAL_POWER && t < stop; t++) {
            V d, m;
            float z[V::N], y[V::N], u[V::N], g[V::N];
            d.raw = reinterpret_cast<const R *>(static_cast<const T *>(a.dy) + t * a.out)[v];
            if (a.times) m.raw = reinterpret_cast<const R *>(static_cast<const T *>(a.times) + t * a.times_stride)[v];
#pragma unroll
            for (int e = 0; e < V::N; e++) z[e] = 0;
            if (a.z) load_floats<V::N>(a.z + t * a.out + v * V::N, z);
            act_and_slope<V::N>(a.activation, z, y, u);
            widen_all(d, g);
#pragma unroll
            for (int e = 0; e < V::N; e++) u[e] *= g[e];
            if (a.times) {
                widen_all(m, g);
#pragma unroll
                for (int e = 0; e < V::N; e++) u[e] *= g[e];
            }
#pragma unroll
            for (int e = 0; e < V::N; e++) u[e] *= two_to(power);
            narrow_all(u, d);
            reinterpret_cast<R *>(static_cast<T *>(a.dz) + t * a.dz_stride)[v] = d.raw;
        }
        t = stop;
    }
}

// A group's bias gradient: what the chunks that its rows lie in have for it; a block's warps take them in turn, and their sums meet in their order.
constexpr uint32_t BJ_WARPS = 16, BJ_AHEAD = 8;
template <class T>
__global__ void __launch_bounds__(32 * BJ_WARPS) k_bias_join(const float *partial, Groups groups, uint64_t out, uint32_t chunk, T *dbias)
{
    __shared__ uint32_t starts[MAX_EXPERTS + 1];
    __shared__ float sums[BJ_WARPS][32];
    wait_for_previous();
    let_next_start();
    group_starts(groups, starts);
    __syncthreads();
    const uint32_t g = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t d = blockIdx.x * 32ull + lane;
    float sum = 0;
    if (starts[g + 1] > starts[g] && d < out) {
        const uint32_t end = (starts[g + 1] - 1) / chunk + 1;
        for (uint32_t c = starts[g] / chunk + warp; c < end; c += BJ_WARPS * BJ_AHEAD) {
            float v[BJ_AHEAD];
#pragma unroll
            for (uint32_t i = 0; i < BJ_AHEAD; i++) v[i] = c + i * BJ_WARPS < end ? partial[(static_cast<uint64_t>(c) + i * BJ_WARPS + g) * out + d] : 0;
#pragma unroll
            for (uint32_t i = 0; i < BJ_AHEAD; i++) sum += v[i];
        }
    }
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp || d >= out) return;
    for (uint32_t w = 1; w < BJ_WARPS; w++) sum += sums[w][lane];
    dbias[g * out + d] = narrow<T>(sum);
}

}  // namespace lmz
