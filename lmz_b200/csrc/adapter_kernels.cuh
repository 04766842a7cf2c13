// A projection through a shared weight with low-rank adapters of many requests beside it, its gradients, and the merge
// of an adapter into a weight.
//
//   y[t] = x[t] W^T + h[t] B_i^T,  h[t] = s_i x[t] A_i^T,  i = index[t];  no adapter where index[t] is outside [0, n)
//   g[t] = s_i dy[t] B_i,  dx[t] = dy[t] W + g[t] A_i,  dA_i = sum of g[t]^T x[t],  dB_i = sum of dy[t]^T h[t] over i's tokens
#pragma once
#include "vectors.cuh"

namespace lmz {

// Which adapter a token has.
struct TokenIndex {
    const void *ids;            // int32 or int64; NULL: every token has adapter 0
    const float *scales;        // per adapter, or NULL
    float scale;
    uint32_t n;
    bool wide;
    __device__ __forceinline__ int of(uint64_t t) const
    {
        if (!ids) return 0;
        const int64_t i = wide ? static_cast<const int64_t *>(ids)[t] : static_cast<const int32_t *>(ids)[t];
        return i >= 0 && i < n ? static_cast<int>(i) : -1;
    }
    __device__ __forceinline__ float scale_of(int i) const { return scales ? scale * scales[i] : scale; }
};

// Elements of adapter i's factor by (its wide coordinate, its place in the rank).
template <class T>
struct Factor {
    const T *p;
    uint64_t each, wide, place;
    __device__ __forceinline__ T at(int i, uint64_t f, uint32_t j) const { return p[i * each + f * wide + j * place]; }
};

// h[t][j] = s_i * sum over k of x[t][k] F_i(k, j): a warp each.
template <class T>
__global__ void __launch_bounds__(256) k_hidden(const T *x, uint64_t stride, uint64_t k, Factor<T> f, TokenIndex index, uint64_t tokens,
                                                uint32_t rank, float *h)
{
    const uint64_t at = static_cast<uint64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5), t = at / rank;
    const uint32_t j = static_cast<uint32_t>(at % rank), lane = threadIdx.x & 31;
    if (t >= tokens) return;
    const int i = index.of(t);
    float sum = 0;
    if (i >= 0)
        for (uint64_t c = lane; c < k; c += 32) sum += widen(x[t * stride + c]) * widen(f.at(i, c, j));
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) h[at] = i >= 0 ? sum * index.scale_of(i) : 0.0f;
}

// y[t][f] = sum over k of x[t][k] W(f, k) + sum over j of h[t][j] F_i(f, j): tiles of 64 by 64.
template <class T>
__global__ void __launch_bounds__(256) k_project(const T *x, uint64_t stride, uint64_t k, const T *w, uint64_t wf, uint64_t wk, Factor<T> fac,
                                                 TokenIndex index, const float *h, uint32_t rank, uint64_t tokens, uint64_t feats, T *y)
{
    __shared__ float xs[16][65], ws[16][65];
    const uint64_t t0 = static_cast<uint64_t>(blockIdx.x) * 64, f0 = static_cast<uint64_t>(blockIdx.y) * 64;
    const uint32_t tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (uint64_t k0 = 0; k0 < k; k0 += 16) {
        for (uint32_t e = threadIdx.x; e < 64 * 16; e += 256) {
            const uint32_t r = e >> 4, c = e & 15;
            xs[c][r] = t0 + r < tokens && k0 + c < k ? widen(x[(t0 + r) * stride + k0 + c]) : 0.0f;
            ws[c][r] = f0 + r < feats && k0 + c < k ? widen(w[(f0 + r) * wf + (k0 + c) * wk]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t c = 0; c < 16; c++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] += xs[c][ty + 16 * i] * ws[c][tx + 16 * j];
        __syncthreads();
    }
    for (int i = 0; i < 4; i++) {
        const uint64_t t = t0 + ty + 16 * i;
        if (t >= tokens) continue;
        const int ad = index.of(t);
        for (int j = 0; j < 4; j++) {
            const uint64_t f = f0 + tx + 16 * j;
            if (f >= feats) continue;
            float sum = acc[i][j];
            if (ad >= 0)
                for (uint32_t c = 0; c < rank; c++) sum += h[t * rank + c] * widen(fac.at(ad, f, c));
            y[t * feats + f] = narrow<T>(sum);
        }
    }
}

// dF_i(f, j) = sum over i's tokens of g[t][j] z[t][f].
template <class T>
__global__ void __launch_bounds__(256) k_factor_grad(const float *g, const T *z, uint64_t stride, TokenIndex index, uint64_t tokens, uint32_t rank,
                                                     uint64_t feats, T *out, uint64_t each, uint64_t wide, uint64_t place)
{
    const uint64_t f = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    const uint32_t j = blockIdx.y, i = blockIdx.z;
    if (f >= feats) return;
    float sum = 0;
    for (uint64_t t = 0; t < tokens; t++)
        if (index.of(t) == static_cast<int>(i)) sum += g[t * rank + j] * widen(z[t * stride + f]);
    out[i * each + f * wide + j * place] = narrow<T>(sum);
}

// W' = W + s B A.
template <class T>
__global__ void __launch_bounds__(256) k_merge(const T *w, uint64_t stride, const T *a, const T *b, uint32_t rank, float scale, uint64_t in, T *out)
{
    const uint64_t c = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x, r = blockIdx.y;
    if (c >= in) return;
    float sum = 0;
    for (uint32_t j = 0; j < rank; j++) sum += widen(b[r * rank + j]) * widen(a[j * in + c]);
    out[r * in + c] = narrow<T>(widen(w[r * stride + c]) + scale * sum);
}

}  // namespace lmz
