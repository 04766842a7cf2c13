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

// Thin products are kept as two halves of 16 bits, [token][2][rp] with rp the rank up to a multiple of 8: a value to the
// nearest T, and what that lacks.  One T alone would cost as much as the result's own rounding.
template <class T>
__device__ __forceinline__ void split_halves(float v, T &hi, T &lo)
{
    hi = narrow<T>(v);
    lo = narrow<T>(isfinite(widen(hi)) ? v - widen(hi) : 0.0f);
}

// h[t][j] = s_i * sum over k of x[t][k] F_i(k, j): a warp each.
template <class T>
__global__ void __launch_bounds__(256) k_hidden(const T *x, uint64_t stride, uint64_t k, Factor<T> f, TokenIndex index, uint64_t tokens,
                                                uint32_t rank, uint32_t rp, T *h)
{
    const uint64_t at = static_cast<uint64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5), t = at / rp;
    const uint32_t j = static_cast<uint32_t>(at % rp), lane = threadIdx.x & 31;
    if (t >= tokens) return;
    const int i = index.of(t);
    float sum = 0;
    if (i >= 0 && j < rank)
        for (uint64_t c = lane; c < k; c += 32) sum += widen(x[t * stride + c]) * widen(f.at(i, c, j));
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) split_halves(i >= 0 && j < rank ? sum * index.scale_of(i) : 0.0f, h[t * 2 * rp + j], h[t * 2 * rp + rp + j]);
}

// A copy whose rows start on a boundary of 16 bytes and end in zeros: out[o][r][c] = in(o, r, c) for r < rows, c < cols, else 0.
template <class T>
__global__ void __launch_bounds__(256) k_pack(const T *in, uint64_t so, uint64_t sr, uint64_t sc, uint64_t rows, uint64_t cols, uint64_t pitch, uint64_t total, T *out)
{
    for (uint64_t e = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; e < total; e += static_cast<uint64_t>(gridDim.x) * 256) {
        const uint64_t c = e % pitch, q = e / pitch, r = q % rows, o = q / rows;
        out[e] = c < cols ? in[o * so + r * sr + c * sc] : narrow<T>(0.0f);
    }
}

// dF_i(f, j) = sum over i's tokens of g[t][j] z[t][f].
template <class T>
__global__ void __launch_bounds__(256) k_factor_grad(const T *g, uint32_t rp, const T *z, uint64_t stride, TokenIndex index, uint64_t tokens, uint32_t rank,
                                                     uint64_t feats, T *out, uint64_t each, uint64_t wide, uint64_t place)
{
    const uint64_t f = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    const uint32_t j = blockIdx.y, i = blockIdx.z;
    if (f >= feats) return;
    float sum = 0;
    for (uint64_t t = 0; t < tokens; t++)
        if (index.of(t) == static_cast<int>(i)) sum += (widen(g[t * 2 * rp + j]) + widen(g[t * 2 * rp + rp + j])) * widen(z[t * stride + f]);
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
