// Products of rows with a weight, or with their experts' weights, their epilogue, and both gradients.
#pragma once
#include <cuda_fp8.h>

#include "epilogue.cuh"
#include "tcgen.cuh"

namespace lmz {

__device__ __forceinline__ float widen(__nv_fp8_e4m3 v) { return static_cast<float>(v); }

// out[c][f] = sum over k of A(f, k) B(c, k), the three that a layer has:
//   forwards         f: the output's features, c: rows,                  k: the input's; A is the weight, B is x
//   rows' gradient   f: the input's features,  c: rows,                  k: the output's; A is the weight (k by k), B is dz
//   weight's         f: the input's features,  c: the output's features, k: rows; A is x, B is dz (both k by k)
// A group is an expert: in the first two its rows are some of c, in the last they are its k.
template <class T>
struct ProductArgs {
    const T *a, *b;
    void *out;
    float *z;
    const void *bias, *times, *residual;
    const float *a_scale, *b_scale;              // of 8-bit features and rows, or NULL
    Groups groups;
    uint64_t feats, cols, depth;                 // of f, c and k (those of c, or of k, in all groups)
    uint64_t a_f, a_k, b_c, b_k, a_plane, times_stride, residual_stride;
    uint32_t activation;
    bool by_k;                                   // groups are of k
};

constexpr uint32_t S_TILE = 64, S_K = 16, S_THREADS = 256;

template <class T, class O>
__global__ void __launch_bounds__(S_THREADS) k_product(const ProductArgs<T> a)
{
    __shared__ float as[S_K][S_TILE + 1], bs[S_K][S_TILE + 1];
    __shared__ uint32_t starts[MAX_EXPERTS + 1];
    wait_for_previous();
    group_starts(a.groups, starts);
    __syncthreads();
    const uint32_t tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
    const uint64_t f0 = static_cast<uint64_t>(blockIdx.x) * S_TILE;
    for (uint32_t g = blockIdx.z; g < a.groups.count; g += gridDim.z) {
        const uint64_t c_lo = a.by_k ? 0 : starts[g], c_hi = a.by_k ? a.cols : starts[g + 1];
        const uint64_t k_lo = a.by_k ? starts[g] : 0, k_hi = a.by_k ? starts[g + 1] : a.depth;
        for (uint64_t c0 = c_lo + static_cast<uint64_t>(blockIdx.y) * S_TILE; c0 < c_hi; c0 += static_cast<uint64_t>(gridDim.y) * S_TILE) {
            float sum[4][4] = {};
            for (uint64_t k0 = k_lo; k0 < k_hi; k0 += S_K) {
                __syncthreads();
                for (uint32_t i = tid; i < S_K * S_TILE; i += S_THREADS) {
                    const uint32_t r = a.a_k == 1 ? i / S_K : i % S_TILE, k = a.a_k == 1 ? i % S_K : i / S_TILE;
                    as[k][r] = f0 + r < a.feats && k0 + k < k_hi ? widen(a.a[(a.by_k ? 0 : g * a.a_plane) + (f0 + r) * a.a_f + (k0 + k) * a.a_k]) : 0;
                    const uint32_t c = a.b_k == 1 ? i / S_K : i % S_TILE, j = a.b_k == 1 ? i % S_K : i / S_TILE;
                    bs[j][c] = c0 + c < c_hi && k0 + j < k_hi ? widen(a.b[(c0 + c) * a.b_c + (k0 + j) * a.b_k]) : 0;
                }
                __syncthreads();
#pragma unroll
                for (uint32_t k = 0; k < S_K; k++)
#pragma unroll
                    for (uint32_t i = 0; i < 4; i++)
#pragma unroll
                        for (uint32_t j = 0; j < 4; j++) sum[i][j] += bs[k][ty + i * 16] * as[k][tx + j * 16];
            }
            for (uint32_t i = 0; i < 4; i++)
                for (uint32_t j = 0; j < 4; j++) {
                    const uint64_t c = c0 + ty + i * 16, f = f0 + tx + j * 16, at = ((a.by_k ? g * a.cols : 0) + c) * a.feats + f;
                    if (c >= c_hi || f >= a.feats) continue;
                    float z = sum[i][j];
                    if (a.a_scale) z *= a.a_scale[f] * a.b_scale[c];
                    if (a.bias) z += widen(static_cast<const O *>(a.bias)[g * a.feats + f]);
                    if (a.z) a.z[at] = z;
                    float y = act(a.activation, z);
                    if (a.times) y *= widen(static_cast<const O *>(a.times)[c * a.times_stride + f]);
                    if (a.residual) y += widen(static_cast<const O *>(a.residual)[c * a.residual_stride + f]);
                    static_cast<O *>(a.out)[at] = narrow<O>(y);
                }
        }
    }
    if (a.by_k) return;
    const uint64_t first = starts[0], last = starts[a.groups.count], idle = first + (a.cols - last);          // rows of no group
    const uint64_t block = (static_cast<uint64_t>(blockIdx.z) * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
    const uint64_t blocks = static_cast<uint64_t>(gridDim.x) * gridDim.y * gridDim.z;
    for (uint64_t i = block * S_THREADS + tid; i < idle * a.feats; i += blocks * S_THREADS) {
        const uint64_t r = i / a.feats, c = r < first ? r : last + (r - first);
        static_cast<O *>(a.out)[c * a.feats + i % a.feats] = narrow<O>(0.0f);
    }
}

}  // namespace lmz
