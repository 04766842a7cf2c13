// An adapter in FP32 merged into its weight.
#pragma once
#include "tcgen.cuh"
#include "vectors.cuh"

namespace lmz {

constexpr uint32_t MW_TILE = 128, MW_STEP = 16, MW_THREADS = 256;
constexpr uint32_t MW_PITCH = MW_TILE + 4;     // of B's rows in shared memory: two of a warp's sixteen places of the rank to a bank

template <class T>
struct MergeWideArgs {
    const T *w;
    const float *a, *b;
    T *out;
    uint64_t rows, cols, w_stride;
    uint32_t rank;
    float scale;
};

// W' = W + s B A with factors in FP32, which the tensor core would take with fewer bits: on the CUDA cores, a tile of 128 x 128 a
// block and 8 x 8 of it a thread, sixteen places of the rank at a time (eight: 315 us).  FOUR: rows of W and W' start on four elements.
// Bound by the multiplications: one B200, 14336 x 4096 at rank 64 246 us in FP32 and 238 in BF16 (31 TFLOP/s), at rank 16, where the
// weight's bytes count as much, 108 and 99; with a load of W behind each store 281 and 287, 178 and 176.
template <class T, bool FOUR>
__global__ void __launch_bounds__(MW_THREADS, 2) k_merge_wide(const MergeWideArgs<T> m)
{
    using V = Vec<T, 4 * sizeof(T)>;
    using Raws = typename Raw<4 * sizeof(T)>::type;
    __shared__ __align__(16) float a[2][MW_STEP][MW_TILE], b[2][MW_STEP][MW_PITCH];
    constexpr uint32_t LOADS = MW_STEP * MW_TILE / MW_THREADS;
    const uint32_t tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
    const uint64_t across = (m.cols + MW_TILE - 1) / MW_TILE, r0 = blockIdx.x / across * MW_TILE, c0 = blockIdx.x % across * MW_TILE;
    float sum[8][8] = {}, next_a[LOADS], next_b[LOADS];
    wait_for_previous();
    auto load = [&](uint32_t j0) {
#pragma unroll
        for (uint32_t i = 0; i < LOADS; i++) {
            const uint32_t e = i * MW_THREADS + tid, ja = j0 + e / MW_TILE, jb = j0 + e % MW_STEP;
            const uint64_t c = c0 + e % MW_TILE, r = r0 + e / MW_STEP;
            next_a[i] = ja < m.rank && c < m.cols ? m.a[ja * m.cols + c] : 0.0f;
            next_b[i] = jb < m.rank && r < m.rows ? m.b[r * m.rank + jb] : 0.0f;
        }
    };
    auto keep = [&](uint32_t side) {
#pragma unroll
        for (uint32_t i = 0; i < LOADS; i++) {
            const uint32_t e = i * MW_THREADS + tid;
            a[side][e / MW_TILE][e % MW_TILE] = next_a[i];
            b[side][e % MW_STEP][e / MW_STEP] = next_b[i];
        }
    };
    load(0);
    keep(0);
    __syncthreads();
    for (uint32_t j0 = 0, side = 0; j0 < m.rank; j0 += MW_STEP, side ^= 1) {
        const bool more = j0 + MW_STEP < m.rank;
        if (more) load(j0 + MW_STEP);
#pragma unroll
        for (uint32_t j = 0; j < MW_STEP; j++) {
            float p[8], q[8];
#pragma unroll
            for (uint32_t h = 0; h < 2; h++) {
                *reinterpret_cast<float4 *>(p + 4 * h) = *reinterpret_cast<const float4 *>(&b[side][j][h * 64 + ty * 4]);
                *reinterpret_cast<float4 *>(q + 4 * h) = *reinterpret_cast<const float4 *>(&a[side][j][h * 64 + tx * 4]);
            }
#pragma unroll
            for (uint32_t x = 0; x < 8; x++)
#pragma unroll
                for (uint32_t y = 0; y < 8; y++) sum[x][y] = fmaf(p[x], q[y], sum[x][y]);
        }
        if (more) {                                              // (the other side was read before the last barrier)
            keep(side ^ 1);
            __syncthreads();
        }
    }
    // W's elements of four rows at a time, all on their way together (W' may be W: no load would pass a store).
#pragma unroll
    for (uint32_t half = 0; half < 2; half++) {
        V v[4][2];
        auto each = [&](auto f) {
#pragma unroll
            for (uint32_t x = 0; x < 4; x++)
#pragma unroll
                for (uint32_t h = 0; h < 2; h++) {
                    const uint64_t r = r0 + half * 64 + ty * 4 + x, c = c0 + h * 64 + tx * 4;
                    if (r < m.rows && c < m.cols) f(v[x][h], sum[half * 4 + x] + h * 4, r, c);
                }
        };
        each([&](V &w, float *, uint64_t r, uint64_t c) {
            const T *from = m.w + r * m.w_stride + c;
            if constexpr (FOUR) {
                w.raw = *reinterpret_cast<const Raws *>(from);
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 4; e++)
                    if (c + e < m.cols) w.e[e] = from[e];
            }
        });
        each([&](V &w, float *s, uint64_t r, uint64_t c) {
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) w.e[e] = narrow<T>(fmaf(m.scale, s[e], widen(w.e[e])));
            T *to = m.out + r * m.cols + c;
            if constexpr (FOUR) {
                *reinterpret_cast<Raws *>(to) = w.raw;
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 4; e++)
                    if (c + e < m.cols) to[e] = w.e[e];
            }
        });
    }
}

}  // namespace lmz
