// An adapter merged into its weight.
#pragma once
#include "adapter_kernels.cuh"
#include "tcgen.cuh"

namespace lmz {

constexpr uint32_t M_ROWS = 128, M_COLS = 128, M_THREADS = 256;
constexpr uint32_t M_PITCH = M_COLS + 4;       // of the sums in shared memory, in words

template <class T>
struct MergeArgs {
    const T *w, *a, *b;
    T *out;
    uint64_t rows, cols, w_stride;
    uint32_t rank, places;                     // places: rank up to a multiple of 16
    float scale;
    bool a_even, b_even;                       // the factors' rows start on boundaries of 16 bytes
};

// Shared memory of a block: both factors' tiles, and over them the sums.
__host__ __device__ constexpr uint32_t merge_smem(uint32_t places)
{
    const uint32_t b = (places + STEP_K - 1) / STEP_K * M_ROWS * ROW_BYTES, a = M_COLS / 64 * places * ROW_BYTES, sums = M_ROWS * M_PITCH * 4;
    return (a + b > sums ? a + b : sums) + ATOM_BYTES;
}

// W' = W + s B A, a tile of 128 x 128 a block.
//
// Bound by HBM: W read and W' written once.  A thread has its part of W on the way into registers before the factors arrive
// (several blocks to an SM keep 128 KiB of it moving), the thin product is a few instructions of the tensor core, and its sums go
// through shared memory so that W and W' move in rows of whole lines: VB bytes a thread, 128 columns by half a warp.
template <class T, int VB>
__global__ void __launch_bounds__(M_THREADS) k_merge(const MergeArgs<T> a)
{
    using V = Vec<T, VB>;
    constexpr uint32_t PER_ROW = M_COLS / V::N, PARTS = M_ROWS * PER_ROW / M_THREADS;
    extern __shared__ uint8_t m_smem[];
    __shared__ uint64_t done;
    __shared__ uint32_t s_tmem, s_over;
    const uint32_t tid = threadIdx.x, warp = tid >> 5;
    const uint64_t r0 = static_cast<uint64_t>(blockIdx.y) * M_ROWS, c0 = static_cast<uint64_t>(blockIdx.x) * M_COLS;
    const uint32_t base = (smem_addr(m_smem) + ATOM_BYTES - 1) & ~(ATOM_BYTES - 1);
    uint8_t *local = m_smem + (base - smem_addr(m_smem));
    const uint32_t b_bytes = (a.places + STEP_K - 1) / STEP_K * M_ROWS * ROW_BYTES, block = a.places * ROW_BYTES;

    // B's rows, K-major; A's, MN-major in blocks of 64 columns
    for (uint32_t e = tid; e < M_ROWS * a.places / 8; e += M_THREADS) {
        const uint32_t row = e / (a.places / 8), c = e % (a.places / 8), j = c * 8;
        const uint32_t at = (c >> 3) * M_ROWS * ROW_BYTES + swizzled(row, c & 7);
        const T *p = a.b + (r0 + row) * a.rank + j;
        const bool on = r0 + row < a.rows;
        if (a.b_even) {
            copy16(base + at, on && j < a.rank ? p : a.b, on && j < a.rank);
        } else {
            Vec<T, 16> v;
            v.raw = {};
#pragma unroll
            for (uint32_t q = 0; q < 8; q++)
                if (on && j + q < a.rank) v.e[q] = p[q];
            *reinterpret_cast<uint4 *>(local + at) = v.raw;
        }
    }
    for (uint32_t e = tid; e < a.places * (M_COLS / 8); e += M_THREADS) {
        const uint32_t j = e / (M_COLS / 8), c = e % (M_COLS / 8);
        const uint32_t at = b_bytes + (c >> 3) * block + swizzled(j, c & 7);
        const uint64_t col = c0 + c * 8;
        const T *p = a.a + j * a.cols + col;
        if (a.a_even) {
            const bool on = j < a.rank && col < a.cols;
            copy16(base + at, on ? p : a.a, on);
        } else {
            Vec<T, 16> v;
            v.raw = {};
#pragma unroll
            for (uint32_t q = 0; q < 8; q++)
                if (j < a.rank && col + q < a.cols) v.e[q] = p[q];
            *reinterpret_cast<uint4 *>(local + at) = v.raw;
        }
    }
    copies_commit();
    V w[VB == 16 ? PARTS : 1];
    if constexpr (VB == 16) {
#pragma unroll
        for (uint32_t i = 0; i < PARTS; i++) {
            const uint32_t e = i * M_THREADS + tid, row = e / PER_ROW;
            const uint64_t col = c0 + e % PER_ROW * V::N;
            w[i].raw = {};
            if (r0 + row < a.rows && col < a.cols)
                w[i].raw = *reinterpret_cast<const typename Raw<VB>::type *>(a.w + (r0 + row) * a.w_stride + col);
        }
    }
    if (tid == 0) {
        s_over = 0;
        bar_init(&done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tmem_alloc(&s_tmem, M_COLS);
    copies_wait<0>();
    publish_smem();
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = s_tmem;
    if (tid == 0) {
        const uint32_t desc = mma_desc(__is_same(T, __nv_bfloat16), false, true, M_ROWS, M_COLS);
        for (uint32_t c = 0; c < a.places / 16; c++)
            mma16(tmem, desc_lo(base + (c >> 2) * M_ROWS * ROW_BYTES + (c & 3) * 32, 16), desc_lo(base + b_bytes + c * 16 * ROW_BYTES, block), desc, c);
        mma_commit(&done);
    }
    const bool ok = __syncthreads_and(bar_wait(&done, 0, &s_over));
    tc_after();
    if (ok) {
        float *sums = reinterpret_cast<float *>(local);
        if (warp < 4) {
            for (uint32_t c = 0; c < M_COLS; c += 16) {
                float v[16];
                tmem_load16(tmem + (warp << 21) + c, v);
#pragma unroll
                for (uint32_t q = 0; q < 16; q += 4) *reinterpret_cast<float4 *>(sums + tid * M_PITCH + c + q) = make_float4(v[q], v[q + 1], v[q + 2], v[q + 3]);
            }
        }
        __syncthreads();
#pragma unroll 8
        for (uint32_t i = 0; i < PARTS; i++) {
            const uint32_t e = i * M_THREADS + tid, row = e / PER_ROW, c = e % PER_ROW * V::N;
            const uint64_t col = c0 + c;
            if (r0 + row >= a.rows || col >= a.cols) continue;
            V x;
            if constexpr (VB == 16) x = w[i];
            else x.raw = *reinterpret_cast<const typename Raw<VB>::type *>(a.w + (r0 + row) * a.w_stride + col);
#pragma unroll
            for (uint32_t q = 0; q < V::N; q++) x.e[q] = narrow<T>(widen(x.e[q]) + a.scale * sums[row * M_PITCH + c + q]);
            *reinterpret_cast<typename Raw<VB>::type *>(a.out + (r0 + row) * a.cols + col) = x.raw;
        }
    }
    tc_before();
    __syncthreads();
    if (warp == 0) {
        tc_after();
        tmem_free(tmem, M_COLS);
    }
}

}  // namespace lmz
