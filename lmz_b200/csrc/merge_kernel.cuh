// An adapter merged into its weight.
#pragma once
#include "adapter_kernels.cuh"
#include "tcgen.cuh"

namespace lmz {

constexpr uint32_t M_ROWS = 128, M_COLS = 128, M_THREADS = 256;
constexpr uint32_t M_BLOCK = M_ROWS * ROW_BYTES;       // 64 columns of the weight's tile, swizzled as operands are

template <class T>
struct MergeArgs {
    const T *w, *a, *b;
    T *out;
    uint64_t rows, cols, w_stride;
    uint32_t rank, places;                     // places: rank up to a multiple of 16
    float scale;
    bool a_even, b_even;                       // the factors' rows start on boundaries of 16 bytes
};

// Shared memory of a block: the weight's tile, and both factors'.
__host__ __device__ constexpr uint32_t merge_smem(uint32_t places)
{
    return M_COLS / 64 * M_BLOCK + (places + STEP_K - 1) / STEP_K * M_BLOCK + M_COLS / 64 * places * ROW_BYTES + ATOM_BYTES;
}

// W' = W + s B A, a tile of 128 x 128 a block.
//
// Bound by HBM: W read and W' written once.  The tile is on its way into shared memory while the thin product, a few
// instructions of the tensor core, is made; sums are added to it there, and it leaves as it came, in whole lines (VB bytes
// an instruction and thread).  Nothing is held in registers meanwhile, so that three or four blocks share an SM and keep some
// 100 KiB of it moving.
template <class T, int VB>
__global__ void __launch_bounds__(M_THREADS) k_merge(const MergeArgs<T> a)
{
    using V = Vec<T, VB>;
    constexpr uint32_t PER_ROW = M_COLS / V::N, PARTS = M_ROWS * PER_ROW / M_THREADS, BATCH = PARTS < 16 ? PARTS : 16;
    extern __shared__ uint8_t m_smem[];
    __shared__ uint64_t done;
    __shared__ uint32_t s_tmem, s_over;
    const uint32_t tid = threadIdx.x, warp = tid >> 5;
    const uint64_t r0 = static_cast<uint64_t>(blockIdx.y) * M_ROWS, c0 = static_cast<uint64_t>(blockIdx.x) * M_COLS;
    const uint32_t base = (smem_addr(m_smem) + ATOM_BYTES - 1) & ~(ATOM_BYTES - 1);
    uint8_t *local = m_smem + (base - smem_addr(m_smem));
    const uint32_t b_at = M_COLS / 64 * M_BLOCK, a_at = b_at + (a.places + STEP_K - 1) / STEP_K * M_BLOCK, block = a.places * ROW_BYTES;
    // where element c of the tile's row lies
    auto place = [](uint32_t row, uint32_t c) { return (c >> 6) * M_BLOCK + swizzled(row, (c & 63) * sizeof(T) >> 4) + (c * sizeof(T) & 15); };

    wait_for_previous();
    // B's rows, K-major; A's, MN-major in blocks of 64 columns
    for (uint32_t e = tid; e < M_ROWS * a.places / 8; e += M_THREADS) {
        const uint32_t row = e / (a.places / 8), c = e % (a.places / 8), j = c * 8;
        const uint32_t at = b_at + (c >> 3) * M_BLOCK + swizzled(row, c & 7);
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
        const uint32_t at = a_at + (c >> 3) * block + swizzled(j, c & 7);
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
    for (uint32_t i0 = 0; i0 < PARTS; i0 += BATCH) {
        V w[BATCH];
#pragma unroll
        for (uint32_t i = 0; i < BATCH; i++) {
            const uint32_t e = (i0 + i) * M_THREADS + tid, row = e / PER_ROW, c = e % PER_ROW * V::N;
            const bool on = r0 + row < a.rows && c0 + c < a.cols;
            const T *p = on ? a.w + (r0 + row) * a.w_stride + c0 + c : a.w;
            if constexpr (VB == 16) {
                copy16(base + place(row, c), p, on);
            } else {
                w[i].raw = {};
                if (on) w[i].raw = *reinterpret_cast<const typename Raw<VB>::type *>(p);
            }
        }
        if constexpr (VB != 16) {
#pragma unroll
            for (uint32_t i = 0; i < BATCH; i++) {
                const uint32_t e = (i0 + i) * M_THREADS + tid, row = e / PER_ROW, c = e % PER_ROW * V::N;
                *reinterpret_cast<typename Raw<VB>::type *>(local + place(row, c)) = w[i].raw;
            }
        }
    }
    copies_commit();
    if (tid == 0) {
        s_over = 0;
        bar_init(&done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tmem_alloc(&s_tmem, M_COLS);
    copies_wait<1>();                                            // the factors
    publish_smem();
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = s_tmem;
    if (warp == 0 && elected()) {
        const uint32_t desc = mma_desc(__is_same(T, __nv_bfloat16), false, true, M_ROWS, M_COLS);
        for (uint32_t c = 0; c < a.places / 16; c++)
            mma16(tmem, desc_lo(base + b_at + (c >> 2) * M_BLOCK + (c & 3) * 32, 16), desc_lo(base + a_at + c * 16 * ROW_BYTES, block), desc, c);
        mma_commit(&done);
    }
    __syncwarp();
    copies_wait<0>();                                            // the weight's tile
    const bool ok = __syncthreads_and(warp_wait(&done, 0, &s_over));
    tc_after();
    if (ok) {
        const uint32_t row = tid & (M_ROWS - 1), half = tid / M_ROWS * (M_COLS / 2);     // a TMEM lane is a row
#pragma unroll
        for (uint32_t c = 0; c < M_COLS / 2; c += 16) {
            float v[16];
            tmem_load16(tmem + ((warp & 3) << 21) + half + c, v);
#pragma unroll
            for (uint32_t q = 0; q < 16; q += 8) {
                uint4 *at = reinterpret_cast<uint4 *>(local + place(row, half + c + q));
                Vec<T, 16> x;
                x.raw = *at;
#pragma unroll
                for (uint32_t e = 0; e < 8; e++) x.e[e] = narrow<T>(widen(x.e[e]) + a.scale * v[q + e]);
                *at = x.raw;
            }
        }
        tc_before();
        __syncthreads();
#pragma unroll 8
        for (uint32_t i = 0; i < PARTS; i++) {
            const uint32_t e = i * M_THREADS + tid, r = e / PER_ROW, c = e % PER_ROW * V::N;
            if (r0 + r < a.rows && c0 + c < a.cols)
                *reinterpret_cast<typename Raw<VB>::type *>(a.out + (r0 + r) * a.cols + c0 + c) = *reinterpret_cast<const typename Raw<VB>::type *>(local + place(r, c));
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
