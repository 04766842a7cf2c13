// An adapter merged into its weight.
#pragma once
#include "adapter_kernels.cuh"
#include "merge_layout.cuh"
#include "tcgen.cuh"

namespace lmz {

constexpr uint32_t M_THREADS = 256;

template <class T>
struct MergeArgs {
    const T *w, *a, *b;
    T *out;
    uint64_t rows, cols, w_stride;
    uint32_t rank, places;                     // places: rank up to a multiple of 16
    float scale;
    bool a_even, b_even;                       // the factors' rows start on boundaries of 16 bytes
};

struct MergeShared {
    uint64_t done;
    uint32_t tmem, over;
};
static_assert(sizeof(MergeShared) == M_SHARED && M_ROW_BYTES == ROW_BYTES);

// W' = W + s B A, in tiles of 128 x 128, a row of them after the other; a block has a run of tiles.
//
// Bound by HBM: W read and W' written once.  The next tile is on its way into shared memory while this one's thin product, a
// few instructions of the tensor core, is made and added to it there; it leaves as it came, in whole lines (VB bytes an
// instruction and thread).  Nothing is held in registers meanwhile, so that two blocks share an SM.  One B200, 14336 x 4096 at
// rank 64: 49 us (4.8 TB/s); a tile a block 57, with the weight held in registers 80.
template <class T, int VB>
__global__ void __launch_bounds__(M_THREADS, 2) k_merge(const MergeArgs<T> a)
{
    using V = Vec<T, VB>;
    constexpr uint32_t PER_ROW = M_COLS / V::N, PARTS = M_ROWS * PER_ROW / M_THREADS, BATCH = PARTS < 16 ? PARTS : 16;
    extern __shared__ __align__(1024) uint8_t m_smem[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, base = smem_addr(m_smem), stage_bytes = merge_stage(a.places);
    const uint32_t stages = merge_stages(a.places), b_at = stages * stage_bytes, block = a.places * ROW_BYTES;
    MergeShared &s = *reinterpret_cast<MergeShared *>(m_smem + merge_smem(a.places) - sizeof(MergeShared));
    const uint64_t across = (a.cols + M_COLS - 1) / M_COLS, tiles = across * ((a.rows + M_ROWS - 1) / M_ROWS);
    const uint64_t first = tiles * blockIdx.x / gridDim.x, last = tiles * (blockIdx.x + 1) / gridDim.x;
    // where element c of a tile's row lies in its stage
    auto place = [](uint32_t row, uint32_t c) { return (c >> 6) * M_BLOCK + swizzled(row, (c & 63) * sizeof(T) >> 4) + (c * sizeof(T) & 15); };

    wait_for_previous();
    if (tid == 0) {
        s.over = 0;
        bar_init(&s.done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tmem_alloc(&s.tmem, M_COLS);
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = s.tmem;

    auto load_b = [&](uint64_t r0) {                             // K-major
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
                *reinterpret_cast<uint4 *>(m_smem + at) = v.raw;
            }
        }
    };
    auto load = [&](uint64_t tile) {                             // the weight's tile, and A's, MN-major in blocks of 64 columns
        const uint64_t r0 = tile / across * M_ROWS, c0 = tile % across * M_COLS;
        const uint32_t stage = ((tile - first) & (stages - 1)) * stage_bytes, a_at = stage + M_COLS / 64 * M_BLOCK;
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
                *reinterpret_cast<uint4 *>(m_smem + at) = v.raw;
            }
        }
        for (uint32_t i0 = 0; i0 < PARTS; i0 += BATCH) {
            V w[BATCH];
#pragma unroll
            for (uint32_t i = 0; i < BATCH; i++) {
                const uint32_t e = (i0 + i) * M_THREADS + tid, row = e / PER_ROW, c = e % PER_ROW * V::N;
                const bool on = r0 + row < a.rows && c0 + c < a.cols;
                const T *p = on ? a.w + (r0 + row) * a.w_stride + c0 + c : a.w;
                if constexpr (VB == 16) {
                    copy16(base + stage + place(row, c), p, on);
                } else {
                    w[i].raw = {};
                    if (on) w[i].raw = *reinterpret_cast<const typename Raw<VB>::type *>(p);
                }
            }
            if constexpr (VB != 16) {
#pragma unroll
                for (uint32_t i = 0; i < BATCH; i++) {
                    const uint32_t e = (i0 + i) * M_THREADS + tid, row = e / PER_ROW, c = e % PER_ROW * V::N;
                    *reinterpret_cast<typename Raw<VB>::type *>(m_smem + stage + place(row, c)) = w[i].raw;
                }
            }
        }
    };

    const uint32_t desc = mma_desc(__is_same(T, __nv_bfloat16), false, true, M_ROWS, M_COLS);
    uint64_t band = ~0ull;                                       // the row of tiles whose B is here
    bool ok = true;
    if (first < last) load(first);
    copies_commit();
    for (uint64_t tile = first; ok && tile < last; tile++) {
        const uint64_t r0 = tile / across * M_ROWS, c0 = tile % across * M_COLS;
        const uint32_t stage = ((tile - first) & (stages - 1)) * stage_bytes, a_at = stage + M_COLS / 64 * M_BLOCK;
        if (tile / across != band) {                             // (the products that read the last one have ended)
            band = tile / across;
            load_b(r0);
        }
        copies_commit();
        if (stages > 1 && tile + 1 < last) load(tile + 1);       // (what its stage held has left: the loop's last barrier)
        copies_commit();
        if (stages > 1) copies_wait<1>();
        else copies_wait<0>();
        publish_smem();
        __syncthreads();
        if (warp == 0 && elected()) {
            tc_after();
            for (uint32_t c = 0; c < a.places / 16; c++)
                mma16(tmem, desc_lo(base + b_at + (c >> 2) * M_BLOCK + (c & 3) * 32, 16), desc_lo(base + a_at + c * 16 * ROW_BYTES, block), desc, c);
            mma_commit(&s.done);
        }
        __syncwarp();
        ok = __syncthreads_and(warp_wait(&s.done, (tile - first) & 1, &s.over));
        tc_after();
        if (!ok) break;
        const uint32_t row = tid & (M_ROWS - 1), half = tid / M_ROWS * (M_COLS / 2);     // a TMEM lane is a row
#pragma unroll
        for (uint32_t c = 0; c < M_COLS / 2; c += 16) {
            float v[16];
            tmem_load16(tmem + ((warp & 3) << 21) + half + c, v);
#pragma unroll
            for (uint32_t q = 0; q < 16; q += 8) {
                uint4 *at = reinterpret_cast<uint4 *>(m_smem + stage + place(row, half + c + q));
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
                *reinterpret_cast<typename Raw<VB>::type *>(a.out + (r0 + r) * a.cols + c0 + c) = *reinterpret_cast<const typename Raw<VB>::type *>(m_smem + stage + place(r, c));
        }
        __syncthreads();
        if (stages == 1 && tile + 1 < last) load(tile + 1);
    }
    copies_wait<0>();
    tc_before();
    __syncthreads();
    if (warp == 0) {
        tc_after();
        tmem_free(tmem, M_COLS);
    }
}

}  // namespace lmz
