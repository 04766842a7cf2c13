// The gradients of adapters' factors.
#pragma once
#include "adapter_kernels.cuh"
#include "tcgen.cuh"

namespace lmz {

constexpr uint32_t FG_FEATS = 128, FG_THREADS = 128, FG_MAX_STAGES = 8;
constexpr uint32_t FG_PITCH = FG_FEATS + 1;

struct FactorGradShared {
    uint64_t full[FG_MAX_STAGES], empty[FG_MAX_STAGES], sums;
    uint32_t tmem, over;
};

// One factor's gradient.
template <class T>
struct FactorGradJob {
    CUtensorMap z, z_rows, thin, thin_rows;    // tiles of 64 x 64, and of one row (for gathers)
    T *out;                                    // dF_i(f, j) at i * each + f * wide + j * place
    const float *scale;                        // F16: per adapter, what its sums are multiplied by (k_thin)
    uint64_t feats, each, wide, place;
    uint32_t clusters;                         // that it takes
};

template <class T>
struct FactorGradArgs {
    FactorGradJob<T> job[2];
    const uint32_t *order, *start;             // tokens sorted by adapter and where each adapter's begin; NULL: all have adapter 0
    uint32_t tokens, rank, rp, split;
    uint32_t blocks;                           // of FG_FEATS features
    uint32_t stages, stage_bytes, tmem_columns;
};

// A row of the thin product, both halves, in blocks of 64 columns; a stage of 64 tokens.
__host__ __device__ constexpr uint32_t thin_blocks(uint32_t rp) { return (2 * rp + 63) / 64; }
constexpr uint32_t FG_TILE = STEP_K * ROW_BYTES;
__host__ __device__ constexpr uint32_t factor_stage_bytes(uint32_t blocks, uint32_t rp) { return (2 * blocks + thin_blocks(rp)) * FG_TILE; }

// dF_i(f, j) = sum over i's tokens of thin[t][j] z[t][f].
//
// Tokens are the tensor core's K, and come in the order of a sort by adapter, so that a sum has its own tokens and no others
// (a foreign token times zero would still bring its infinities in), in one order.  Rows are brought as they lie, both
// operands MN-major: 64 neighbours by a tile's copy, others by gathers of four rows, whose places behind the last token read
// as zeros.  The halves of the thin rows are columns of their own, added at the end; an infinity or NaN is the upper halves' alone.  Bound by reading z (256 features a block,
// so that the thin rows are read half as often as by 128); the CTAs of a cluster share an adapter's tokens.  One B200, 8192 tokens
// of 4096 and 14336 features at rank 64: both factors 79 us (3.9 TB/s of HBM).
// The two factors' gradients are one launch: its first clusters make the one, the others the other.
template <class T>
__global__ void __launch_bounds__(FG_THREADS) k_factor_grad(const __grid_constant__ FactorGradArgs<T> a)
{
    extern __shared__ uint8_t f_smem[];
    __shared__ FactorGradShared s;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = a.split > 1 ? cluster_rank() : 0;
    const uint32_t place = blockIdx.x / a.split, which = place >= a.job[0].clusters;
    const FactorGradJob<T> &g = a.job[which];
    const uint32_t f0 = (which ? place - a.job[0].clusters : place) * a.blocks * FG_FEATS, i = blockIdx.y;
    wait_for_previous();
    const uint32_t begin = a.start ? a.start[i] : 0, end = a.start ? a.start[i + 1] : i ? 0 : a.tokens;
    const uint32_t all = (end - begin + STEP_K - 1) / STEP_K;
    const uint32_t n0 = static_cast<uint32_t>(static_cast<uint64_t>(all) * rank / a.split), n1 = static_cast<uint32_t>(static_cast<uint64_t>(all) * (rank + 1) / a.split);
    const uint32_t ring = (smem_addr(f_smem) + ATOM_BYTES - 1) & ~(ATOM_BYTES - 1);
    constexpr float LOWER = __is_same(T, __half) ? THIN_LOWER : 1.0f;
    const uint32_t thins = thin_blocks(a.rp), thin_at = 2 * a.blocks * FG_TILE;
    volatile uint32_t *over = &s.over;

    if (tid == 0) {
        s.over = 0;
        for (uint32_t st = 0; st < a.stages; st++) bar_init(&s.full[st], 1), bar_init(&s.empty[st], 1);
        bar_init(&s.sums, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(&s.tmem, a.tmem_columns);
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = s.tmem;

    if (warp == 0) {
        RingPlace at;
        for (uint32_t n = n0; n < n1; n++, at.next(a.stages)) {
            const uint32_t p = begin + n * STEP_K, left = end - p, st = at.stage, dst = ring + st * a.stage_bytes;
            // four rows of a lane: its gathers', and the first and last tell whether all are neighbours
            uint32_t row[4];
#pragma unroll
            for (uint32_t q = 0; q < 4; q++) {
                const uint32_t o = (lane & 15) * 4 + q;
                row[q] = o < left ? (a.order ? a.order[p + o] : p + o) : a.tokens;
            }
            const uint32_t first = __shfl_sync(~0u, row[0], 0), last = __shfl_sync(~0u, row[3], 15);
            const bool tile = left >= STEP_K && last - first == STEP_K - 1;      // (an adapter's tokens ascend)
            if (at.turn && !warp_wait(&s.empty[st], (at.turn - 1) & 1, over)) break;
            if (lane == 0) bar_expect(&s.full[st], a.stage_bytes);
            __syncwarp();
            if (tile) {
                if (elected()) {
                    for (uint32_t b = 0; b < 2 * a.blocks; b++) tma_load_2d(&g.z, smem_addr(&s.full[st]), dst + b * FG_TILE, f0 + b * 64, first);
                    for (uint32_t b = 0; b < thins; b++) tma_load_2d(&g.thin, smem_addr(&s.full[st]), dst + thin_at + b * FG_TILE, b * 64, first);
                }
            } else if (lane < 16) {
                for (uint32_t b = 0; b < 2 * a.blocks; b++) tma_gather4(&g.z_rows, &s.full[st], dst + b * FG_TILE + lane * 4 * ROW_BYTES, f0 + b * 64, row);
                for (uint32_t b = 0; b < thins; b++) tma_gather4(&g.thin_rows, &s.full[st], dst + thin_at + b * FG_TILE + lane * 4 * ROW_BYTES, b * 64, row);
            }
            __syncwarp();
        }
        if (*over)                                               // nothing may still be on its way into this block's memory
            for (uint32_t st = 0; st < a.stages; st++) {
                const uint32_t used = at.turn - (st >= at.stage);                // the last turn that filled this stage
                if (used != ~0u) bar_drain(&s.full[st], used & 1);
            }
    } else if (warp == 1) {
        // at most 256 columns a product, in whole blocks
        const uint32_t columns = 2 * a.rp, one = columns < 256 ? columns : 256, two = columns - one;
        constexpr bool bf16 = __is_same(T, __nv_bfloat16);
        const uint32_t desc = mma_desc(bf16, true, true, FG_FEATS, one), desc2 = mma_desc(bf16, true, true, FG_FEATS, two);
        const uint32_t z_lo = desc_lo(ring, FG_TILE), t_lo = desc_lo(ring + thin_at, FG_TILE);
        RingPlace at;
        for (uint32_t n = n0; n < n1; n++, at.next(a.stages)) {
            const uint32_t st = at.stage, off = st * a.stage_bytes >> 4;
            if (!warp_wait(&s.full[st], at.turn & 1, over)) break;
            if (elected()) {
                for (uint32_t b = 0; b < a.blocks; b++) {
                    const uint32_t z = z_lo + off + (b * 2 * FG_TILE >> 4), d = tmem + b * columns;
#pragma unroll
                    for (uint32_t c = 0; c < STEP_K / 16; c++) {
                        mma16(d, z + (c * 16 * ROW_BYTES >> 4), t_lo + off + (c * 16 * ROW_BYTES >> 4), desc, n != n0 || c);
                        if (two) mma16(d + one, z + (c * 16 * ROW_BYTES >> 4), t_lo + off + (4 * FG_TILE + c * 16 * ROW_BYTES >> 4), desc2, n != n0 || c);
                    }
                }
                mma_commit(&s.empty[st]);
            }
            __syncwarp();
        }
        if (elected()) mma_commit(&s.sums);
        __syncwarp();
    }
    __syncwarp();
    const bool ok = __syncthreads_and(warp_wait(&s.sums, 0, over));
    float *part = reinterpret_cast<float *>(f_smem + (ring - smem_addr(f_smem)));
    tc_after();
    if (ok && !*over) {                                          // the halves' sums, over the stages
        for (uint32_t b = 0; b < a.blocks; b++)
            for (uint32_t c = 0; c < a.rp; c += 8) {
                float v[8] = {}, w[8] = {};
                if (n1 > n0) {
                    tmem_load8(tmem + (warp << 21) + b * 2 * a.rp + c, v);
                    tmem_load8(tmem + (warp << 21) + b * 2 * a.rp + a.rp + c, w);
                }
#pragma unroll
                for (uint32_t e = 0; e < 8; e++) part[(b * a.rp + c + e) * FG_PITCH + tid] = isfinite(v[e]) ? v[e] + w[e] * LOWER : v[e];
            }
    }
    tc_before();
    __syncwarp();
    if (a.split > 1) cluster_barrier();
    else __syncthreads();
    if (ok && !*over) {
        T *out = g.out + i * g.each;
        const float scale = __is_same(T, __half) ? g.scale[i] : 1.0f;
        const uint32_t wide = a.blocks * FG_FEATS;
        const Peers peers(ring, a.split);
        // Eight neighbours of the result a thread: along f, threads side by side on neighbouring j; or along j, threads on
        // neighbouring f (either way they read neighbouring banks).
        const bool along_f = g.wide == 1;
        const uint64_t next = along_f ? g.place : g.wide;
        const uint64_t bits = reinterpret_cast<uint64_t>(g.out) | next * 2;      // stores of 16 bytes, 8, 4, or each by itself
        const uint32_t tasks = along_f ? a.rank * (wide / 8) : (a.rank + 7) / 8 * wide;
        const uint32_t e1 = static_cast<uint32_t>(static_cast<uint64_t>(tasks) * (rank + 1) / a.split);
        for (uint32_t e = static_cast<uint32_t>(static_cast<uint64_t>(tasks) * rank / a.split) + tid; e < e1; e += FG_THREADS) {
            const uint32_t j = along_f ? e % a.rank : e / wide * 8, row = along_f ? e / a.rank * 8 : e % wide;
            const uint64_t f = f0 + static_cast<uint64_t>(row);
            if (f >= g.feats) continue;
            float sum[8];
            peers.sum8(((row / FG_FEATS * a.rp + j) * FG_PITCH + row % FG_FEATS) * 4, along_f ? 4 : FG_PITCH * 4, sum);
            Vec<T, 16> v;
#pragma unroll
            for (uint32_t q = 0; q < 8; q++) v.e[q] = narrow<T>(__is_same(T, __half) ? sum[q] * scale : sum[q]);
            T *to = out + f * g.wide + j * g.place;
            const uint64_t left = along_f ? g.feats - f : a.rank - j;
            if (left >= 8 && (bits & 15) == 0) {
                *reinterpret_cast<uint4 *>(to) = v.raw;
            } else if (left >= 8 && (bits & 7) == 0) {
                reinterpret_cast<uint2 *>(to)[0] = make_uint2(v.raw.x, v.raw.y), reinterpret_cast<uint2 *>(to)[1] = make_uint2(v.raw.z, v.raw.w);
            } else if (left >= 8 && (bits & 3) == 0) {
                uint32_t *words = reinterpret_cast<uint32_t *>(to);
                words[0] = v.raw.x, words[1] = v.raw.y, words[2] = v.raw.z, words[3] = v.raw.w;
            } else {
#pragma unroll
                for (uint32_t q = 0; q < 8; q++)
                    if (q < left) to[q] = v.e[q];
            }
        }
    }
    if (a.split > 1) cluster_barrier();                          // nobody leaves while another reads its sums
    tc_before();
    __syncthreads();
    if (warp == 1) {
        tc_after();
        tmem_free(tmem, a.tmem_columns);
    }
}

}  // namespace lmz
