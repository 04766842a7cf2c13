// The gradients of adapters' factors.
#pragma once
#include "adapter_kernels.cuh"
#include "tcgen.cuh"

namespace lmz {

constexpr uint32_t FG_FEATS = 128, FG_THREADS = 256, FG_MAX_STAGES = 4;
constexpr uint32_t FG_PITCH = FG_FEATS + 1;

template <class T>
struct FactorGradArgs {
    const T *z, *thin;                         // rows of the tokens: `stride` elements apart, and [2][rp]
    const uint32_t *order, *start;             // tokens sorted by adapter and where each adapter's begin; NULL: all have adapter 0
    T *out;                                    // dF_i(f, j) at i * each + f * wide + j * place
    uint64_t stride, feats, each, wide, place;
    uint32_t tokens, rank, rp, split;
    uint32_t stages, stage_bytes, tmem_columns;
};

// Bytes of a half of the thin rows' tile: blocks of 64 columns by 64 tokens.
__host__ __device__ constexpr uint32_t thin_tile_bytes(uint32_t rp) { return (rp + 63) / 64 * STEP_K * ROW_BYTES; }

// dF_i(f, j) = sum over i's tokens of thin[t][j] z[t][f].
//
// Tokens are the tensor core's K.  They come one by one in the order of a sort by adapter, so that a sum has its own tokens and
// no others (a foreign token times zero would still bring its infinities in), in one order.  Rows are copied as they lie,
// both operands MN-major; z's tile meets both halves of the thin rows.  Bound by reading z once, 128 features a block;
// the CTAs of a cluster share an adapter's tokens.
template <class T>
__global__ void __launch_bounds__(FG_THREADS) k_factor_grad(const FactorGradArgs<T> a)
{
    extern __shared__ uint8_t f_smem[];
    __shared__ uint64_t freed[FG_MAX_STAGES];
    __shared__ uint64_t sums;
    __shared__ uint32_t s_tmem, s_over;
    const uint32_t tid = threadIdx.x, warp = tid >> 5;
    const uint32_t rank = a.split > 1 ? cluster_rank() : 0;
    const uint64_t f0 = static_cast<uint64_t>(blockIdx.x / a.split) * FG_FEATS;
    const uint32_t i = blockIdx.y;
    const uint32_t begin = a.start ? a.start[i] : 0, total = a.start ? a.start[i + 1] - begin : a.tokens;
    const uint32_t lo = begin + static_cast<uint32_t>(static_cast<uint64_t>(total) * rank / a.split);
    const uint32_t hi = begin + static_cast<uint32_t>(static_cast<uint64_t>(total) * (rank + 1) / a.split);
    const uint32_t steps = (hi - lo + STEP_K - 1) / STEP_K;
    const uint32_t ring = (smem_addr(f_smem) + ATOM_BYTES - 1) & ~(ATOM_BYTES - 1);
    const uint32_t half = thin_tile_bytes(a.rp), z_bytes = FG_FEATS * STEP_K * 2;
    float *part = reinterpret_cast<float *>(f_smem + (ring - smem_addr(f_smem)));
    volatile uint32_t *over = &s_over;

    if (tid == 0) {
        s_over = 0;
        for (uint32_t st = 0; st < a.stages; st++) bar_init(&freed[st], 1);
        bar_init(&sums, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) tmem_alloc(&s_tmem, a.tmem_columns);
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = s_tmem;

    auto load = [&](uint32_t n) {
        if (n < steps) {
            const uint32_t dst = ring + n % a.stages * a.stage_bytes, at = lo + n * STEP_K;
            for (uint32_t e = tid; e < STEP_K * 16; e += FG_THREADS) {
                const uint32_t row = e >> 4, c = e & 15;
                const uint64_t f = f0 + c * 8;
                const bool on = at + row < hi && f < a.feats;
                const uint64_t t = on ? (a.order ? a.order[at + row] : at + row) : 0;
                copy16(dst + (c >> 3) * STEP_K * ROW_BYTES + swizzled(row, c & 7), on ? a.z + t * a.stride + f : a.z, on);
            }
            const uint32_t parts = a.rp / 8;
            for (uint32_t e = tid; e < STEP_K * parts * 2; e += FG_THREADS) {
                const uint32_t row = e / (parts * 2), q = e % (parts * 2), lower = q >= parts, c = lower ? q - parts : q;
                const bool on = at + row < hi;
                const uint64_t t = on ? (a.order ? a.order[at + row] : at + row) : 0;
                copy16(dst + z_bytes + lower * half + (c >> 3) * STEP_K * ROW_BYTES + swizzled(row, c & 7),
                       on ? a.thin + t * 2 * a.rp + q * 8 : a.thin, on);
            }
        }
        copies_commit();
    };
    const uint32_t desc = mma_desc(__is_same(T, __nv_bfloat16), true, true, FG_FEATS, (a.rp + 15) & ~15u);
    for (uint32_t n = 0; n + 1 < a.stages; n++) load(n);
    bool ok = true;
    for (uint32_t n = 0; n < steps && ok; n++) {
        if (a.stages == 2) copies_wait<0>();
        else if (a.stages == 3) copies_wait<1>();
        else copies_wait<2>();
        publish_smem();
        __syncthreads();
        if (tid == 0) {
            const uint32_t src = ring + n % a.stages * a.stage_bytes;
            tc_after();
            for (uint32_t h = 0; h < 2; h++)
#pragma unroll
                for (uint32_t c = 0; c < STEP_K / 16; c++)
                    mma16(tmem, desc_lo(src + c * 16 * ROW_BYTES, STEP_K * ROW_BYTES),
                          desc_lo(src + z_bytes + h * half + c * 16 * ROW_BYTES, STEP_K * ROW_BYTES), desc, n || h || c);
            mma_commit(&freed[n % a.stages]);
        }
        if (n + a.stages - 1 < steps) {                          // the stage of the step before is next to be filled
            ok = n == 0 || bar_wait(&freed[(n - 1) % a.stages], ((n - 1) / a.stages) & 1, over);
            ok = __syncthreads_and(ok);
        }
        if (ok) load(n + a.stages - 1);
    }
    copies_wait<0>();
    if (tid == 0) mma_commit(&sums);
    ok = __syncthreads_and(bar_wait(&sums, 0, over) && ok);
    tc_after();
    if (warp < 4 && ok) {
        for (uint32_t c = 0; c < a.rp; c += 8) {
            float v[8] = {};
            if (steps) tmem_load8(tmem + (warp << 21) + c, v);
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) part[(c + e) * FG_PITCH + tid] = v[e];
        }
        tc_before();
    }
    __syncwarp();
    if (a.split > 1) cluster_barrier();
    else __syncthreads();
    if (ok) {
        T *out = a.out + i * a.each;
        const uint32_t share = FG_FEATS / a.split, mine = a.wide == 1 ? FG_FEATS : share;
        // neighbouring threads write neighbouring elements: along f (a CTA every split-th j), or along j (a CTA its share of the f)
        for (uint32_t e = tid; e < (a.wide == 1 ? (a.rank + a.split - 1 - rank) / a.split : a.rank) * mine; e += FG_THREADS) {
            const uint32_t j = a.wide == 1 ? rank + e / FG_FEATS * a.split : e % a.rank, row = a.wide == 1 ? e % FG_FEATS : rank * share + e / a.rank;
            if (f0 + row >= a.feats) continue;
            float sum = 0;
            for (uint32_t q = 0; q < a.split; q++) sum += peer_float(ring + (j * FG_PITCH + row) * 4, q);
            out[(f0 + row) * a.wide + j * a.place] = narrow<T>(sum);
        }
    }
    if (a.split > 1) cluster_barrier();
    tc_before();
    __syncthreads();
    if (warp == 0) {
        tc_after();
        tmem_free(tmem, a.tmem_columns);
    }
}

}  // namespace lmz
