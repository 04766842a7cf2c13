// The thin products h = s x A^T and g = s dy B.
#pragma once
#include "adapter_kernels.cuh"
#include "tcgen.cuh"

namespace lmz {

constexpr uint32_t H_TOKENS = 128;             // tokens of a tile: the tensor core's M, a TMEM lane each
constexpr uint32_t H_COLUMNS = 256;            // most columns of a tile: its N
constexpr uint32_t H_THREADS = H_TOKENS + 64, H_MAX_STAGES = 8;
constexpr uint32_t H_PITCH = H_TOKENS + 1;     // of the partial sums in shared memory: neighbouring columns in neighbouring banks

struct HiddenShared {
    uint64_t full[H_MAX_STAGES], empty[H_MAX_STAGES], sums;
    uint32_t tmem, over, present;
    alignas(16) int32_t adapter[H_TOKENS];     // per token
    int32_t list[H_TOKENS];                    // the tile's adapters in the order of their first tokens
    int32_t slot[H_TOKENS];                    // per token: where its adapter stands in that list, -1: none
    uint32_t firsts[H_TOKENS / 32];
};

template <class T>
struct HiddenArgs {
    CUtensorMap x, f;                          // f: adapters x rank x K
    CUtensorMap xs;                            // x in the order of `sorted`
    TokenIndex index;
    SortedTokens sorted;
    Thin *h;                                   // [token][2][rp], in that order if x is
    void *kept;                                // NULL, or for the factors' gradients in the tokens' own order: the same for BF16
                                               // tensors, for F16 ones [token][rp] in 32 bits
    uint64_t tokens;
    uint32_t rank, rp, steps, split;
    uint32_t each;                             // adapters of a block: as many as have room in H_COLUMNS columns
    uint32_t stages, stage_bytes, tmem_columns;
};

// h[t][j] = s_i * sum over k of x[t][k] F_i[j][k], for tokens with an adapter, as two halves.
//
// A block multiplies 128 tokens by up to 256 / rp of the adapters they have side by side, and each token keeps the columns of
// its own: nothing of another adapter or token comes into a sum.  Reads x once per 256 columns of present adapters (for one
// adapter, and for most batches of prompts: once) and is bound by that; for few tokens by latency, so K is shared by the CTAs
// of a cluster and their sums meet in distributed shared memory.  One B200, us: 8192 tokens x 14336, one adapter of rank 64 48 (4.9
// TB/s of HBM), x 4096 21; 4096 x 4096 for eight of rank 32 14.5; one token 9.
template <class T>
__global__ void __launch_bounds__(H_THREADS) k_hidden(const __grid_constant__ HiddenArgs<T> a)
{
    extern __shared__ uint8_t h_smem[];
    __shared__ HiddenShared s;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = a.split > 1 ? cluster_rank() : 0;
    const uint32_t tile = blockIdx.x / a.split;
    const uint64_t t0 = static_cast<uint64_t>(tile) * H_TOKENS;
    const uint32_t k0 = static_cast<uint32_t>(static_cast<uint64_t>(a.steps) * rank / a.split);
    const uint32_t k1 = static_cast<uint32_t>(static_cast<uint64_t>(a.steps) * (rank + 1) / a.split);
    const uint32_t ring = (smem_addr(h_smem) + ATOM_BYTES - 1) & ~(ATOM_BYTES - 1);
    volatile uint32_t *over = &s.over;

    // (Neither kernel leaves an SM room for a block of the other, so the next one's cannot take this block's TMEM.)
    wait_for_previous();
    let_next_start();
    // Which adapters the tile has: a token is its adapter's first if none before it has it.
    if (tid == 0) {
        s.over = 0;
        for (uint32_t i = 0; i < a.stages; i++) bar_init(&s.full[i], 1), bar_init(&s.empty[i], 1);
        bar_init(&s.sums, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const bool sorted = a.sorted.on();
    const TokenIndex index = a.sorted.index(a.index, sorted);
    int mine = -1;
    if (tid < H_TOKENS) {
        if (t0 + tid < a.tokens) mine = index.of(t0 + tid);
        s.adapter[tid] = mine;
    }
    __syncthreads();
    uint32_t first = 0;
    if (tid < H_TOKENS) {
        first = tid;
        if (!a.index.ids) first = 0;
        else
            for (int i = H_TOKENS - 4; i >= 0; i -= 4) {         // (backwards: the lowest match stays)
                const int4 v = *reinterpret_cast<const int4 *>(s.adapter + i);
                if (v.w == mine) first = i + 3;
                if (v.z == mine) first = i + 2;
                if (v.y == mine) first = i + 1;
                if (v.x == mine) first = i;
            }
        const uint32_t firsts = __ballot_sync(~0u, first == tid && mine >= 0);
        if (lane == 0) s.firsts[warp] = firsts;
    }
    __syncthreads();
    if (tid < H_TOKENS) {
        uint32_t at = __popc(s.firsts[first >> 5] & ((1u << (first & 31)) - 1));
        for (uint32_t w = 0; w < first >> 5; w++) at += __popc(s.firsts[w]);
        s.slot[tid] = mine >= 0 ? static_cast<int>(at) : -1;
        if (first == tid && mine >= 0) s.list[at] = mine;
    }
    const uint32_t present = __popc(s.firsts[0]) + __popc(s.firsts[1]) + __popc(s.firsts[2]) + __popc(s.firsts[3]);
    const uint32_t from = blockIdx.y * a.each;
    if (from >= present) return;                                 // (all CTAs of the cluster)
    const uint32_t count = present - from < a.each ? present - from : a.each;
    if (warp == 5) tmem_alloc(&s.tmem, a.tmem_columns);
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = s.tmem;

    if (warp == 4) {
        RingPlace at;
        for (uint32_t k = k0; k < k1; k++, at.next(a.stages)) {
            const uint32_t st = at.stage, dst = ring + st * a.stage_bytes;
            if (at.turn && !warp_wait(&s.empty[st], (at.turn - 1) & 1, over)) break;
            if (elected()) {
                bar_expect(&s.full[st], H_TOKENS * ROW_BYTES + count * a.rank * ROW_BYTES);
                tma_load_2d(sorted ? &a.xs : &a.x, smem_addr(&s.full[st]), dst, k * STEP_K, tile * H_TOKENS);
            }
            __syncwarp();
            for (uint32_t i = lane; i < count; i += 32)
                tma_load_3d(&a.f, smem_addr(&s.full[st]), dst + H_TOKENS * ROW_BYTES + i * a.rp * ROW_BYTES, k * STEP_K, 0, s.list[from + i]);
            __syncwarp();
        }
        if (*over)                                               // nothing may still be on its way into this block's memory
            for (uint32_t i = 0; i < a.stages; i++) {
                const uint32_t used = at.turn - (i >= at.stage);                 // the last turn that filled this stage
                if (used != ~0u) bar_drain(&s.full[i], used & 1);
            }
    } else if (warp == 5) {
        const uint32_t desc = mma_desc(__is_same(T, __nv_bfloat16), false, false, H_TOKENS, (count * a.rp + 15) & ~15u);
        RingPlace at;
        const uint32_t a_lo = desc_lo(ring, 16), b_lo = desc_lo(ring + H_TOKENS * ROW_BYTES, 16);
        for (uint32_t k = k0; k < k1; k++, at.next(a.stages)) {
            const uint32_t st = at.stage, off = st * a.stage_bytes >> 4;
            if (!warp_wait(&s.full[st], at.turn & 1, over)) break;
            if (elected()) {
#pragma unroll
                for (uint32_t c = 0; c < STEP_K / 16; c++) mma16(tmem, a_lo + off + c * 2, b_lo + off + c * 2, desc, k != k0 || c);
                mma_commit(&s.empty[st]);
            }
            __syncwarp();
        }
        if (elected()) mma_commit(&s.sums);
        __syncwarp();
        if (*over)
            bar_drain(&s.sums, 0);
    } else if (warp_wait(&s.sums, 0, over)) {
        // every token's own columns, over the stages (all products have ended)
        tc_after();
        float *part = reinterpret_cast<float *>(h_smem + (ring - smem_addr(h_smem)));
        const int slot = s.slot[tid] - static_cast<int>(from);
        for (uint32_t i = 0; i < count; i++) {
            if (!__any_sync(~0u, slot == static_cast<int>(i))) continue;
            for (uint32_t c = 0; c < a.rp; c += 8) {
                float v[8];
                tmem_load8(tmem + (warp << 21) + i * a.rp + c, v);
                if (slot == static_cast<int>(i)) {
#pragma unroll
                    for (uint32_t e = 0; e < 8; e++) part[(c + e) * H_PITCH + tid] = v[e];
                }
            }
        }
        tc_before();
    }
    __syncwarp();
    if (a.split > 1) cluster_barrier();
    else __syncthreads();
    if (!*over) {                                                // a CTA's share of the tokens: the sums of all, in order, eight at a time
        const Peers peers(ring, a.split);
        const uint32_t each = H_TOKENS / a.split, lo = rank * each;
        for (uint32_t e = tid; e < each * (a.rp / 8); e += H_THREADS) {
            const uint32_t row = lo + e % each, c = e / each * 8;
            const int slot = s.slot[row] - static_cast<int>(from);
            if (slot < 0 || slot >= static_cast<int>(count)) continue;
            const float scale = a.index.scale_of(s.adapter[row]);
            float sum[8];
            peers.sum8((c * H_PITCH + row) * 4, H_PITCH * 4, sum);
            Vec<Thin, 16> upper, lower;
#pragma unroll
            for (uint32_t q = 0; q < 8; q++) {
                sum[q] = c + q < a.rank ? sum[q] * scale : 0.0f;
                split_halves(sum[q], upper.e[q], lower.e[q]);
            }
            Thin *to = a.h + (t0 + row) * 2 * a.rp + c;
            *reinterpret_cast<uint4 *>(to) = upper.raw;
            *reinterpret_cast<uint4 *>(to + a.rp) = lower.raw;
            if (a.kept) {
                const uint64_t t = sorted ? a.sorted.order[t0 + row] : t0 + row;
                if constexpr (__is_same(T, __half)) {
                    float4 *wide = reinterpret_cast<float4 *>(static_cast<float *>(a.kept) + t * a.rp + c);
                    wide[0] = make_float4(sum[0], sum[1], sum[2], sum[3]), wide[1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
                } else {
                    to = static_cast<Thin *>(a.kept) + t * 2 * a.rp + c;
                    *reinterpret_cast<uint4 *>(to) = upper.raw;
                    *reinterpret_cast<uint4 *>(to + a.rp) = lower.raw;
                }
            }
        }
    }
    if (a.split > 1) cluster_barrier();                          // nobody leaves while another reads its sums
    tc_before();
    __syncthreads();
    if (warp == 5) {
        tc_after();
        tmem_free(tmem, a.tmem_columns);
    }
}

}  // namespace lmz
