// Positions sorted by a whole-number key, stably: what the gradients of rows that several tokens share are summed by.
#pragma once
#include <cooperative_groups.h>
#include <cstdint>

#include "tcgen.cuh"

namespace lmz {

constexpr uint32_t SORT_CTAS = 8, SORT_THREADS = 1024, SORT_WARPS = SORT_THREADS / 32, SORT_DIGIT = 10;
constexpr uint32_t CLEAR_THREADS = 512;
constexpr uint64_t CLEAR_BYTES = 64 << 10;     // of a block

struct SortArgs {
    const void *ids;            // int32 or int64, n of them
    uint64_t n;
    uint64_t nkeys;             // ids outside [0, nkeys) get the key nkeys, and so come last
    uint32_t *keys[2], *pos[2]; // n each: pass p writes to side p & 1
    uint32_t *start;            // NULL, or nkeys + 1: how many keys are below each
    uint32_t *scattered;        // NULL, or a word: 1 if more than a quarter of the sixteens have several keys; without `start`
                                // there is no sort for a 0
    uint32_t passes, digit;     // of `digit` bits of the key, lowest first
    bool wide;                  // ids are int64
};

// Dynamic shared memory for digits of so many bits.
__host__ __device__ constexpr uint32_t sort_smem(uint32_t digit) { return ((SORT_WARPS + 2) << digit) * 4 + SORT_WARPS * 4; }

__device__ __forceinline__ uint32_t sort_key(const SortArgs &a, uint64_t i)
{
    const int64_t id = a.wide ? static_cast<const int64_t *>(a.ids)[i] : static_cast<const int32_t *>(a.ids)[i];
    return id >= 0 && static_cast<uint64_t>(id) < a.nkeys ? static_cast<uint32_t>(id) : static_cast<uint32_t>(a.nkeys);
}

// A radix sort in one cluster, so that the passes follow each other behind the cluster's barrier and not behind a launch
// each.  Every warp owns a run of consecutive elements: it counts its digits, the counts are summed over warps, CTAs (in
// distributed shared memory) and digits, and the warp deals its run out in order, lanes with one digit ranked by a match; so
// equal keys stay in order and every later sum over them has one order.
// Bound by the latency of its passes, so digits are as wide as shared memory holds counters for: 18 bits of a vocabulary in
// two passes.  One B200: 8192 ids of 18 bits 18 us, of 3 bits 8.  (What is launched behind it may start at once.)
static __global__ void __launch_bounds__(SORT_THREADS) k_sort(const SortArgs a)
{
    namespace cg = cooperative_groups;
    extern __shared__ uint32_t sort_words[];
    wait_for_previous();
    let_next_start();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t bins = 1u << a.digit;
    uint32_t *cnt = sort_words;                                 // [warp][bin]: counts, then where the warp's next element goes
    uint32_t *tot = cnt + SORT_WARPS * bins;                    // this CTA's count per bin (read by the others)
    uint32_t *base = tot + bins;                                // where this CTA's elements of a bin start
    uint32_t *sums = base + bins;                               // of the scan over bins, per warp
    const uint32_t ctas = cluster.num_blocks(), me = cluster.block_rank();
    const uint64_t run = ((a.n + ctas * SORT_WARPS - 1) / (ctas * SORT_WARPS) + 31) & ~31ull;
    const uint64_t lo = (me * SORT_WARPS + warp) * run, hi = lo + run < a.n ? lo + run : a.n;
    uint32_t *mine = cnt + warp * bins;
    if (a.scattered) {
        uint32_t mixed = 0;
        for (uint64_t i = static_cast<uint64_t>(me) * SORT_THREADS + tid; i - lane < a.n; i += ctas * SORT_THREADS) {
            const uint32_t k = sort_key(a, i < a.n ? i : a.n - 1), head = __shfl_sync(~0u, k, lane & 16);
            const uint32_t others = __ballot_sync(~0u, i < a.n && k != head);
            mixed += ((others & 0xFFFF) != 0) + (others >> 16 != 0);
        }
        if (lane == 0) sums[warp] = mixed;
        __syncthreads();
        if (tid == 0) {
            for (uint32_t w = 1; w < SORT_WARPS; w++) mixed += sums[w];
            tot[0] = mixed;
        }
        cluster.sync();
        mixed = 0;
        for (uint32_t c = 0; c < ctas; c++) mixed += cluster.map_shared_rank(tot, c)[0];
        const bool scattered = mixed * 64ull > a.n;
        cluster.sync();                                         // (nobody reads `tot` any more)
        if (me == 0 && tid == 0) *a.scattered = scattered;
        if (!scattered && !a.start) return;
    }
    for (uint32_t p = 0; p < a.passes; p++) {
        const uint32_t *ks = a.keys[(p + 1) & 1], *ps = a.pos[(p + 1) & 1];
        uint32_t *kd = a.keys[p & 1], *pd = a.pos[p & 1];
        const uint32_t shift = a.digit * p;
        auto key_at = [&](uint64_t i) { return p ? __ldcg(ks + i) : sort_key(a, i); };
        for (uint32_t i = tid; i < SORT_WARPS * bins / 4; i += SORT_THREADS) reinterpret_cast<uint4 *>(cnt)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        for (uint64_t i = lo; i < hi; i += 32) {
            const bool on = i + lane < hi;
            const uint32_t d = on ? (key_at(i + lane) >> shift) & (bins - 1) : bins + lane;
            const uint32_t same = __match_any_sync(~0u, d);
            if (on && lane == __ffs(same) - 1) mine[d] += __popc(same);
            __syncwarp();
        }
        __syncthreads();
        if (tid < bins) {
            uint32_t c[SORT_WARPS], s = 0;
#pragma unroll
            for (uint32_t w = 0; w < SORT_WARPS; w++) c[w] = cnt[w * bins + tid];
#pragma unroll
            for (uint32_t w = 0; w < SORT_WARPS; w++) {
                cnt[w * bins + tid] = s;
                s += c[w];
            }
            tot[tid] = s;
        }
        cluster.sync();
        uint32_t all = 0, before = 0;
        if (tid < bins)
            for (uint32_t c = 0; c < ctas; c++) {
                const uint32_t t = cluster.map_shared_rank(tot, c)[tid];
                all += t;
                if (c < me) before += t;
            }
        uint32_t scan = all;
        for (uint32_t o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(~0u, scan, o);
            if (lane >= o) scan += v;
        }
        if (lane == 31) sums[warp] = scan;
        __syncthreads();
        if (tid < bins) {
            for (uint32_t w = 0; w < warp; w++) scan += sums[w];
            base[tid] = scan - all + before;
            if (a.start && a.passes == 1 && me == 0 && tid <= a.nkeys) a.start[tid] = scan - all;
        }
        __syncthreads();
        for (uint64_t i = lo; i < hi; i += 32) {
            const bool on = i + lane < hi;
            const uint32_t k = on ? key_at(i + lane) : 0;
            const uint32_t d = on ? (k >> shift) & (bins - 1) : bins + lane;
            const uint32_t same = __match_any_sync(~0u, d);
            uint32_t at = 0;
            if (on) at = mine[d];
            __syncwarp();
            if (on) {
                const uint32_t rank = __popc(same & ((1u << lane) - 1)), to = base[d] + at + rank;
                kd[to] = k;
                pd[to] = p ? __ldcg(ps + i + lane) : static_cast<uint32_t>(i + lane);
                if (rank == 0) mine[d] = at + __popc(same);
            }
            __syncwarp();
        }
        cluster.sync();                                         // (also: nobody reads `tot` any more, all elements are in place)
    }
    if (!a.start || a.passes == 1) return;
    const uint32_t *keys = a.keys[(a.passes - 1) & 1];
    for (uint64_t v = me * SORT_THREADS + tid; v <= a.nkeys; v += ctas * SORT_THREADS) {
        uint64_t l = 0, h = a.n;
        while (l < h) {
            const uint64_t mid = l + (h - l) / 2;
            if (__ldcg(keys + mid) < v) l = mid + 1;
            else h = mid;
        }
        a.start[v] = static_cast<uint32_t>(l);
    }
}

// Zeros, beside the sort launched in front of it and ended no sooner than that.
// (One B200, 1.05 GB: a block per 64 KiB 142 us, as many blocks as fit in strides 170.)
static __global__ void __launch_bounds__(CLEAR_THREADS) k_clear(uint8_t *p, uint64_t bytes)
{
    const uint64_t lo = blockIdx.x * CLEAR_BYTES, hi = lo + CLEAR_BYTES < bytes ? lo + CLEAR_BYTES : bytes, tid = threadIdx.x;
    uint8_t *const to = p + lo;
    if ((reinterpret_cast<uint64_t>(to) & 15) == 0) {
        for (uint64_t i = tid; i < (hi - lo) / 16; i += CLEAR_THREADS) reinterpret_cast<uint4 *>(to)[i] = make_uint4(0, 0, 0, 0);
        if (tid < (hi - lo) % 16) to[(hi - lo) / 16 * 16 + tid] = 0;
    } else {
        for (uint64_t i = tid; i < hi - lo; i += CLEAR_THREADS) to[i] = 0;
    }
    if (blockIdx.x == 0) wait_for_previous();
}

}  // namespace lmz
