// Positions sorted by a whole-number key, stably: what the gradients of rows that several tokens share are summed by.
#pragma once
#include <cooperative_groups.h>
#include <cstdint>

namespace lmz {

constexpr uint32_t SORT_CTAS = 8, SORT_THREADS = 1024, SORT_WARPS = SORT_THREADS / 32, SORT_BINS = 256;
constexpr uint32_t SORT_SMEM = (SORT_WARPS * SORT_BINS + 3 * SORT_BINS) * 4;

struct SortArgs {
    const void *ids;            // int32 or int64, n of them
    uint64_t n;
    uint64_t nkeys;             // ids outside [0, nkeys) get the key nkeys, and so come last
    uint32_t *keys[2], *pos[2]; // n each: pass p writes to side p & 1
    uint32_t passes;            // of eight bits of the key, lowest first
    bool wide;                  // ids are int64
};

__device__ __forceinline__ uint32_t sort_key(const SortArgs &a, uint64_t i)
{
    const int64_t id = a.wide ? static_cast<const int64_t *>(a.ids)[i] : static_cast<const int32_t *>(a.ids)[i];
    return id >= 0 && static_cast<uint64_t>(id) < a.nkeys ? static_cast<uint32_t>(id) : static_cast<uint32_t>(a.nkeys);
}

// A radix sort by digits of eight bits in one cluster, so that the passes follow each other behind the cluster's barrier
// and not behind a launch each.  Every warp owns a run of consecutive elements: it counts its digits, the counts are
// summed over warps, CTAs (in distributed shared memory) and digits, and the warp deals its run out in order, lanes with
// one digit ranked by a match; so equal keys stay in order and every later sum over them has one order.
// Bound by the latency of its passes (a load, a match and a dependent shared-memory update per 32 elements of a warp).
__global__ void __launch_bounds__(SORT_THREADS) k_sort(SortArgs a)
{
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ uint32_t sort_smem[];
    uint32_t *cnt = sort_smem;                                  // [warp][bin]: counts, then where the warp's next element goes
    uint32_t *tot = cnt + SORT_WARPS * SORT_BINS;               // this CTA's count per bin (read by the others)
    uint32_t *base = tot + SORT_BINS;                           // where this CTA's elements of a bin start
    uint32_t *sums = base + SORT_BINS;                          // of the scan over bins, per warp
    const uint32_t ctas = cluster.num_blocks(), me = cluster.block_rank();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint64_t run = ((a.n + ctas * SORT_WARPS - 1) / (ctas * SORT_WARPS) + 31) & ~31ull;
    const uint64_t lo = (me * SORT_WARPS + warp) * run, hi = lo + run < a.n ? lo + run : a.n;
    uint32_t *mine = cnt + warp * SORT_BINS;
    for (uint32_t p = 0; p < a.passes; p++) {
        const uint32_t *ks = a.keys[(p + 1) & 1], *ps = a.pos[(p + 1) & 1];
        uint32_t *kd = a.keys[p & 1], *pd = a.pos[p & 1];
        const uint32_t shift = 8 * p;
        auto key_at = [&](uint64_t i) { return p ? __ldcg(ks + i) : sort_key(a, i); };
        for (uint32_t i = tid; i < SORT_WARPS * SORT_BINS; i += SORT_THREADS) cnt[i] = 0;
        __syncthreads();
        for (uint64_t i = lo; i < hi; i += 32) {
            const bool on = i + lane < hi;
            const uint32_t d = on ? (key_at(i + lane) >> shift) & 255 : SORT_BINS + lane;
            const uint32_t same = __match_any_sync(~0u, d);
            if (on && lane == __ffs(same) - 1) mine[d] += __popc(same);
            __syncwarp();
        }
        __syncthreads();
        if (tid < SORT_BINS) {
            uint32_t s = 0;
            for (uint32_t w = 0; w < SORT_WARPS; w++) {
                const uint32_t c = cnt[w * SORT_BINS + tid];
                cnt[w * SORT_BINS + tid] = s;
                s += c;
            }
            tot[tid] = s;
        }
        cluster.sync();
        uint32_t all = 0, before = 0, scan = 0;
        if (tid < SORT_BINS) {
            for (uint32_t c = 0; c < ctas; c++) {
                const uint32_t t = cluster.map_shared_rank(tot, c)[tid];
                all += t;
                if (c < me) before += t;
            }
            scan = all;
            for (uint32_t o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(~0u, scan, o);
                if (lane >= o) scan += v;
            }
            if (lane == 31) sums[warp] = scan;
        }
        __syncthreads();
        if (tid < SORT_BINS) {
            for (uint32_t w = 0; w < warp; w++) scan += sums[w];
            base[tid] = scan - all + before;
        }
        __syncthreads();
        for (uint64_t i = lo; i < hi; i += 32) {
            const bool on = i + lane < hi;
            const uint32_t k = on ? key_at(i + lane) : 0;
            const uint32_t d = on ? (k >> shift) & 255 : SORT_BINS + lane;
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
}

// start[v] = how many of the sorted keys are below v, for v in [0, nkeys].
__global__ void __launch_bounds__(256) k_key_starts(const uint32_t *keys, uint32_t n, uint32_t nkeys, uint32_t *start)
{
    const uint64_t v = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (v > nkeys) return;
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (keys[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    start[v] = lo;
}

}  // namespace lmz
