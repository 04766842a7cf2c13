// The projection through a shared weight with low-rank adapters beside it, and by the same kernel the gradient of its input.
#pragma once
#include "adapter_kernels.cuh"
#include "slot_ring.cuh"
#include "tcgen.cuh"

#include <type_traits>

namespace lmz {

constexpr uint32_t P_FEATS = 128;              // features of a tile: the tensor core's M, a TMEM lane each
constexpr uint32_t P_TOKENS = 256;             // most tokens of a tile: its N, a TMEM column each
constexpr uint32_t P_GROUP = 16;               // tokens of a TMEM load, and the steps that N comes in (a pair's: 32)
constexpr uint32_t P_INFOS = 3, P_MAX_STAGES = 10, P_MAX_SLOTS = 8;
constexpr uint32_t P_SLOT_BYTES = P_GROUP * P_FEATS * 4, P_PLACES = 64;     // places of the rank that mixed groups take at a time
constexpr uint32_t P_EPILOGUE = 128, P_FEED = 128, P_THREADS = P_EPILOGUE + P_FEED + 64;

// What a tile's tokens have for adapters.
struct TileInfo {
    int32_t adapter[P_TOKENS];                 // per token, -1: none
    uint32_t mixed;                            // bit per group: its tokens have different adapters
    uint32_t runs;
    struct { int32_t adapter; uint32_t column, tokens; } run[P_TOKENS / P_GROUP];
};

struct ProjectShared {
    uint64_t full[P_MAX_STAGES], empty[P_MAX_STAGES];
    uint64_t info_full[P_INFOS], info_empty[P_INFOS];
    uint64_t sums_full[2], sums_empty[2];
    uint64_t slot_full[P_MAX_SLOTS], slot_empty[P_MAX_SLOTS];
    uint32_t tmem, over;
    uint32_t same[P_TOKENS / 32];              // bit 0, 1: the tokens of these two sixteens have one adapter; bit 2: both the same
    TileInfo info[P_INFOS];
};

template <class T>
struct ProjectArgs {
    CUtensorMap x, w;
    CUtensorMap xs;                            // x in the order of `sorted`
    CUtensorMap h, f;                          // hidden as tokens x 2 x rp, and the factors as adapters x their two sides (F16:
                                               // as slots x 2 x those, in BF16)
    TokenIndex index;
    SortedTokens sorted;
    const Thin *hidden;                        // [token][2][rp]: the thin product, its upper and its lower half (in that order if x is)
    const T *factor;                           // of adapter i from i * factor_each; rows of factor_row elements, multiples of 8
    const uint32_t *slot;                      // F16: where an adapter's parts are (k_parts)
    uint64_t factor_each, factor_row;
    T *y;
    uint64_t tokens, feats;
    uint32_t rank, rp;                         // rp: rank up to a multiple of 8
    uint32_t steps;                            // of 64 along K
    uint32_t nt;                               // tokens of a tile
    uint32_t split;                            // CTAs of a cluster that share K
    uint32_t feat_tiles, token_tiles;          // of P_FEATS (a pair: twice that) and nt
    uint32_t stages, stage_bytes, tmem_columns;
    uint32_t slots;                            // mixed groups' sums that wait for their way out
};

// Tiles of a stage: W's 128 rows, and the tokens' (of a pair's 256 each CTA has half).
__host__ __device__ constexpr uint32_t project_stage_bytes(uint32_t nt, bool pair) { return (P_FEATS + (pair ? nt / 2 : nt)) * ROW_BYTES; }

// Of sixteen tokens' adapters, factors [feature][rank]: L threads have a feature's up to 64 places of the rank, eight each, so
// that a warp's load is of whole lines; their sums meet by shuffles, in which each thread ends with another feature's.
// `factor`: at the tile's first feature and place, of adapter 0; `live`: the tile's features; `left`: places, from here on.
template <class T, uint32_t L>
__device__ __forceinline__ void mixed_rows(const T *factor, uint64_t factor_each, uint32_t factor_row, uint32_t live, uint32_t left, const int32_t *adapter,
                                        uint32_t id, bool add, const float *places, float *slot)
{
    constexpr uint32_t FLIGHT = 16, BATCH = FLIGHT / L;          // loads under way
    const uint32_t part = id % L, row = id / L;
    auto load = [&](int i, Vec<T, 16> *fac) {
        const T *p = factor + (i < 0 ? 0 : i) * factor_each + part * 8;
#pragma unroll
        for (uint32_t m = 0; m < L; m++) {
            const uint32_t f = row + m * (P_FEATS / L);
            fac[m].raw = {};
            if (i >= 0 && f < live && part * 8 < left) fac[m].raw = *reinterpret_cast<const uint4 *>(p + static_cast<uint64_t>(f) * factor_row);
        }
    };
    auto give = [&](uint32_t c, const Vec<T, 16> *fac) {
        float h[8], v[L];
        *reinterpret_cast<float4 *>(h) = *reinterpret_cast<const float4 *>(places + c * P_PLACES + part * 8);
        *reinterpret_cast<float4 *>(h + 4) = *reinterpret_cast<const float4 *>(places + c * P_PLACES + part * 8 + 4);
#pragma unroll
        for (uint32_t m = 0; m < L; m++) {
            v[m] = 0;
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) v[m] += h[e] * widen(fac[m].e[e]);
        }
#pragma unroll
        for (uint32_t o = L / 2; o; o /= 2)
#pragma unroll
            for (uint32_t m = 0; m < o; m++) {
                const float other = part & o ? v[m] : v[m + o], own = part & o ? v[m + o] : v[m];
                v[m] = own + __shfl_xor_sync(~0u, other, o);
            }
        float &to = slot[c * P_FEATS + row + part * (P_FEATS / L)];
        to = add ? to + v[0] : v[0];
    };
    uint32_t runs = 1;
#pragma unroll
    for (uint32_t c = 1; c < P_GROUP; c++) runs += adapter[c] != adapter[c - 1];
    if (runs <= L / 2) {                                         // (where an adapter's tokens end: fewer loads to wait for than batches)
        for (uint32_t c = 0; c < P_GROUP;) {
            Vec<T, 16> fac[L];
            const int i = adapter[c];
            load(i, fac);
            do give(c++, fac);
            while (c < P_GROUP && adapter[c] == i);
        }
        return;
    }
    for (uint32_t c0 = 0; c0 < P_GROUP; c0 += BATCH) {
        Vec<T, 16> fac[BATCH][L];
#pragma unroll
        for (uint32_t c = 0; c < BATCH; c++) load(adapter[c0 + c], fac[c]);
#pragma unroll
        for (uint32_t c = 0; c < BATCH; c++) give(c0 + c, fac[c]);
    }
}

// What the adapters add to a tile's features of sixteen tokens that have different ones, into `slot` ([token][feature]), by
// four warps.  Not on the tensor core: a factor multiplied by the zeros of tokens it does not belong to would
// still hand them its infinities and NaN.  Bound by the latency of the factors' loads, of which a thread has sixteen
// under way; `places`: room for 64 places of the rank of the tokens' h.
template <class T, bool MN>
__device__ __forceinline__ void mixed_group(const ProjectArgs<T> &a, const int32_t *adapter, uint64_t t0, uint64_t f0, uint32_t id, uint32_t barrier, float *places, float *slot)
{
    float sum[P_GROUP] = {};                                     // MN: two tokens' eight features
    const uint32_t fg = id & 15, tg = id >> 4;
    for (uint32_t j0 = 0; j0 < a.rp; j0 += P_PLACES) {
        sync_threads(barrier, P_FEED);
        {
            const uint32_t c = id >> 3, j = j0 + (id & 7) * 8;
            Vec<Thin, 16> upper, lower;
            upper.raw = lower.raw = {};
            if (adapter[c] >= 0 && j < a.rp) {
                const Thin *h = a.hidden + (t0 + c) * 2 * a.rp + j;
                upper.raw = *reinterpret_cast<const uint4 *>(h), lower.raw = *reinterpret_cast<const uint4 *>(h + a.rp);
            }
            float v[8];
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) v[e] = widen(upper.e[e]) + widen(lower.e[e]);
            float4 *to = reinterpret_cast<float4 *>(places + c * P_PLACES + (id & 7) * 8);
            to[0] = make_float4(v[0], v[1], v[2], v[3]), to[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
        sync_threads(barrier, P_FEED);
        if constexpr (MN) {
            constexpr uint32_t BATCH = 16;
            for (uint32_t j1 = 0; j1 < P_PLACES && j0 + j1 < a.rp; j1 += BATCH) {
#pragma unroll
                for (uint32_t half = 0; half < 2; half++) {
                    const uint32_t c = tg + half * 8;
                    const int i = adapter[c];
                    const uint64_t f = f0 + fg * 8;
                    if (i < 0 || f >= a.feats) continue;
                    const T *p = a.factor + i * a.factor_each + (j0 + j1) * a.factor_row + f;
                    Vec<T, 16> fac[BATCH];
#pragma unroll
                    for (uint32_t j = 0; j < BATCH; j++) {
                        fac[j].raw = {};
                        if (j0 + j1 + j < a.rank) fac[j].raw = *reinterpret_cast<const uint4 *>(p + j * a.factor_row);
                    }
#pragma unroll
                    for (uint32_t j = 0; j < BATCH; j++) {
                        const float h = places[c * P_PLACES + j1 + j];
                        if (j0 + j1 + j < a.rank) {
#pragma unroll
                            for (uint32_t e = 0; e < 8; e++) sum[half * 8 + e] += h * widen(fac[j].e[e]);
                        }
                    }
                }
            }
        } else {
            const T *factor = a.factor + f0 * a.factor_row + j0;
            const uint32_t live = a.feats > f0 ? static_cast<uint32_t>(a.feats - f0 < P_FEATS ? a.feats - f0 : P_FEATS) : 0, left = a.rp - j0;
            const uint32_t row = static_cast<uint32_t>(a.factor_row);
            if (left > 32) mixed_rows<T, 8>(factor, a.factor_each, row, live, left, adapter, id, j0 != 0, places, slot);
            else if (left > 16) mixed_rows<T, 4>(factor, a.factor_each, row, live, left, adapter, id, j0 != 0, places, slot);
            else if (left > 8) mixed_rows<T, 2>(factor, a.factor_each, row, live, left, adapter, id, j0 != 0, places, slot);
            else mixed_rows<T, 1>(factor, a.factor_each, row, live, left, adapter, id, j0 != 0, places, slot);
        }
    }
    if constexpr (MN) {
#pragma unroll
        for (uint32_t half = 0; half < 2; half++) {
            float *to = slot + (tg + half * 8) * P_FEATS + fg * 8;
            *reinterpret_cast<float4 *>(to) = make_float4(sum[half * 8], sum[half * 8 + 1], sum[half * 8 + 2], sum[half * 8 + 3]);
            *reinterpret_cast<float4 *>(to + 4) = make_float4(sum[half * 8 + 4], sum[half * 8 + 5], sum[half * 8 + 6], sum[half * 8 + 7]);
        }
    }
    sync_threads(barrier, P_FEED);
}

// Two tokens' sums of a lane's feature, to y: where rows allow it two lanes exchange halves, so that a store has two features.
template <class T, bool SORTED>
__device__ __forceinline__ void store_two(const ProjectArgs<T> &a, uint64_t t, uint64_t f, bool pairs, float v0, float v1)
{
    auto row = [&](uint64_t t) {
        if constexpr (SORTED) t = a.sorted.order[t];
        return a.y + t * a.feats;
    };
    const uint32_t odd = threadIdx.x & 1;
    if (pairs) {
        const float got = __shfl_xor_sync(~0u, odd ? v0 : v1, 1);
        union { T e[2]; uint32_t raw; } both;
        both.e[0] = narrow<T>(odd ? got : v0);
        both.e[1] = narrow<T>(odd ? v1 : got);
        if (t + odd < a.tokens && f < a.feats) *reinterpret_cast<uint32_t *>(row(t + odd) + (f & ~1ull)) = both.raw;
    } else if (f < a.feats) {
        if (t < a.tokens) row(t)[f] = narrow<T>(v0);
        if (t + 1 < a.tokens) row(t + 1)[f] = narrow<T>(v1);
    }
}

// y[t][f] = sum over k of x[t][k] W(f, k) + sum over j of h[t][j] F_i(f, j), i = index[t].
// MN false: W is [f][k], F_i [f][j] (the projection).  MN true: W is [k][f], F_i [j][f] (the gradient of its input: x is
// dy, k runs over the output's features, h is g).
//
// Features are the tensor core's M and tokens its N, whatever their number: a single token streams the weight past 16 columns,
// a prompt past 256, and what an adapter adds to a run of its own tokens is one more product into just their columns.
//
// Roles: a TMA warp loads tiles of W and x (64 along K) into a ring of stages, and behind them, for every run of tokens with
// one adapter, tiles of its factor and of either half of h; a warp issues the MMAs; four warps look at the next tile's tokens
// and work out what has no run (mixed_group); four take the sums out of TMEM, which holds two tiles' sums, so that a tile's way
// out runs under the next tile's products.
// Tokens that came scattered are taken in the order of their adapters: x has been copied into it, y's rows are found by it.
// The weight's first tiles are under way while the kernel that makes h still runs.
// Few tiles: the CTAs of a cluster share K, and their sums meet in distributed shared memory.
// Many (PAIR): two CTAs multiply 256 features by 256 tokens together, each loading half of both, so that a step brings
// 32 KiB into an SM for the products that took 48.
//
// One B200, kernel alone: 8192 tokens of 4096 to 14336 features at rank 64 633 us, the gradient of its input 617 us (the tensor
// pipe 91 and 93 % active: 1.54 and 1.59 PFLOP/s); 4096 tokens 4096 x 4096 of eight adapters 114 us (a fifth of that in a last
// wave of tiles that fills half of the multiprocessors); 64 tokens of 48 adapters 4096 x 14336 35 to 40 us, bound by reading
// the weight (22 us) and then by the mixed groups' factors; one token 4096 x 4096 19 us, of which the weight is 6.
template <class T, bool MN, bool PAIR>
__global__ void __launch_bounds__(P_THREADS, 1) k_project(const __grid_constant__ ProjectArgs<T> a)
{
    constexpr uint32_t CTAS = PAIR ? 2 : 1, GROUP = CTAS * P_GROUP;
    extern __shared__ uint8_t p_smem[];
    __shared__ ProjectShared s;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t side = PAIR ? cluster_rank() : 0, rank = !PAIR && a.split > 1 ? cluster_rank() : 0;
    const uint32_t team = PAIR ? 2 : a.split;
    const uint32_t first = blockIdx.x / team, stride = gridDim.x / team, tiles = a.feat_tiles * a.token_tiles;
    const uint32_t k0 = static_cast<uint32_t>(static_cast<uint64_t>(a.steps) * rank / a.split);
    const uint32_t k1 = static_cast<uint32_t>(static_cast<uint64_t>(a.steps) * (rank + 1) / a.split);
    const uint32_t ring = (smem_addr(p_smem) + ATOM_BYTES - 1) & ~(ATOM_BYTES - 1);
    uint8_t *const local = p_smem + (ring - smem_addr(p_smem));
    float *const slots = reinterpret_cast<float *>(local + a.stages * a.stage_bytes), *const room = slots + a.slots * (P_SLOT_BYTES / 4);
    volatile uint32_t *over = &s.over;
    const bool sorted = a.sorted.on();                           // (found before the kernel in front could let this one start)

    if (tid == 0) {
        s.over = 0;
        for (uint32_t i = 0; i < a.stages; i++) bar_init(&s.full[i], CTAS), bar_init(&s.empty[i], 1);
        for (uint32_t i = 0; i < P_INFOS; i++) bar_init(&s.info_full[i], 1), bar_init(&s.info_empty[i], (side ? 1 : 2) + P_EPILOGUE / 32);
        for (uint32_t i = 0; i < 2; i++) bar_init(&s.sums_full[i], 1), bar_init(&s.sums_empty[i], CTAS * P_EPILOGUE / 32);
        for (uint32_t i = 0; i < a.slots; i++) bar_init(&s.slot_full[i], 1), bar_init(&s.slot_empty[i], P_EPILOGUE / 32);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if constexpr (PAIR) {
        __syncthreads();
        cluster_barrier();
    }
    if (warp == 9) tmem_alloc<PAIR>(&s.tmem, a.tmem_columns);
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = s.tmem;

    // Eight token tiles side by side, features outside: what a wave reads of x and W stays in L2.
    auto place = [&](uint32_t tile, uint32_t &ft, uint32_t &tt) {
        const uint32_t band = 8 * a.feat_tiles, b = tile / band, in = tile - b * band;
        const uint32_t w = a.token_tiles - 8 * b < 8 ? a.token_tiles - 8 * b : 8;
        ft = in / w, tt = 8 * b + in % w;
    };
    constexpr uint32_t PARTS = __is_same(T, __half) ? 2 : 1;     // of a factor
    const uint32_t places = (a.rp + STEP_K - 1) / STEP_K;        // steps of a run, for each half of h and each part of the factor
    auto mine = [&](uint32_t run) { return run % a.split == rank; };
    auto mixed = [&](const TileInfo &info, uint32_t g) { return (info.mixed >> g & 1) && (a.split == 1 || g % a.split == rank); };
    auto features = [&](uint32_t ft) { return (ft * CTAS + side) * P_FEATS; };      // where this CTA's begin

    auto add_slot = [&](RingPlace &slot, float *v) {             // a mixed group's sums
        if (!warp_wait(&s.slot_full[slot.stage], slot.turn & 1, over)) return false;
        const float *from = slots + slot.stage * (P_SLOT_BYTES / 4) + tid;
#pragma unroll
        for (uint32_t c = 0; c < P_GROUP; c++) v[c] += from[c * P_FEATS];
        __syncwarp();
        if (lane == 0) bar_arrive(&s.slot_empty[slot.stage]);
        slot.next(a.slots);
        return true;
    };

    if (warp == 8) {
        RingPlace at;
        uint32_t n = 0;
        const uint32_t full = peer_addr(s.full, 0);
        bool h_here = false;                                     // (the kernel before has made h)
        for (uint32_t tile = first; tile < tiles; tile += stride, n++) {
            uint32_t ft, tt;
            place(tile, ft, tt);
            const uint32_t f = features(ft), t = tt * a.nt + side * (P_TOKENS / 2);
            bool ok = true;
            for (uint32_t k = k0; k < k1; k++, at.next(a.stages)) {
                const uint32_t st = at.stage;
                ok = !at.turn || warp_wait(&s.empty[st], (at.turn - 1) & 1, over);
                if (!ok) break;
                if (elected()) {
                    const uint32_t dst = ring + st * a.stage_bytes;
                    const uint32_t bar = PAIR ? full + st * 8 : smem_addr(&s.full[st]);
                    if (side) peer_expect(bar, a.stage_bytes);
                    else bar_expect(&s.full[st], a.stage_bytes);
                    if constexpr (MN) {
                        tma_load_2d<PAIR>(&a.w, bar, dst, f, k * STEP_K);
                        tma_load_2d<PAIR>(&a.w, bar, dst + STEP_K * ROW_BYTES, f + 64, k * STEP_K);
                    } else {
                        tma_load_2d<PAIR>(&a.w, bar, dst, k * STEP_K, f);
                    }
                    tma_load_2d<PAIR>(sorted ? &a.xs : &a.x, bar, dst + P_FEATS * ROW_BYTES, k * STEP_K, t);
                }
                __syncwarp();
            }
            ok = ok && warp_wait(&s.info_full[n % P_INFOS], (n / P_INFOS) & 1, over);
            if (!ok) break;
            const TileInfo &info = s.info[n % P_INFOS];
            for (uint32_t r = 0; r < info.runs && ok; r++) {
                if (!mine(r)) continue;
                const uint32_t token = tt * a.nt + info.run[r].column + side * (info.run[r].tokens / CTAS), adapter = info.run[r].adapter;
                uint32_t plane = adapter;
                if constexpr (PARTS > 1) {
                    if (!h_here) wait_for_previous(), h_here = true;
                    plane = __ldcg(a.slot + adapter) * PARTS;
                }
                for (uint32_t q = 0; q < 2 * PARTS && ok; q++) {          // the factor's parts with the upper half, then with the lower
                    const uint32_t half = q / PARTS;
                    for (uint32_t j0 = 0; j0 < places * STEP_K; j0 += STEP_K, at.next(a.stages)) {
                        const uint32_t st = at.stage;
                        ok = !at.turn || warp_wait(&s.empty[st], (at.turn - 1) & 1, over);
                        if (!ok) break;
                        if (elected()) {
                            const uint32_t dst = ring + st * a.stage_bytes, bar = PAIR ? full + st * 8 : smem_addr(&s.full[st]);
                            if (side) peer_expect(bar, a.stage_bytes);
                            else bar_expect(&s.full[st], a.stage_bytes);
                            if constexpr (MN) {
                                tma_load_3d<PAIR>(&a.f, bar, dst, f, j0, plane + q % PARTS);
                                tma_load_3d<PAIR>(&a.f, bar, dst + STEP_K * ROW_BYTES, f + 64, j0, plane + q % PARTS);
                            } else {
                                tma_load_3d<PAIR>(&a.f, bar, dst, j0, f, plane + q % PARTS);
                            }
                        }
                        __syncwarp();
                        if (!h_here) wait_for_previous(), h_here = true;
                        if (elected()) tma_load_3d<PAIR>(&a.h, PAIR ? full + st * 8 : smem_addr(&s.full[st]), ring + st * a.stage_bytes + P_FEATS * ROW_BYTES, j0, half, token);
                        __syncwarp();
                    }
                }
            }
            if (!ok) break;
            __syncwarp();
            if (lane == 0) bar_arrive(&s.info_empty[n % P_INFOS]);
        }
        // Nothing may still be on its way into this block's memory (a pair's barriers are the first CTA's, and stand for both).
        if (*over && !side)
            for (uint32_t i = 0; i < a.stages; i++) {
                const uint32_t used = at.turn - (i >= at.stage);                 // the last turn that filled this stage
                if (used != ~0u) bar_drain(&s.full[i], used & 1);
            }
    } else if (warp == 9) {
        if (!side) {
            const uint32_t a_step = MN ? 16 * ROW_BYTES : 32, a_block = MN ? STEP_K * ROW_BYTES : 16;
            constexpr bool bf16 = __is_same(T, __nv_bfloat16);
            RingPlace at;
            uint32_t n = 0;
            const uint32_t desc = mma_desc(bf16, MN, false, CTAS * P_FEATS, a.nt);
            const uint32_t a_lo = desc_lo(ring, a_block), b_lo = desc_lo(ring + P_FEATS * ROW_BYTES, 16);
            bool ok = true;
            for (uint32_t tile = first; tile < tiles; tile += stride, n++) {
                const uint32_t buf = n & 1, sums = tmem + buf * a.nt;
                ok = n < 2 || warp_wait(&s.sums_empty[buf], (n / 2 - 1) & 1, over);
                if (!ok) break;
                tc_after();
                for (uint32_t k = k0; k < k1; k++, at.next(a.stages)) {
                    const uint32_t st = at.stage, off = st * a.stage_bytes >> 4;
                    ok = warp_wait(&s.full[st], at.turn & 1, over);
                    if (!ok) break;
                    if (elected()) {
#pragma unroll
                        for (uint32_t c = 0; c < STEP_K / 16; c++)
                            mma16<PAIR>(sums, a_lo + off + (c * a_step >> 4), b_lo + off + c * 2, desc, k != k0 || c);
                        mma_commit<PAIR>(&s.empty[st]);
                    }
                    __syncwarp();
                }
                ok = ok && warp_wait(&s.info_full[n % P_INFOS], (n / P_INFOS) & 1, over);
                if (!ok) break;
                const TileInfo &info = s.info[n % P_INFOS];
                for (uint32_t r = 0; r < info.runs && ok; r++) {
                    if (!mine(r)) continue;
                    const uint32_t column = info.run[r].column, rdesc = mma_desc(true, MN, false, CTAS * P_FEATS, info.run[r].tokens);
                    for (uint32_t q = 0; q < 2 * PARTS && ok; q++)
                        for (uint32_t j0 = 0; j0 < places * STEP_K; j0 += STEP_K, at.next(a.stages)) {
                            const uint32_t st = at.stage, off = st * a.stage_bytes >> 4;
                            ok = warp_wait(&s.full[st], at.turn & 1, over);
                            if (!ok) break;
                            if (elected()) {
                                for (uint32_t c = 0; c < STEP_K / 16 && j0 + c * 16 < a.rp; c++)
                                    mma16<PAIR>(sums + column, a_lo + off + (c * a_step >> 4), b_lo + off + c * 2, rdesc, true);
                                mma_commit<PAIR>(&s.empty[st]);
                            }
                            __syncwarp();
                        }
                }
                if (!ok) break;
                __syncwarp();
                if (elected()) {
                    bar_arrive(&s.info_empty[n % P_INFOS]);
                    mma_commit<PAIR>(&s.sums_full[buf]);
                }
                __syncwarp();
            }
            if (!ok) {                                           // the products under way end before their memory goes
                if (elected()) mma_commit<PAIR>(&s.sums_full[n & 1]);
                __syncwarp();
                bar_drain(&s.sums_full[n & 1], (n / 2) & 1);
            }
        }
    } else if (warp >= 4) {
        const uint32_t id = tid - P_EPILOGUE;
        const TokenIndex index = a.sorted.index(a.index, sorted);
        auto look = [&](uint32_t tile, uint32_t n) {             // the tile's tokens and their adapters
            uint32_t ft, tt;
            place(tile, ft, tt);
            TileInfo &info = s.info[n % P_INFOS];
            if (!sync_all(1, P_FEED, n < P_INFOS || id || bar_wait(&s.info_empty[n % P_INFOS], (n / P_INFOS - 1) & 1, over))) return false;
            const uint64_t t0 = static_cast<uint64_t>(tt) * a.nt;
            for (uint32_t c = id; c < P_TOKENS; c += P_FEED) {
                const bool in = c < a.nt && t0 + c < a.tokens;
                const int i = in ? index.of(t0 + c) : -1;
                info.adapter[c] = i;
                const int head = __shfl_sync(~0u, i, lane & 16);
                const uint32_t agree = __ballot_sync(~0u, !in || i == head);
                const int other = __shfl_sync(~0u, i, 16);
                const bool whole = t0 + c + 16 >= a.tokens || other == i;        // (lane 0's: the halves have the same one)
                if (lane == 0) s.same[c / 32] = ((agree & 0xFFFF) == 0xFFFF) | ((agree >> 16) == 0xFFFF) << 1 | whole << 2;
            }
            sync_threads(1, P_FEED);
            if (id == 0) {
                uint32_t runs = 0, mixed = 0, end = ~0u;
                for (uint32_t g = 0; g * GROUP < a.nt; g++) {
                    const int i = info.adapter[g * GROUP];
                    if (!(PAIR ? s.same[g] == 7 : s.same[g / 2] >> (g & 1) & 1)) {
                        mixed |= (PAIR && t0 + g * GROUP + P_GROUP < a.tokens ? 3u : 1u) << g * CTAS;    // (sixteens that have tokens)
                    } else if (i >= 0) {
                        if (end == g && info.run[runs - 1].adapter == i) info.run[runs - 1].tokens += GROUP;
                        else info.run[runs].adapter = i, info.run[runs].column = g * GROUP, info.run[runs].tokens = GROUP, runs++;
                        end = g + 1;
                    }
                }
                info.mixed = mixed, info.runs = runs;
                bar_arrive(&s.info_full[n % P_INFOS]);
            }
            sync_threads(1, P_FEED);
            return true;
        };
        RingPlace slot;
        uint32_t n = 0;
        bool go = first < tiles && look(first, 0);
        wait_for_previous();                                     // (h)
        for (uint32_t tile = first; go && tile < tiles; tile += stride, n++) {
            if (tile + stride < tiles) go = look(tile + stride, n + 1);
            uint32_t ft, tt;
            place(tile, ft, tt);
            const uint64_t t0 = static_cast<uint64_t>(tt) * a.nt, f0 = features(ft);
            const TileInfo &info = s.info[n % P_INFOS];
            uint32_t order = 0;
            for (uint32_t g = 0; go && g * P_GROUP < a.nt; g++) {
                if (!mixed(info, g)) continue;
                if (slot_by_feed(PAIR, order)) {
                    const bool waits = slot_feed_waits(PAIR, order, slot.turn);
                    go = sync_all(1, P_FEED, !waits || id || bar_wait(&s.slot_empty[slot.stage], (slot.turn - 1) & 1, over));
                    if (!go) break;
                    mixed_group<T, MN>(a, info.adapter + g * P_GROUP, t0 + g * P_GROUP, f0, id, 1, room, slots + slot.stage * (P_SLOT_BYTES / 4));
                    if (id == 0) bar_arrive(&s.slot_full[slot.stage]);
                }
                order++;
                slot.next(a.slots);
            }
        }
    } else {
        const bool pairs = a.feats % 2 == 0 && (reinterpret_cast<uint64_t>(a.y) & 3) == 0;
        uint32_t n = 0;
        RingPlace slot;
        wait_for_previous();
        for (uint32_t tile = first; tile < tiles; tile += stride, n++) {
            uint32_t ft, tt;
            place(tile, ft, tt);
            const uint32_t buf = n & 1;
            if (!sync_all(2, P_EPILOGUE, warp_wait(&s.info_full[n % P_INFOS], (n / P_INFOS) & 1, over))) break;
            const TileInfo &info = s.info[n % P_INFOS];
            const uint64_t f = features(ft) + tid, t0 = static_cast<uint64_t>(tt) * a.nt;
            if constexpr (!PAIR) {                               // every other mixed group (each has a slot here) while the sums are made
                RingPlace at = slot;
                uint32_t order = 0;
                for (uint32_t g = 0; g * P_GROUP < a.nt; g++) {
                    if (!mixed(info, g)) continue;
                    if (!slot_by_feed(PAIR, order++)) {
                        mixed_group<T, MN>(a, info.adapter + g * P_GROUP, t0 + g * P_GROUP, features(ft), tid, 2, room + P_GROUP * P_PLACES,
                                           slots + at.stage * (P_SLOT_BYTES / 4));
                        if (tid == 0) bar_arrive(&s.slot_full[at.stage]);
                    }
                    at.next(a.slots);
                }
            }
            if (!warp_wait(&s.sums_full[buf], (n / 2) & 1, over)) break;
            tc_after();
            for (uint32_t g = 0; g * P_GROUP < a.nt; g++) {
                if ((PAIR || a.split == 1) && t0 + g * P_GROUP >= a.tokens) break;
                float v[P_GROUP];
                tmem_load16(tmem + (warp << 21) + buf * a.nt + g * P_GROUP, v);
                if (mixed(info, g) && !add_slot(slot, v)) break;
                if (!PAIR && a.split > 1) {                      // (the stages are free: all products have ended)
                    float *sums = reinterpret_cast<float *>(local);
#pragma unroll
                    for (uint32_t c = 0; c < P_GROUP; c++)
                        if (t0 + g * P_GROUP + c < a.tokens) sums[(g * P_GROUP + c) * P_FEATS + tid] = v[c];
                } else {
                    auto store = [&](auto in_order) {
#pragma unroll
                        for (uint32_t c = 0; c < P_GROUP; c += 2) store_two<T, decltype(in_order)::value>(a, t0 + g * P_GROUP + c, f, pairs, v[c], v[c + 1]);
                    };
                    if (sorted) store(std::true_type{});
                    else store(std::false_type{});
                }
            }
            tc_before();
            __syncwarp();
            if (lane == 0) {
                if (side) peer_arrive(peer_addr(&s.sums_empty[buf], 0));
                else bar_arrive(&s.sums_empty[buf]);
                bar_arrive(&s.info_empty[n % P_INFOS]);
            }
        }
    }
    __syncwarp();
    if (!PAIR && a.split > 1) {                                  // one tile per cluster: every CTA adds up its share of the tokens
        cluster_barrier();
        if (warp < 8 && !*over) {
            uint32_t ft, tt;
            place(first, ft, tt);
            const bool pairs = a.feats % 2 == 0 && (reinterpret_cast<uint64_t>(a.y) & 3) == 0;
            const uint32_t feat = tid & (P_FEATS - 1), share = a.nt / a.split;
            const uint64_t f = static_cast<uint64_t>(ft) * P_FEATS + feat, t0 = static_cast<uint64_t>(tt) * a.nt;
            const uint32_t live = a.tokens - t0 < a.nt ? static_cast<uint32_t>(a.tokens - t0) : a.nt;
            const Peers peers(ring, a.split);
#pragma unroll 2
            for (uint32_t c = rank * share + 2 * (tid / P_FEATS); c < (rank + 1) * share && c < live; c += 4) {
                const float v0 = peers.sum((c * P_FEATS + feat) * 4), v1 = c + 1 < live ? peers.sum(((c + 1) * P_FEATS + feat) * 4) : 0.0f;
                if (sorted) store_two<T, true>(a, t0 + c, f, pairs, v0, v1);
                else store_two<T, false>(a, t0 + c, f, pairs, v0, v1);
            }
        }
        cluster_barrier();
    }
    if constexpr (PAIR) cluster_barrier();                       // nobody's barriers or tiles go while the other may use them
    tc_before();
    __syncthreads();
    if (warp == 9) {
        tc_after();
        tmem_free<PAIR>(tmem, a.tmem_columns);
    }
}

}  // namespace lmz
