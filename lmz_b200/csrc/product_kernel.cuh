// Products of rows with a weight, or with their experts' weights, their epilogue, and both gradients, on the tensor cores.
#pragma once
#include <cuda_fp8.h>

#include "epilogue.cuh"
#include "tcgen.cuh"

namespace lmz {

// out[c][f] = sum over k of A(f, k) B(c, k), the three products that a layer has:
//   FORWARD      f: the output's features, c: rows,                  k: the input's features;  A is the weight, B is x, both with their k side by side
//   ROWS_GRAD    f: the input's features,  c: rows,                  k: the output's features; A is the weight with its f side by side, B is dz
//   WEIGHT_GRAD  f: the input's features,  c: the output's features, k: rows;                  A is x, B is dz, with their f and c side by side
// A group is an expert: in the first two its rows are some of c, in the last they are its k.
enum Product : int { FORWARD, ROWS_GRAD, WEIGHT_GRAD };

constexpr uint32_t G_FEATS = 128;              // features of a tile: the tensor core's M, a TMEM lane each
constexpr uint32_t G_GROUP = 16;               // columns of a TMEM load
constexpr uint32_t G_MAX_STAGES = 10, G_EPILOGUE = 512, G_THREADS = G_EPILOGUE + 96, G_TMA_WARP = G_EPILOGUE / 32;
constexpr uint32_t G_PITCH = 36;               // words from one column to the next where a warp turns 32 lanes' features round
constexpr uint32_t G_TURN_BYTES = G_GROUP / 2 * G_PITCH * 4;  // a warp's
constexpr uint32_t G_BLOCK = STEP_K * ROW_BYTES;              // 64 k of 64 f or c side by side

struct ProductShared {
    uint64_t full[G_MAX_STAGES], empty[G_MAX_STAGES], tail[G_MAX_STAGES];
    uint64_t sums_full[2], sums_empty[2];
    uint32_t tmem, over;
    uint32_t starts[MAX_EXPERTS + 1], tiles[MAX_EXPERTS + 1];  // where a group's rows, and its tiles of columns, begin
};

struct ProductArgs {
    CUtensorMap a, b;
    void *out;                                   // [c][f], a group's behind the one before where k has the groups
    float *z;                                    // the sums and the bias, or NULL
    const void *bias, *times, *residual;         // [group][f], [c][f], [c][f], or NULL
    const float *a_scale, *b_scale;              // per f and per c: of 8-bit operands
    const uint32_t *most;                        // per group: B is dz times a power of two (dz_power) that goes by these; or NULL
    Groups groups;
    uint64_t feats, cols;                        // of f and c (those of c in all groups)
    uint64_t times_stride, residual_stride;
    uint32_t activation;
    uint32_t steps;                              // of 128 bytes along k (not where k has the groups)
    uint32_t nt;                                 // columns of a tile
    uint32_t split, split_log;                   // CTAs of a cluster that share k: a power of two
    uint32_t feat_tiles, col_tiles;              // of G_FEATS (a pair: twice that) and, where c has no groups, of nt
    uint32_t stages, stage_bytes, tmem_columns;
    bool vectors;                                // rows of all tensors that the epilogue has to do with start on 16 bytes
    bool plain;                                  // and they are the result's alone: what else there is goes by feature or by column
};

// Tiles of a stage: A's 128 f, and the columns' (of a pair's each CTA has half); of columns side by side in blocks of 64.
__host__ __device__ constexpr uint32_t product_stage_bytes(uint32_t nt, bool pair, bool side_by_side)
{
    const uint32_t cols = pair ? nt / 2 : nt;
    return (G_FEATS + (side_by_side ? (cols + 63) / 64 * 64 : cols)) * ROW_BYTES;
}

// A tile's place.
struct TilePlace {
    uint32_t group, ft;
    uint32_t c, c_end;                           // its first column, and its group's end
    uint32_t n;                                  // its columns as the products have them: a multiple of 16 (a pair's: 32), nt at most
    uint32_t k, k_rows;                          // WEIGHT_GRAD: the group's rows
};

// N elements in 32 bits.
template <class O, int N>
__device__ __forceinline__ void widen_some(const O *from, float *to)
{
    if constexpr (N * sizeof(O) == 16) {
        Vec<O, 16> v;
#pragma unroll
        for (int e = 0; e < N; e++) v.e[e] = from[e];
        widen_all(v, to);
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) to[e] = widen(from[e]);
    }
}

// Scales (8 bits) whose product, and its product with any sum of 8-bit products (2^-18 to 2^39), stays within 32 bits.  Rows and weights of ordinary size have such;
// other sums are multiplied in 64 bits, one scale after the other, and meet scales of 1 in the epilogue.
__device__ __forceinline__ bool mild(float scale) { return fabsf(scale) >= 0x1p-40f && fabsf(scale) <= 0x1p40f; }
__device__ __forceinline__ float scaled_in_64(float sum, float a, float b) { return static_cast<float>(static_cast<double>(sum) * a * b); }

// N neighbours of f of each of J columns, from sums to result: z = sums + bias, y = act(z) times + residual.  `on`: whether there is such a column.
template <class O, bool SCALED, int J, int N>
__device__ __forceinline__ void finish(const ProductArgs &a, const uint64_t *at, const bool *on, float (*v)[N], const O *bias, const float *a_scale, const float *b_scale,
                                       const O *const *times, const O *const *residual)
{
    if constexpr (SCALED) {
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int e = 0; e < N; e++) v[j][e] *= a_scale[e] * b_scale[j];
    }
    if (a.bias) {
        float w[N];
        widen_some<O, N>(bias, w);
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int e = 0; e < N; e++) v[j][e] += w[e];
    }
    if (a.z) {
#pragma unroll
        for (int j = 0; j < J; j++) {
            if (!on[j]) continue;
            if constexpr (N % 4 == 0) {
#pragma unroll
                for (int e = 0; e < N; e += 4) *reinterpret_cast<float4 *>(a.z + at[j] + e) = make_float4(v[j][e], v[j][e + 1], v[j][e + 2], v[j][e + 3]);
            } else {
                for (int e = 0; e < N; e++) a.z[at[j] + e] = v[j][e];
            }
        }
    }
    act_all<J * N>(a.activation, v[0]);
    if (a.times) {
#pragma unroll
        for (int j = 0; j < J; j++) {
            float w[N];
            widen_some<O, N>(times[j], w);
#pragma unroll
            for (int e = 0; e < N; e++) v[j][e] *= w[e];
        }
    }
    if (a.residual) {
#pragma unroll
        for (int j = 0; j < J; j++) {
            float w[N];
            widen_some<O, N>(residual[j], w);
#pragma unroll
            for (int e = 0; e < N; e++) v[j][e] += w[e];
        }
    }
}

// One of them.
template <class O, bool SCALED>
__device__ __forceinline__ void finish_one(const ProductArgs &a, uint32_t group, uint32_t c, uint64_t f, uint64_t at, float sum)
{
    const O *const times = static_cast<const O *>(a.times) + c * a.times_stride + f, *const residual = static_cast<const O *>(a.residual) + c * a.residual_stride + f;
    const bool on = true;
    float a_scale = 1, b_scale = 1;
    if constexpr (SCALED) {
        a_scale = a.a_scale[f], b_scale = a.b_scale[c];
        if (!mild(a_scale) || !mild(b_scale)) sum = scaled_in_64(sum, a_scale, b_scale), a_scale = b_scale = 1;
    }
    float v[1][1] = {{sum}};
    finish<O, SCALED, 1, 1>(a, &at, &on, v, static_cast<const O *>(a.bias) + group * a.feats + f, &a_scale, &b_scale, &times, &residual);
    static_cast<O *>(a.out)[at] = narrow<O>(v[0][0]);
}

// Features are the tensor core's M and columns its N, whatever their number: a single row streams the weight past 16 columns, a batch past 256.
//
// Roles: a TMA warp loads tiles of A and B (128 bytes along k, or 64 k) into a ring of stages; a warp issues the MMAs; sixteen warps take the
// sums out of TMEM, which holds two tiles' sums, so that a tile's way out runs under the next tile's products (eight warps took 9 to 11 us
// a tile, more than 1024 k's products; these take 5).  They turn 32 features and 16 columns round in shared memory, so that a lane has eight neighbours
// of a row, and what stands in the epilogue comes and goes by 16 bytes, on its way since the sixteen columns before.  Where nothing of the rows' own
// stands in it the results are turned round and not the sums, in half the bytes: the products want shared memory's bandwidth, and the epilogue's
// bytes are time of theirs (16384 rows 1024x4096 100 to 95 us).
//
// Tiles are those of all groups: where the groups' rows begin is found on the device.  A tile ends with its group, to a multiple of 16 columns;
// what is behind the group's last column is another group's rows, whose sums are left where they are (a column's sums are its own).  Where k has
// the groups (WEIGHT_GRAD) the rows behind the group's last are made zeros in both operands' tiles by a warp between the copies and the
// products: of either alone the other's infinities would make NaN.  Only such steps go by that warp (all of them did at first: handing a step on to
// another CTA takes 1 us, and the weight's gradient of 8192 rows 4096x14336 took 2070 us and not 634).
//
// Few tiles: the CTAs of a cluster share k, and their sums meet in distributed shared memory.
// Many (PAIR): two CTAs multiply 256 features by up to 256 columns together, each loading half of both.
//
// Bound by the tensor pipe, whose clock is bound by power, where there are many rows; by reading the weight where there are few.  One B200, us for the
// kernel alone (and its share of the tensor pipe's cycles, at the clock that 1000 W leave, 1.45 to 1.6 GHz by the box): 4096 rows 4096x14336 288 (95 %), with z and
// a factor 344 (80 %), rows' gradient 302 (92 %), weight's 306 (89 %), in 8 bits 148 (90 %); 16384 rows of 16 experts 2048x4096 175, 177 and 216
// (theirs come from HBM for a few tiles each); in a graph one row 4096x14336 21.5 (5.5 TB/s), 4096x4096 9.7.
template <class T, class O, int P, bool PAIR>
__global__ void __launch_bounds__(G_THREADS, 1) k_product(const __grid_constant__ ProductArgs a)
{
    constexpr uint32_t CTAS = PAIR ? 2 : 1, STEP = ROW_BYTES / sizeof(T);
    constexpr bool A_MN = P != FORWARD, B_MN = P == WEIGHT_GRAD, BY_K = P == WEIGHT_GRAD, SCALED = sizeof(T) == 1;
    constexpr bool POWERS = P != FORWARD && __is_same(T, __half);
    static_assert(sizeof(T) == 2 || P == FORWARD);
    extern __shared__ uint8_t g_smem[];
    __shared__ ProductShared s;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t side = PAIR ? cluster_rank() : 0, rank = !PAIR && a.split > 1 ? cluster_rank() : 0;
    const uint32_t team_log = PAIR ? 1 : a.split_log;
    const uint32_t first = blockIdx.x >> team_log, stride = gridDim.x >> team_log;
    const uint32_t ring = (smem_addr(g_smem) + ATOM_BYTES - 1) & ~(ATOM_BYTES - 1);
    uint8_t *const local = g_smem + (ring - smem_addr(g_smem));
    volatile uint32_t *over = &s.over;
    const bool tails = BY_K && a.groups.offsets;                 // (without groups what is behind the last row reads as zeros)

    if (tid == 0) {
        s.over = 0;
        for (uint32_t i = 0; i < a.stages; i++) bar_init(&s.full[i], CTAS), bar_init(&s.empty[i], 1), bar_init(&s.tail[i], 1);
        for (uint32_t i = 0; i < 2; i++) bar_init(&s.sums_full[i], 1), bar_init(&s.sums_empty[i], CTAS * G_EPILOGUE / 32);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if constexpr (PAIR) {
        __syncthreads();
        cluster_barrier();
    }
    if (warp == G_TMA_WARP + 1) tmem_alloc<PAIR>(&s.tmem, a.tmem_columns);
    if (warp == G_TMA_WARP) {
        if (elected()) map_prefetch(&a.a), map_prefetch(&a.b);
        __syncwarp();
        // The weight's first tiles come to L2 while the kernel before still runs (whose tiles is known without it where there are no groups).
        if (!BY_K && !a.groups.offsets) {
            const uint32_t wide = a.col_tiles < 8 ? a.col_tiles : 8;
            const uint32_t f = ((first < a.feat_tiles * wide ? first / wide : first % (8 * a.feat_tiles) / wide) * CTAS + side) * G_FEATS;
            const uint32_t k0 = a.steps * rank >> a.split_log, k1 = a.steps * (rank + 1) >> a.split_log;
            for (uint32_t k = k0; k < k1 && k - k0 < a.stages; k++) {
                if (elected()) {
                    if constexpr (P == FORWARD) {
                        tma_prefetch_3d(&a.a, k * STEP, f, 0);
                    } else if constexpr (P == ROWS_GRAD) {
                        tma_prefetch_3d(&a.a, f, k * STEP, 0);
                        tma_prefetch_3d(&a.a, f + 64, k * STEP, 0);
                    }
                }
                __syncwarp();
            }
        }
    }
    wait_for_previous();
    if (!a.groups.offsets) {
        if (tid == 0) s.starts[0] = s.tiles[0] = 0, s.starts[1] = static_cast<uint32_t>(a.groups.rows), s.tiles[1] = a.col_tiles;
    } else {
        group_starts(a.groups, s.starts);
    }
    if (warp == 0 && !BY_K && a.groups.offsets) {
        __syncwarp();
        uint32_t sum = 0;
        for (uint32_t i0 = 0; i0 <= a.groups.count; i0 += 32) {
            const uint32_t i = i0 + lane, mine = i < a.groups.count ? (s.starts[i + 1] - s.starts[i] + a.nt - 1) / a.nt : 0;
            uint32_t v = mine;
#pragma unroll
            for (uint32_t o = 1; o < 32; o <<= 1) {
                const uint32_t below = __shfl_up_sync(~0u, v, o);
                if (lane >= o) v += below;
            }
            if (i <= a.groups.count) s.tiles[i] = sum + v - mine;
            sum += __shfl_sync(~0u, v, 31);
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = s.tmem, groups = a.groups.count;
    const uint32_t col_tiles = BY_K ? a.col_tiles : s.tiles[groups], tiles = a.feat_tiles * col_tiles * (BY_K ? groups : 1);

    // Group by group, in a group eight column tiles side by side, features outside: what a wave reads of A and B stays in L2.
    auto place = [&](uint32_t tile) {
        TilePlace p;
        p.group = 0;
        uint32_t cols = col_tiles, before = 0;                   // column tiles of the group, and of those in front of it
        if (BY_K) {
            p.group = tile / (a.feat_tiles * col_tiles), before = p.group * col_tiles;
        } else if (groups > 1) {
            p.group = group_of(s.tiles, groups, tile / a.feat_tiles);
            before = s.tiles[p.group], cols = s.tiles[p.group + 1] - before;
        }
        // (a division takes a hundred cycles, which a kernel of few tiles waits for)
        const uint32_t in_group = tile - before * a.feat_tiles;
        const uint32_t band = 8 * a.feat_tiles, b = cols <= 8 ? 0 : in_group / band, in = in_group - b * band;
        const uint32_t w = cols - 8 * b < 8 ? cols - 8 * b : 8;
        p.ft = w == 1 ? in : in / w;
        const uint32_t ct = 8 * b + in - p.ft * w;
        if (BY_K) p.c = ct * a.nt, p.c_end = static_cast<uint32_t>(a.cols), p.k = s.starts[p.group], p.k_rows = s.starts[p.group + 1] - p.k;
        else p.c = s.starts[p.group] + ct * a.nt, p.c_end = s.starts[p.group + 1], p.k = p.k_rows = 0;
        const uint32_t left = (p.c_end - p.c + 16 * CTAS - 1) / (16 * CTAS) * (16 * CTAS);
        p.n = left < a.nt ? left : a.nt;
        return p;
    };
    auto all_steps = [&](const TilePlace &p) { return BY_K ? (p.k_rows + STEP_K - 1) / STEP_K : a.steps; };
    auto step_from = [&](uint32_t steps, uint32_t r) { return steps * r >> a.split_log; };       // (below 2^26 steps, and eight CTAs)
    auto undo = [&](const TilePlace &p) { return POWERS && a.most ? two_to(-dz_power(a.most[p.group])) : 1.0f; };
    auto features = [&](const TilePlace &p) { return (p.ft * CTAS + side) * G_FEATS; };      // where this CTA's begin

    if (warp == G_TMA_WARP) {
        RingPlace at;
        const uint32_t full = peer_addr(s.full, 0), own_tail = peer_addr(s.tail, side);
        uint32_t last_tail = 0, tail_turn = 0;                   // bits per stage: its last use was a tail; how many of its tails there were
        for (uint32_t tile = first; tile < tiles; tile += stride) {
            const TilePlace p = place(tile);
            const uint32_t f = features(p), c = p.c + (PAIR ? side * (p.n / 2) : 0), steps = all_steps(p), k1 = step_from(steps, rank + 1);
            bool ok = true;
            for (uint32_t k = step_from(steps, rank); k < k1; k++, at.next(a.stages)) {
                const uint32_t st = at.stage;
                ok = !at.turn || warp_wait(&s.empty[st], (at.turn - 1) & 1, over);
                if (!ok) break;
                const bool tail = tails && (k + 1) * STEP_K > p.k_rows;
                last_tail = (last_tail & ~(1u << st)) | static_cast<uint32_t>(tail) << st, tail_turn ^= static_cast<uint32_t>(tail) << st;
                if (elected()) {
                    const uint32_t dst = ring + st * a.stage_bytes, to_b = dst + G_FEATS * ROW_BYTES;
                    uint32_t bar = PAIR ? full + st * 8 : smem_addr(&s.full[st]);
                    if (tail) {
                        bar = PAIR ? own_tail + st * 8 : smem_addr(&s.tail[st]);
                        bar_expect(&s.tail[st], a.stage_bytes);
                    } else if (side) {
                        peer_expect(bar, a.stage_bytes);
                    } else {
                        bar_expect(&s.full[st], a.stage_bytes);
                    }
                    if constexpr (P == FORWARD) {
                        tma_load_3d<PAIR>(&a.a, bar, dst, k * STEP, f, p.group);
                    } else if constexpr (P == ROWS_GRAD) {
                        tma_load_3d<PAIR>(&a.a, bar, dst, f, k * STEP, p.group);
                        tma_load_3d<PAIR>(&a.a, bar, dst + G_BLOCK, f + 64, k * STEP, p.group);
                    } else {
                        tma_load_2d<PAIR>(&a.a, bar, dst, f, p.k + k * STEP);
                        tma_load_2d<PAIR>(&a.a, bar, dst + G_BLOCK, f + 64, p.k + k * STEP);
                    }
                    if constexpr (B_MN) {
                        for (uint32_t b = 0; b < a.nt / CTAS; b += 64) tma_load_2d<PAIR>(&a.b, bar, to_b + b * ROW_BYTES, c + b, p.k + k * STEP);
                    } else {
                        tma_load_2d<PAIR>(&a.b, bar, to_b, k * STEP, c);
                    }
                }
                __syncwarp();
            }
            if (!ok) break;
        }
        let_next_start();                                        // (all tensor memory that this kernel wants is its own by now)
        // Nothing may still be on its way into this block's memory (a pair's barriers are the first CTA's, and stand for both; those of tails are each
        // CTA's own).
        if (*over)
            for (uint32_t i = 0; i < a.stages; i++) {
                const uint32_t used = at.turn - (i >= at.stage);                 // the last turn that filled this stage
                if (used == ~0u) continue;
                if (last_tail >> i & 1) bar_drain(&s.tail[i], ~(tail_turn >> i) & 1);
                else if (!side) bar_drain(&s.full[i], used & 1);
            }
    } else if (warp == G_TMA_WARP + 1) {
        if (!side) {
            const uint32_t a_step = A_MN ? 16 * ROW_BYTES : 32, b_step = B_MN ? 16 * ROW_BYTES : 32;
            RingPlace at;
            uint32_t n = 0;
            const uint32_t a_lo = desc_lo(ring, A_MN ? G_BLOCK : 16), b_lo = desc_lo(ring + G_FEATS * ROW_BYTES, B_MN ? G_BLOCK : 16);
            bool ok = true;
            for (uint32_t tile = first; tile < tiles; tile += stride, n++) {
                const TilePlace p = place(tile);
                const uint32_t steps = all_steps(p), k0 = step_from(steps, rank), k1 = step_from(steps, rank + 1);
                const uint32_t buf = n & 1, sums = tmem + buf * a.nt;
                const uint32_t desc = sizeof(T) == 1 ? mma_desc_e4m3(CTAS * G_FEATS, p.n) : mma_desc(__is_same(T, __nv_bfloat16), A_MN, B_MN, CTAS * G_FEATS, p.n);
                ok = n < 2 || warp_wait(&s.sums_empty[buf], (n / 2 - 1) & 1, over);
                if (!ok) break;
                tc_after();
                for (uint32_t k = k0; k < k1; k++, at.next(a.stages)) {
                    const uint32_t st = at.stage, off = st * a.stage_bytes >> 4;
                    ok = warp_wait(&s.full[st], at.turn & 1, over);
                    if (!ok) break;
                    // (a group's last rows: as many sixteens as they take)
                    const uint32_t parts = tails && (k + 1) * STEP_K > p.k_rows ? (p.k_rows - k * STEP_K + 15) / 16 : 4;
                    if (elected()) {
#pragma unroll
                        for (uint32_t q = 0; q < 4; q++) {
                            if (BY_K && q >= parts) break;
                            if constexpr (sizeof(T) == 1) mma32_e4m3<PAIR>(sums, a_lo + off + (q * a_step >> 4), b_lo + off + (q * b_step >> 4), desc, k != k0 || q);
                            else mma16<PAIR>(sums, a_lo + off + (q * a_step >> 4), b_lo + off + (q * b_step >> 4), desc, k != k0 || q);
                        }
                        mma_commit<PAIR>(&s.empty[st]);
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (elected()) mma_commit<PAIR>(&s.sums_full[buf]);
                __syncwarp();
            }
            if (!ok) {                                           // the products under way end before their memory goes
                if (elected()) mma_commit<PAIR>(&s.sums_full[n & 1]);
                __syncwarp();
                bar_drain(&s.sums_full[n & 1], (n / 2) & 1);
            }
        }
    } else if (warp == G_TMA_WARP + 2) {
        if (tails) {                                             // rows that are not the group's become zeros
            RingPlace at;
            uint32_t turns = 0;                                  // bit per stage: the phase that its next tail is
            const uint32_t blocks = a.stage_bytes / G_BLOCK;
            for (uint32_t tile = first; tile < tiles; tile += stride) {
                const TilePlace p = place(tile);
                const uint32_t steps = all_steps(p), n = step_from(steps, rank + 1) - step_from(steps, rank), left = p.k_rows % STEP_K;
                if (n && left && step_from(steps, rank + 1) == steps) {
                    at.skip(n - 1, a.stages);
                    const uint32_t st = at.stage;
                    if (!warp_wait(&s.tail[st], turns >> st & 1, over)) break;
                    turns ^= 1u << st;
                    const uint32_t each = (-left & 15) * 8;                      // 16-byte parts of a block's rows up to the next sixteen
                    for (uint32_t i = lane; i < blocks * each; i += 32)
                        *reinterpret_cast<uint4 *>(local + st * a.stage_bytes + i / each * G_BLOCK + left * ROW_BYTES + i % each * 16) = make_uint4(0, 0, 0, 0);
                    publish_smem();
                    __syncwarp();
                    if (lane == 0) {
                        if (side) peer_arrive(peer_addr(&s.full[st], 0));
                        else bar_arrive(&s.full[st]);
                    }
                    at.next(a.stages);
                } else {
                    at.skip(n, a.stages);
                }
            }
        }
    } else {
        O *const out = static_cast<O *>(a.out);
        const O *const times = static_cast<const O *>(a.times), *const residual = static_cast<const O *>(a.residual);
        const uint32_t quarter = warp & 3, share = warp >> 2;     // of the lanes, and of the groups of columns
        constexpr uint32_t SHARES = G_EPILOGUE / 128;
        float *const turn = reinterpret_cast<float *>(local + a.stages * a.stage_bytes + warp * G_TURN_BYTES);
        if (!BY_K && a.groups.offsets) {                         // rows of no group
            const uint64_t lead = s.starts[0], idle = (lead + (a.cols - s.starts[groups])) * a.feats;
            for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * G_EPILOGUE + tid; i < idle; i += static_cast<uint64_t>(gridDim.x) * G_EPILOGUE)
                out[i < lead * a.feats ? i : i + (s.starts[groups] - lead) * a.feats] = narrow<O>(0.0f);
        }
        uint32_t n = 0;
        for (uint32_t tile = first; tile < tiles; tile += stride, n++) {
            const TilePlace p = place(tile);
            const uint32_t buf = n & 1, steps = all_steps(p);
            const bool any = step_from(steps, rank + 1) > step_from(steps, rank), vectors = a.vectors && a.split == 1;
            const uint64_t plane = BY_K ? p.group * a.cols : 0;
            const uint64_t f = features(p) + quarter * 32 + (vectors ? (lane & 3) * 8 : lane);     // this lane's, eight of them or one
            const uint64_t in = f < a.feats ? f : a.feats - 1;
            auto live = [&](uint32_t g) { return g * G_GROUP < a.nt && p.c + g * G_GROUP < p.c_end; };
            Vec<O, 16> bias, m[2], r[2];
            float a_scale[SCALED ? 8 : 1], b_scale[2];
            // (8 bits) the lane's own feature's scale, and those of two of the warp's columns: are all that its sums meet mild?
            float own_scale = 1, column_scale[2] = {1, 1};
            bool quick = true;
            if (SCALED && vectors) {
                const uint64_t own = features(p) + quarter * 32 + lane;
                if (own < a.feats) own_scale = a.a_scale[own];
#pragma unroll
                for (uint32_t j = 0; j < 2; j++) {
                    const uint32_t g = share + SHARES * (2 * j + (lane >> 4)), c = p.c + g * G_GROUP + (lane & 15);
                    if (live(g) && c < p.c_end) column_scale[j] = a.b_scale[c];
                }
            }
            auto ask = [&](uint32_t g) {                         // what sixteen columns meet in the epilogue
#pragma unroll
                for (uint32_t j = 0; j < 2; j++) {
                    const uint32_t c = p.c + g * G_GROUP + j * 8 + (lane >> 2);
                    m[j].raw = r[j].raw = make_uint4(0, 0, 0, 0);
                    if (SCALED) b_scale[j] = quick && c < p.c_end ? a.b_scale[c] : 1.0f;
                    if (c < p.c_end && f < a.feats) {
                        if (times) m[j].raw = *reinterpret_cast<const uint4 *>(times + c * a.times_stride + f);
                        if (residual) r[j].raw = *reinterpret_cast<const uint4 *>(residual + c * a.residual_stride + f);
                    }
                }
            };
            float f_bias = 0;                                    // of the lane's own feature
            const float by_power = undo(p);
            if (vectors && a.plain) {
                const uint64_t own = features(p) + quarter * 32 + lane;
                if (own < a.feats) {
                    if (a.bias) f_bias = widen(static_cast<const O *>(a.bias)[p.group * a.feats + own]);
                }
            } else if (vectors) {
                bias.raw = make_uint4(0, 0, 0, 0);
                if (a.bias) bias.raw = *reinterpret_cast<const uint4 *>(static_cast<const O *>(a.bias) + p.group * a.feats + (f < a.feats ? f : 0));
                if constexpr (SCALED) {
#pragma unroll
                    for (uint32_t e = 0; e < 8; e++) a_scale[e] = a.a_scale[in + e < a.feats ? in + e : in];
                }
                if (live(share)) ask(share);
                if (times || residual)                           // (the others' come to L2 under the products)
                    for (uint32_t g = share + SHARES; live(g); g += SHARES) {
#pragma unroll
                        for (uint32_t j = 0; j < 2; j++) {
                            const uint32_t c = p.c + g * G_GROUP + j * 8 + (lane >> 2);
                            if (c < p.c_end && f < a.feats) {
                                if (times) asm volatile("prefetch.global.L2 [%0];" ::"l"(times + c * a.times_stride + f));
                                if (residual) asm volatile("prefetch.global.L2 [%0];" ::"l"(residual + c * a.residual_stride + f));
                            }
                        }
                    }
            }
            if (!warp_wait(&s.sums_full[buf], (n / 2) & 1, over)) break;
            tc_after();
            const uint32_t sums = tmem + (quarter << 21) + buf * a.nt;
            float f_scale = own_scale;
            if (SCALED && !__all_sync(~0u, mild(own_scale) && mild(column_scale[0]) && mild(column_scale[1]))) {
                quick = false, f_scale = b_scale[0] = b_scale[1] = 1;
#pragma unroll
                for (uint32_t e = 0; e < 8; e++) a_scale[SCALED ? e : 0] = 1;
            }
            for (uint32_t g = share; live(g); g += SHARES) {
                uint32_t v[G_GROUP];
                __syncwarp();
                tmem_ask16(sums + g * G_GROUP, v);
                tmem_wait16(v);
                if (SCALED && !quick) {
#pragma unroll
                    for (uint32_t j = 0; j < 2; j++) {
#pragma unroll
                        for (uint32_t q = 0; q < 8; q++) turn[q * G_PITCH + lane] = __uint_as_float(v[j * 8 + q]);
#pragma unroll 1
                        for (uint32_t q = 0; q < 8; q++) {
                            const uint32_t c = p.c + g * G_GROUP + j * 8 + q;
                            turn[q * G_PITCH + lane] = scaled_in_64(turn[q * G_PITCH + lane], own_scale, c < p.c_end ? a.b_scale[c] : 0.0f);
                        }
#pragma unroll
                        for (uint32_t q = 0; q < 8; q++) v[j * 8 + q] = __float_as_uint(turn[q * G_PITCH + lane]);
                    }
                    __syncwarp();
                }
                if (vectors && a.plain) {
                    float u[G_GROUP];
#pragma unroll
                    for (uint32_t q = 0; q < G_GROUP; q++) u[q] = !BY_K || any ? __uint_as_float(v[q]) : 0.0f;
                    if constexpr (POWERS) {
#pragma unroll
                        for (uint32_t q = 0; q < G_GROUP; q++) u[q] *= by_power;
                    }
                    if constexpr (SCALED) {
                        const uint32_t c = p.c + g * G_GROUP;
#pragma unroll
                        for (uint32_t q = 0; q < G_GROUP; q += 4) {
                            float4 s4;
                            if (!quick) s4 = make_float4(1, 1, 1, 1);
                            else if (c + q + 3 < a.cols) s4 = *reinterpret_cast<const float4 *>(a.b_scale + c + q);
                            else s4 = make_float4(c + q < a.cols ? a.b_scale[c + q] : 0, c + q + 1 < a.cols ? a.b_scale[c + q + 1] : 0, c + q + 2 < a.cols ? a.b_scale[c + q + 2] : 0, 0);
                            u[q] *= s4.x * f_scale, u[q + 1] *= s4.y * f_scale, u[q + 2] *= s4.z * f_scale, u[q + 3] *= s4.w * f_scale;
                        }
                    }
                    if (a.bias) {
#pragma unroll
                        for (uint32_t q = 0; q < G_GROUP; q++) u[q] += f_bias;
                    }
                    act_all<G_GROUP>(a.activation, u);
                    // two columns to a word on their way round
                    uint32_t *words = reinterpret_cast<uint32_t *>(turn);
#pragma unroll
                    for (uint32_t q = 0; q < 8; q++) words[q * G_PITCH + lane] = narrow_two<O>(u[2 * q], u[2 * q + 1]);
                    __syncwarp();
                    uint32_t w[8];
                    const uint4 *from = reinterpret_cast<const uint4 *>(words + (lane >> 2) * G_PITCH + (lane & 3) * 8);
                    *reinterpret_cast<uint4 *>(w) = from[0], *reinterpret_cast<uint4 *>(w + 4) = from[1];
                    __syncwarp();
                    const uint32_t c = p.c + g * G_GROUP + (lane >> 2) * 2;
                    O *to = out + (plane + c) * a.feats + f;
                    if (f < a.feats) {
                        if (c < p.c_end)
                            *reinterpret_cast<uint4 *>(to) = make_uint4(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410), __byte_perm(w[4], w[5], 0x5410), __byte_perm(w[6], w[7], 0x5410));
                        if (c + 1 < p.c_end)
                            *reinterpret_cast<uint4 *>(to + a.feats) = make_uint4(__byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632), __byte_perm(w[4], w[5], 0x7632), __byte_perm(w[6], w[7], 0x7632));
                    }
                } else if (vectors) {
                    float u[2][8];
#pragma unroll
                    for (uint32_t j = 0; j < 2; j++) {
#pragma unroll
                        for (uint32_t q = 0; q < 8; q++) turn[q * G_PITCH + lane] = __uint_as_float(v[j * 8 + q]);
                        __syncwarp();
                        const float4 *from = reinterpret_cast<const float4 *>(turn + (lane >> 2) * G_PITCH + (lane & 3) * 8);
                        *reinterpret_cast<float4 *>(u[j]) = from[0], *reinterpret_cast<float4 *>(u[j] + 4) = from[1];
                        __syncwarp();
                    }
                    if (BY_K && !any) {
#pragma unroll
                        for (uint32_t e = 0; e < 16; e++) u[e / 8][e % 8] = 0;
                    }
                    uint64_t at[2];
                    bool on[2];
#pragma unroll
                    for (uint32_t j = 0; j < 2; j++) {
                        const uint32_t c = p.c + g * G_GROUP + j * 8 + (lane >> 2);
                        at[j] = (plane + c) * a.feats + f, on[j] = c < p.c_end && f < a.feats;
                    }
                    const O *const ms[2] = {m[0].e, m[1].e}, *const rs[2] = {r[0].e, r[1].e};
                    finish<O, SCALED, 2, 8>(a, at, on, u, bias.e, a_scale, b_scale, ms, rs);
                    if (live(g + SHARES)) ask(g + SHARES);
#pragma unroll
                    for (uint32_t j = 0; j < 2; j++) {
                        Vec<O, 16> y;
                        narrow_all(u[j], y);
                        if (on[j]) *reinterpret_cast<uint4 *>(out + at[j]) = y.raw;
                    }
                } else {
#pragma unroll
                    for (uint32_t q = 0; q < G_GROUP; q++) {
                        const float sum = any ? __uint_as_float(v[q]) : 0.0f;
                        const uint32_t c = p.c + g * G_GROUP + q;
                        if (!PAIR && a.split > 1)                // (the stages are free: all products have ended)
                            reinterpret_cast<float *>(local)[(g * G_GROUP + q) * G_FEATS + quarter * 32 + lane] = sum;
                        else if (c < p.c_end && f < a.feats)
                            finish_one<O, SCALED>(a, p.group, c, f, (plane + c) * a.feats + f, POWERS ? sum * by_power : sum);
                    }
                }
            }
            tc_before();
            __syncwarp();
            if (lane == 0) {
                if (side) peer_arrive(peer_addr(&s.sums_empty[buf], 0));
                else bar_arrive(&s.sums_empty[buf]);
            }
        }
    }
    __syncwarp();
    if (!PAIR && a.split > 1) {                                  // one tile per cluster: every CTA adds up its share of the columns
        cluster_barrier();
        if (warp < G_TMA_WARP && first < tiles && !*over) {
            const TilePlace p = place(first);
            const uint64_t plane = BY_K ? p.group * a.cols : 0;
            // A warp has a column, a lane four neighbours of f.
            const uint32_t share = a.nt >> a.split_log;
            const float by_power = undo(p);
            const uint64_t f = features(p) + lane * 4;
            uint32_t peer[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) peer[i] = peer_addr(local, i < a.split ? i : 0);
#pragma unroll 2
            for (uint32_t q = rank * share + warp; q < (rank + 1) * share && p.c + q < p.c_end; q += G_TMA_WARP) {
                float4 part[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; i++) {
                    part[i] = make_float4(0, 0, 0, 0);
                    if (i < a.split)
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(part[i].x), "=f"(part[i].y), "=f"(part[i].z), "=f"(part[i].w)
                                     : "r"(peer[i] + (q * G_FEATS + lane * 4) * 4) : "memory");
                }
                float v[1][4] = {{part[0].x, part[0].y, part[0].z, part[0].w}};
#pragma unroll
                for (uint32_t i = 1; i < 8; i++) v[0][0] += part[i].x, v[0][1] += part[i].y, v[0][2] += part[i].z, v[0][3] += part[i].w;
                if constexpr (POWERS) v[0][0] *= by_power, v[0][1] *= by_power, v[0][2] *= by_power, v[0][3] *= by_power;
                const uint32_t c = p.c + q;
                const uint64_t at = (plane + c) * a.feats + f;
                if (a.vectors) {
                    if (f >= a.feats) continue;
                    O *const out = static_cast<O *>(a.out);
                    auto four = [&](const void *from, uint64_t i) {
                        Vec<O, 8> w;
                        w.raw = make_uint2(0, 0);
                        if (from) w.raw = *reinterpret_cast<const uint2 *>(static_cast<const O *>(from) + i);
                        return w;
                    };
                    const Vec<O, 8> bias = four(a.bias, p.group * a.feats + f), m = four(a.times, c * a.times_stride + f), r = four(a.residual, c * a.residual_stride + f);
                    float a_scale[4] = {}, b_scale = 0;
                    if constexpr (SCALED) {
                        b_scale = a.b_scale[c];
#pragma unroll
                        for (uint32_t e = 0; e < 4; e++) a_scale[e] = a.a_scale[f + e];
                        if (!mild(b_scale) || !mild(a_scale[0]) || !mild(a_scale[1]) || !mild(a_scale[2]) || !mild(a_scale[3])) {
#pragma unroll
                            for (uint32_t e = 0; e < 4; e++) v[0][e] = scaled_in_64(v[0][e], a_scale[e], b_scale), a_scale[e] = 1;
                            b_scale = 1;
                        }
                    }
                    const bool on = true;
                    const O *const ms = m.e, *const rs = r.e;
                    finish<O, SCALED, 1, 4>(a, &at, &on, v, bias.e, a_scale, &b_scale, &ms, &rs);
                    Vec<O, 8> y;
                    narrow_all(v[0], y);
                    *reinterpret_cast<uint2 *>(out + at) = y.raw;
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < 4; e++)
                        if (f + e < a.feats) finish_one<O, SCALED>(a, p.group, c, f + e, at + e, v[0][e]);
                }
            }
        }
        cluster_barrier();
    }
    if constexpr (PAIR) cluster_barrier();                       // nobody's barriers or tiles go while the other may use them
    tc_before();
    __syncthreads();
    if (warp == G_TMA_WARP + 1) {
        tc_after();
        tmem_free<PAIR>(tmem, a.tmem_columns);
    }
}

// Rows that start on 16 bytes: out[plane][r][c] = in[plane][r][c], and zeros behind a row's last element.  16 bytes of the result a thread.
struct AlignJob {
    const void *in;
    void *out;
    uint64_t plane_stride, row_stride, rows, cols, pitch, total;   // in elements; total: rows of all planes
};
struct AlignArgs {
    AlignJob job[2];
};
constexpr uint32_t ALIGN_THREADS = 256;
template <class E>
__global__ void __launch_bounds__(ALIGN_THREADS) k_align(const __grid_constant__ AlignArgs a)
{
    constexpr uint32_t N = 16 / sizeof(E);
    const AlignJob &j = a.job[blockIdx.y];
    const uint64_t each = j.pitch / N, all = j.total * each;
    wait_for_previous();
    for (uint64_t u = static_cast<uint64_t>(blockIdx.x) * ALIGN_THREADS + threadIdx.x; u < all; u += static_cast<uint64_t>(gridDim.x) * ALIGN_THREADS) {
        const uint64_t row = u / each, plane = row / j.rows, c = (u - row * each) * N;
        const E *in = static_cast<const E *>(j.in) + plane * j.plane_stride + (row - plane * j.rows) * j.row_stride + c;
        union { E e[N]; uint4 raw; } v;
#pragma unroll
        for (uint32_t e = 0; e < N; e++) v.e[e] = c + e < j.cols ? in[e] : E(0);
        reinterpret_cast<uint4 *>(j.out)[u] = v.raw;
    }
}

}  // namespace lmz
