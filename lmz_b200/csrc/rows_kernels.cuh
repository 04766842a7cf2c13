// Rows of an embedding table, and the table's gradient.
#pragma once
#include "tcgen.cuh"
#include "vectors.cuh"

namespace lmz {

constexpr uint32_t ROW_THREADS = 256;

struct RowsArgs {
    const uint8_t *table;
    const void *ids;
    uint8_t *out;
    uint64_t rows, n, row_bytes, stride_bytes;   // stride: from one row of the table to the next
    uint32_t vectors;                            // of a row
    uint32_t lane_log;                           // 2^lane_log threads share a row, at most ROW_THREADS
    float scale;
    bool wide;
};

// y[t] = scale * E[id[t]]; an id outside the table gives a row of zeros.
//
// Bound by HBM: every row read and written once, in vectors of VB bytes (the widest that row size, stride and bases
// allow).  The id has to arrive before the row can be asked for, so a thread keeps U rows on their way.  One B200: 16384 rows of
// 1024 FP32 16.4 us (134 MB written and read, many rows more than once: 8.2 TB/s of L2 and HBM).
template <class T, int VB, int U>
__global__ void __launch_bounds__(ROW_THREADS) k_rows(const RowsArgs a)
{
    using V = Vec<T, VB>;
    const uint32_t lane = threadIdx.x & ((1u << a.lane_log) - 1), sub = threadIdx.x >> a.lane_log;
    const uint32_t per = ROW_THREADS >> a.lane_log;
    const uint64_t t0 = static_cast<uint64_t>(blockIdx.x) * per * U + sub;
    const uint8_t *src[U];
    wait_for_previous();
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint64_t t = t0 + static_cast<uint64_t>(u) * per;
        int64_t id = -1;
        if (t < a.n) id = a.wide ? static_cast<const int64_t *>(a.ids)[t] : static_cast<const int32_t *>(a.ids)[t];
        src[u] = id >= 0 && static_cast<uint64_t>(id) < a.rows ? a.table + static_cast<uint64_t>(id) * a.stride_bytes : nullptr;
    }
    for (uint32_t v = lane; v < a.vectors; v += 1u << a.lane_log) {
        V x[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            x[u].raw = {};
            if (src[u]) x[u].raw = reinterpret_cast<const typename Raw<VB>::type *>(src[u])[v];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint64_t t = t0 + static_cast<uint64_t>(u) * per;
            if (t >= a.n) continue;
            if (a.scale != 1.0f) {                               // (a scale of one leaves every bit as it is)
#pragma unroll
                for (int e = 0; e < V::N; e++) x[u].e[e] = narrow<T>(widen(x[u].e[e]) * a.scale);
            }
            reinterpret_cast<typename Raw<VB>::type *>(a.out + t * a.row_bytes)[v] = x[u].raw;
        }
    }
}

struct RowsGradArgs {
    const uint8_t *dy;
    const uint32_t *keys, *pos;                  // the sorted ids, and the tokens that have them
    float *partial;                              // [window][2][dim]
    uint8_t *out;
    uint64_t row_bytes, dim;
    uint32_t rows, n, window;                    // window: sorted tokens that are summed up in a row
    uint32_t vectors, lane_log;
    float scale;
};

constexpr uint32_t ROWS_STEP = 32;               // tokens whose ids a window has in shared memory at a time

// dE[v] = scale * sum of dy[t] over the tokens t with id v, for the rows that have tokens (the others are zeros already).
// Sums in 32 bits and one order (the tokens' own), no atomics: the same result every time.
//
// A window of sorted tokens after the other: a row whose tokens lie within one is finished there; the others leave a sum
// per window, in slot 0 where they began before it and in slot 1 where they go on behind it, which k_rows_join adds up.
// Bound by reading dy (and, before it, by the zeros of the table's other rows); 8 tokens' rows are under way at a time.  One B200,
// 8192 tokens of 4096 BF16: 27 us here and 9 in k_rows_join, behind 142 of zeros; windows of 16 took 24 and 12.
template <class T, int VB>
__global__ void __launch_bounds__(ROW_THREADS) k_rows_sums(const RowsGradArgs a)
{
    using V = Vec<T, VB>;
    constexpr int N = V::N, AHEAD = 8;
    __shared__ uint32_t s_key[ROW_THREADS / 32][ROWS_STEP + 1], s_pos[ROW_THREADS / 32][ROWS_STEP];
    const uint32_t threads = 1u << a.lane_log, lane = threadIdx.x & (threads - 1), sub = threadIdx.x >> a.lane_log;
    const uint64_t w = static_cast<uint64_t>(blockIdx.x) * (ROW_THREADS >> a.lane_log) + sub;
    const uint32_t v = (blockIdx.z * gridDim.y + blockIdx.y) * ROW_THREADS + lane;
    const uint64_t w0 = w * a.window, w1 = w0 + a.window < a.n ? w0 + a.window : a.n;
    let_next_start();
    wait_for_previous();
    const uint32_t before = w0 && w0 < a.n ? a.keys[w0 - 1] : ~0u;
    float sum[N] = {};
    bool began = true;                                           // the row began in this window
    uint32_t key = ~0u;
    for (uint64_t s0 = w0; s0 < w0 + a.window; s0 += ROWS_STEP) {
        __syncthreads();                                         // (all threads of a block take as many steps)
        for (uint32_t i = lane; i <= ROWS_STEP; i += threads) {
            const uint64_t at = s0 + i;
            s_key[sub][i] = at < a.n ? a.keys[at] : ~0u;
            if (i < ROWS_STEP) s_pos[sub][i] = at < a.n ? a.pos[at] : 0;
        }
        __syncthreads();
        if (v >= a.vectors || s0 >= w1) continue;
        const uint32_t count = w1 - s0 < ROWS_STEP ? static_cast<uint32_t>(w1 - s0) : ROWS_STEP;
        for (uint32_t i = 0; i < count; i += AHEAD) {
            V x[AHEAD];
#pragma unroll
            for (uint32_t j = 0; j < AHEAD; j++) {
                x[j].raw = {};
                if (i + j < count && s_key[sub][i + j] < a.rows)
                    x[j].raw = reinterpret_cast<const typename Raw<VB>::type *>(a.dy + s_pos[sub][i + j] * a.row_bytes)[v];
            }
#pragma unroll
            for (uint32_t j = 0; j < AHEAD; j++) {
                if (i + j >= count) break;
                const uint32_t mine = s_key[sub][i + j];
                if (mine >= a.rows) break;
                if (mine != key) {
                    began = mine != before;                      // (a row before this window can only be its first)
                    key = mine;
#pragma unroll
                    for (int e = 0; e < N; e++) sum[e] = 0;
                }
#pragma unroll
                for (int e = 0; e < N; e++) sum[e] += widen(x[j].e[e]);
                const bool ends = s_key[sub][i + j + 1] != mine, last = s0 + i + j + 1 == w1;
                if (!ends && !last) continue;
                if (ends && began) {
                    V y;
#pragma unroll
                    for (int e = 0; e < N; e++) y.e[e] = narrow<T>(sum[e] * a.scale);
                    reinterpret_cast<typename Raw<VB>::type *>(a.out + mine * a.row_bytes)[v] = y.raw;
                } else {
                    float *to = a.partial + (w * 2 + began) * a.dim + static_cast<uint64_t>(v) * N;
#pragma unroll
                    for (int e = 0; e < N; e++) to[e] = sum[e];
                }
            }
        }
    }
}

// The rows whose tokens lie in more than one window: by the window that they begin in.
template <class T, int VB>
__global__ void __launch_bounds__(ROW_THREADS) k_rows_join(const RowsGradArgs a)
{
    using V = Vec<T, VB>;
    constexpr int N = V::N, AHEAD = 8;
    const uint32_t threads = 1u << a.lane_log, lane = threadIdx.x & (threads - 1), sub = threadIdx.x >> a.lane_log;
    const uint64_t w = static_cast<uint64_t>(blockIdx.x) * (ROW_THREADS >> a.lane_log) + sub;
    const uint32_t v = (blockIdx.z * gridDim.y + blockIdx.y) * ROW_THREADS + lane;
    const uint64_t w0 = w * a.window, w1 = w0 + a.window;
    wait_for_previous();
    if (v >= a.vectors || w1 >= a.n) return;
    const uint32_t key = a.keys[w1 - 1];
    if (key >= a.rows || a.keys[w1] != key || (w0 && a.keys[w0 - 1] == key)) return;
    uint64_t lo = w1, hi = a.n;                                  // where the row's tokens end
    while (lo < hi) {
        const uint64_t mid = lo + (hi - lo) / 2;
        if (a.keys[mid] <= key) lo = mid + 1;
        else hi = mid;
    }
    const uint64_t last = (lo - 1) / a.window;
    const float *from = a.partial + (w * 2 + 1) * a.dim + static_cast<uint64_t>(v) * N;
    float sum[N];
#pragma unroll
    for (int e = 0; e < N; e++) sum[e] = from[e];
    for (uint64_t i = w + 1; i <= last; i += AHEAD) {
        float x[AHEAD][N];
#pragma unroll
        for (int j = 0; j < AHEAD; j++)
#pragma unroll
            for (int e = 0; e < N; e++) x[j][e] = i + j <= last ? a.partial[(i + j) * 2 * a.dim + static_cast<uint64_t>(v) * N + e] : 0.0f;
#pragma unroll
        for (int j = 0; j < AHEAD; j++)
#pragma unroll
            for (int e = 0; e < N; e++) sum[e] += x[j][e];
    }
    V y;
#pragma unroll
    for (int e = 0; e < N; e++) y.e[e] = narrow<T>(sum[e] * a.scale);
    reinterpret_cast<typename Raw<VB>::type *>(a.out + key * a.row_bytes)[v] = y.raw;
}

}  // namespace lmz
