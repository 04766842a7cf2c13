// Rows of an embedding table, and the table's gradient.
#pragma once
#include "sort_kernel.cuh"
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
// allow).  The id has to arrive before the row can be asked for, so a thread keeps U rows on their way.
template <class T, int VB, int U>
__global__ void __launch_bounds__(ROW_THREADS) k_rows(RowsArgs a)
{
    using V = Vec<T, VB>;
    const uint32_t lane = threadIdx.x & ((1u << a.lane_log) - 1), sub = threadIdx.x >> a.lane_log;
    const uint32_t per = ROW_THREADS >> a.lane_log;
    const uint64_t t0 = static_cast<uint64_t>(blockIdx.x) * per * U + sub;
    const uint8_t *src[U];
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
    const uint32_t *keys, *pos, *start;          // the sorted ids, the tokens that have them, and where each row's begin
    float *partial;                              // [window][2][dim]
    uint8_t *out;
    uint64_t rows, row_bytes, dim;
    uint32_t n, window;                          // tokens of a window: a row with more of them is summed window by window
    uint32_t vectors, lane_log;
    float scale;
};

template <class T, int VB>
__device__ __forceinline__ void add_rows(const RowsGradArgs &a, uint32_t from, uint32_t to, uint32_t v, float *sum)
{
    using V = Vec<T, VB>;
    constexpr int AHEAD = 4;
    for (uint32_t i = from; i < to; i += AHEAD) {
        V x[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            x[j].raw = {};
            if (i + j < to) x[j].raw = reinterpret_cast<const typename Raw<VB>::type *>(a.dy + a.pos[i + j] * a.row_bytes)[v];
        }
#pragma unroll
        for (int j = 0; j < AHEAD; j++)
            if (i + j < to) {
#pragma unroll
                for (int e = 0; e < V::N; e++) sum[e] += widen(x[j].e[e]);
            }
    }
}

// The rows that more than `window` tokens have: what each window of sorted tokens adds to the row it begins in and to
// the row it ends in.  (No window holds parts of a third: that row would lie between them, with fewer tokens.)
template <class T, int VB>
__global__ void __launch_bounds__(ROW_THREADS) k_rows_grad_windows(RowsGradArgs a)
{
    constexpr int N = Vec<T, VB>::N;
    const uint32_t v = blockIdx.y * ROW_THREADS + threadIdx.x;
    const uint32_t w0 = blockIdx.x * a.window, w1 = a.n - w0 < a.window ? a.n : w0 + a.window;
    if (v >= a.vectors) return;
    const uint32_t ends[2] = {a.keys[w0], a.keys[w1 - 1]};
#pragma unroll
    for (int side = 0; side < 2; side++) {
        const uint32_t key = ends[side];
        if (key >= a.rows || (side && key == ends[0])) continue;
        const uint32_t s = a.start[key], e = a.start[key + 1];
        if (e - s <= a.window) continue;
        float sum[N] = {};
        add_rows<T, VB>(a, s > w0 ? s : w0, e < w1 ? e : w1, v, sum);
        float *to = a.partial + (static_cast<uint64_t>(blockIdx.x) * 2 + side) * a.dim + static_cast<uint64_t>(v) * N;
#pragma unroll
        for (int i = 0; i < N; i++) to[i] = sum[i];
    }
}

// dE[v] = scale * sum of dy[t] over the tokens t with id v, every row of the gradient written once, zeros for rows
// without tokens.  Sums in 32 bits and one order (the tokens' own), no atomics: the same result every time.
//
// Bound by HBM: dy read and dE written once; for a large vocabulary the zeros are most of it.
template <class T, int VB, int U>
__global__ void __launch_bounds__(ROW_THREADS) k_rows_grad(RowsGradArgs a)
{
    using V = Vec<T, VB>;
    constexpr int N = V::N;
    const uint32_t lane = threadIdx.x & ((1u << a.lane_log) - 1), sub = threadIdx.x >> a.lane_log;
    const uint32_t per = ROW_THREADS >> a.lane_log;
    const uint32_t v = blockIdx.y * ROW_THREADS + lane;
    if (v >= a.vectors) return;
    uint32_t s[U], e[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint64_t row = (static_cast<uint64_t>(blockIdx.x) * U + u) * per + sub;
        s[u] = e[u] = 0;
        if (row < a.rows) s[u] = a.start[row], e[u] = a.start[row + 1];
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint64_t row = (static_cast<uint64_t>(blockIdx.x) * U + u) * per + sub;
        if (row >= a.rows) continue;
        float sum[N] = {};
        if (e[u] - s[u] <= a.window) {
            add_rows<T, VB>(a, s[u], e[u], v, sum);
        } else {
            const uint32_t first = s[u] / a.window, last = (e[u] - 1) / a.window;
            for (uint32_t w = first; w <= last; w++) {
                const uint32_t side = w == first && s[u] != w * a.window;
                const float *from = a.partial + (static_cast<uint64_t>(w) * 2 + side) * a.dim + static_cast<uint64_t>(v) * N;
#pragma unroll
                for (int i = 0; i < N; i++) sum[i] += from[i];
            }
        }
        V y;
#pragma unroll
        for (int i = 0; i < N; i++) y.e[i] = narrow<T>(sum[i] * a.scale);
        reinterpret_cast<typename Raw<VB>::type *>(a.out + row * a.row_bytes)[v] = y.raw;
    }
}

}  // namespace lmz
