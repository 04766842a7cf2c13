// A projection through a shared weight with low-rank adapters of many requests beside it, its gradients, and the merge
// of an adapter into a weight.
//
//   y[t] = x[t] W^T + h[t] B_i^T,  h[t] = s_i x[t] A_i^T,  i = index[t];  no adapter where index[t] is outside [0, n)
//   g[t] = s_i dy[t] B_i,  dx[t] = dy[t] W + g[t] A_i,  dA_i = sum of g[t]^T x[t],  dB_i = sum of dy[t]^T h[t] over i's tokens
#pragma once
#include "tcgen.cuh"
#include "vectors.cuh"

namespace lmz {

// Which adapter a token has.
struct TokenIndex {
    const void *ids;            // int32 or int64; NULL: every token has adapter 0
    const float *scales;        // per adapter, or NULL
    float scale;
    uint32_t n;
    bool wide;
    __device__ __forceinline__ int of(uint64_t t) const
    {
        if (!ids) return 0;
        const int64_t i = wide ? static_cast<const int64_t *>(ids)[t] : static_cast<const int32_t *>(ids)[t];
        return i >= 0 && i < n ? static_cast<int>(i) : -1;
    }
    __device__ __forceinline__ float scale_of(int i) const { return scales ? scale * scales[i] : scale; }
};

// Thin products are kept as two halves of 16 bits, [token][2][rp] with rp the rank up to a multiple of 8: a value cut to T, and
// what that lacks.  One T alone would cost as much as the result's own rounding.
//
// The upper half is always short of the value (of one that T holds, too: then by T's last place), so that both halves of a value
// other than zero are other than zero and have its sign.  Both are multiplied by the same factor, and infinity times them
// has to be the infinity that the value would give: a lower half of zero, or of the other sign, makes NaN of it.
template <class T>
__device__ __forceinline__ T shorter(float v)
{
    if constexpr (__is_same(T, __nv_bfloat16)) {
        const uint32_t u = __float_as_uint(v);
        return __ushort_as_bfloat16(static_cast<uint16_t>((u & 0x7FFFFFFF ? u - 1 : u) >> 16));
    } else {
        const T hi = __float2half_rz(v);
        const uint16_t bits = __half_as_ushort(hi);
        return widen(hi) == v && (bits & 0x7FFF) ? __ushort_as_half(static_cast<uint16_t>(bits - 1)) : hi;
    }
}
template <class T>
__device__ __forceinline__ void split_halves(float v, T &hi, T &lo)
{
    hi = isfinite(v) ? shorter<T>(v) : narrow<T>(v);
    lo = narrow<T>(isfinite(v) ? v - widen(hi) : v);
}

// Tokens in the order of their adapters, if they came scattered: what the projection's kernels then read in place of x.
struct SortedTokens {
    const uint32_t *scattered;                 // NULL: never; else 1 if they are
    const uint32_t *order, *keys;              // per place: the token, and its adapter (n: none)
    __device__ __forceinline__ bool on() const { return scattered && __ldcg(scattered); }
    __device__ __forceinline__ TokenIndex index(TokenIndex index, bool on) const
    {
        if (on) index.ids = keys, index.wide = false;
        return index;
    }
};

// A row per place, rows of `cols` elements that start on 16 bytes (what is behind a row's last is not written).  Bound by HBM:
// one B200, 8192 rows of 4096 (134 MB read and written) 19 us, behind a sort of 12.
constexpr uint32_t GATHER_WARPS = 8;
template <class T>
__global__ void __launch_bounds__(32 * GATHER_WARPS) k_gather(const SortedTokens sorted, const T *from, uint64_t stride, uint32_t cols, uint64_t tokens, T *to, uint64_t pitch)
{
    constexpr uint32_t AHEAD = 8;
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t t = static_cast<uint64_t>(blockIdx.x) * GATHER_WARPS + threadIdx.x / 32;
    let_next_start();
    wait_for_previous();
    if (t >= tokens || !sorted.on()) return;
    const T *in = from + sorted.order[t] * stride;
    T *out = to + t * pitch;
    for (uint32_t v = lane; v < cols / 8; v += 32 * AHEAD) {
        uint4 q[AHEAD];
#pragma unroll
        for (uint32_t e = 0; e < AHEAD; e++)
            if (v + e * 32 < cols / 8) q[e] = reinterpret_cast<const uint4 *>(in)[v + e * 32];
#pragma unroll
        for (uint32_t e = 0; e < AHEAD; e++)
            if (v + e * 32 < cols / 8) reinterpret_cast<uint4 *>(out)[v + e * 32] = q[e];
    }
    if (lane < cols % 8) out[cols / 8 * 8 + lane] = in[cols / 8 * 8 + lane];
}

// Copies whose rows start on a boundary of 16 bytes and end in zeros: out[o][r][c] = in(o, r, c) for c < cols, else 0.
template <class T>
struct PackJob {
    const T *in;
    T *out;
    uint64_t so, sr, sc, rows, cols, pitch, total;      // total: outer * rows
};
template <class T>
struct PackArgs {
    PackJob<T> job[5];
};
constexpr uint32_t PACK_WARPS = 8, PACK_COLS = 256;
// Where a row's elements are next to each other a thread has eight of them, whatever the row's length.  Else (a transposed tensor)
// a warp has 256 columns of a row, and neighbouring warps neighbouring rows: they read the same lines.  One B200, the factors, weight and
// tokens of 434 tokens 121 x 8064 and 20 adapters of rank 100 (36 MB): 27 us.
template <class T>
__global__ void __launch_bounds__(32 * PACK_WARPS) k_pack(const __grid_constant__ PackArgs<T> a)
{
    const PackJob<T> &j = a.job[blockIdx.y];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    wait_for_previous();
    if (j.sc == 1) {
        const uint64_t each = j.pitch / 8, all = j.total * each;
        for (uint64_t u = blockIdx.x * 32ull * PACK_WARPS + threadIdx.x; u < all; u += gridDim.x * 32ull * PACK_WARPS) {
            const uint64_t row = all >> 32 ? u / each : static_cast<uint32_t>(u) / static_cast<uint32_t>(each), o = j.rows == j.total ? 0 : row / j.rows;
            const uint64_t c = (u - row * each) * 8;
            const T *in = j.in + o * j.so + (row - o * j.rows) * j.sr + c;
            Vec<T, 16> v;
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) v.e[e] = c + e < j.cols ? in[e] : narrow<T>(0.0f);
            *reinterpret_cast<uint4 *>(j.out + u * 8) = v.raw;
        }
        return;
    }
    const uint64_t parts = (j.pitch + PACK_COLS - 1) / PACK_COLS, units = j.total * parts;
    for (uint64_t u = static_cast<uint64_t>(blockIdx.x) * PACK_WARPS + warp; u < units; u += static_cast<uint64_t>(gridDim.x) * PACK_WARPS) {
        const uint64_t part = u / j.total, row = u - part * j.total, o = row / j.rows;
        const T *in = j.in + o * j.so + (row - o * j.rows) * j.sr;
        T *out = j.out + row * j.pitch;
        T v[PACK_COLS / 32];
#pragma unroll
        for (uint32_t q = 0; q < PACK_COLS / 32; q++) {
            const uint64_t c = part * PACK_COLS + q * 32 + lane;
            v[q] = c < j.cols ? in[c * j.sc] : narrow<T>(0.0f);
        }
#pragma unroll
        for (uint32_t q = 0; q < PACK_COLS / 32; q++) {
            const uint64_t c = part * PACK_COLS + q * 32 + lane;
            if (c < j.pitch) out[c] = v[q];
        }
    }
}

}  // namespace lmz
