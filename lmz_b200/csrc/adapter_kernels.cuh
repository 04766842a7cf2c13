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

// Thin products go into the second product as two halves, [token][2][rp] with rp the rank up to a multiple of 8: a value cut to
// 16 bits, and what that lacks.  One 16-bit number alone would cost as much as the result's own rounding.
//
// The halves are BF16 for F16 tensors, too: F16 would lose values above 65504, and bits of those below 2^-14, that the result
// still needs.  (A factor in F16 then comes as two BF16 parts: k_parts.)
//
// The upper half is always short of the value (of one that 16 bits hold, too: then by its last place), so that both halves of a
// value other than zero are other than zero and have its sign.  Both are multiplied by the same factor, and infinity
// times them has to be the infinity that the value would give: a lower half of zero, or of the other sign, makes NaN of it.
using Thin = __nv_bfloat16;
__device__ __forceinline__ void split_halves(float v, Thin &hi, Thin &lo)
{
    const uint32_t u = __float_as_uint(v);
    hi = isfinite(v) ? __ushort_as_bfloat16(static_cast<uint16_t>((u & 0x7FFFFFFF ? u - 1 : u) >> 16)) : narrow<Thin>(v);
    lo = narrow<Thin>(isfinite(v) ? v - widen(hi) : v);
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

// F16's factors as BF16, for the product with thin halves: each value as two parts (split_halves, exact: 11 bits of 16), so that a
// sum over both parts is the sum over the factor.  out[slot][part][each], for the adapters that have a sixteen of tokens to
// themselves; only those are asked for.
//
// A block's row of the grid is a slot: an adapter's own where there are no more adapters than sixteens, else a sixteen's, for the
// adapter whose first sixteen it is (one token beside a thousand adapters of 4096 x 16: 14 us of the call were blocks with nothing
// to do).  Runs beside the thin product, which has waited for all that is read here.  Bound by latency and HBM: 2 bytes read and 4
// written a value.  One B200, 8 factors of 4096 x 32: 10 us alone, and 1 to 3 of a call's.
struct PartsArgs {
    const __half *in;                          // of adapter i from i * each
    Thin *out;
    uint32_t *slot;                            // per adapter, written
    TokenIndex index;
    SortedTokens sorted;
    uint64_t each, tokens, sixteens;
};
constexpr uint32_t PARTS_THREADS = 256, PARTS_VALUES = PARTS_THREADS * 8 * 4;        // of a block
static __global__ void __launch_bounds__(PARTS_THREADS) k_parts(const PartsArgs a)
{
    __shared__ uint32_t s_first;
    const uint32_t tid = threadIdx.x, slot = blockIdx.y;
    let_next_start();
    int i = slot;
    bool own = true;
    if (a.index.ids) {                                           // the adapter's first sixteen, if it has one
        const TokenIndex index = a.sorted.index(a.index, a.sorted.on());
        const bool by_sixteen = a.index.n > a.sixteens;
        const uint64_t end = by_sixteen ? slot + 1ull : a.sixteens;
        if (by_sixteen) i = index.of(slot * 16ull);
        if (tid == 0) s_first = ~0u;
        __syncthreads();
        uint32_t first = ~0u;
        for (uint64_t g0 = 0; i >= 0 && g0 < end && first == ~0u; g0 += PARTS_THREADS) {
            const uint64_t g = g0 + tid, t0 = g * 16;
            if (g < end && index.of(t0) == i) {
                bool all = true;
                for (uint32_t c = 1; c < 16; c++)
                    if (t0 + c < a.tokens) all = all && index.of(t0 + c) == i;
                if (all) atomicMin(&s_first, static_cast<uint32_t>(g));
            }
            __syncthreads();
            first = s_first;
            __syncthreads();
        }
        own = by_sixteen ? first == slot : first != ~0u;
    }
    if (own) {
        if (blockIdx.x == 0 && tid == 0) a.slot[i] = slot;
        const __half *in = a.in + i * a.each;
        Thin *out = a.out + slot * 2ull * a.each;
        const uint64_t lo = static_cast<uint64_t>(blockIdx.x) * PARTS_VALUES + tid * 8;
        Vec<__half, 16> v[4];
#pragma unroll
        for (uint32_t q = 0; q < 4; q++)
            if (lo + q * PARTS_THREADS * 8 < a.each) v[q].raw = *reinterpret_cast<const uint4 *>(in + lo + q * PARTS_THREADS * 8);
#pragma unroll
        for (uint32_t q = 0; q < 4; q++) {
            const uint64_t at = lo + q * PARTS_THREADS * 8;
            if (at >= a.each) continue;
            Vec<Thin, 16> hi, rest;
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) split_halves(widen(v[q].e[e]), hi.e[e], rest.e[e]);
            *reinterpret_cast<uint4 *>(out + at) = hi.raw;
            *reinterpret_cast<uint4 *>(out + a.each + at) = rest.raw;
        }
    }
    if (blockIdx.x == 0 && slot == 0) wait_for_previous();       // (this one ends no sooner than the thin product)
}

// F16's thin products for the factors' gradients, where they are multiplied by F16 tensors: [token][rp] in 32 bits, as two halves
// in F16 times a power of two.  Each adapter has a power of its own, by which its largest value comes to 2^14 and more; the
// lower half is 2^11 times what the upper one lacks.  So a value keeps 16 bits and more down to 2^-34 of the largest one, and
// both powers go out of the sums again exactly.  (The upper half is zero only where the value is: see above.)
//
// A cluster has an adapter's tokens: their largest value, then their halves.  Bound by latency: the products were just made.  One B200, both
// products of 4096 tokens at rank 32: 11 us.
struct ThinJob {
    const float *from;
    __half *to;                                // [token][2][rp]
    float *scale;                              // per adapter: what its sums are to be multiplied by
};
struct ThinArgs {
    ThinJob job[2];
    const uint32_t *order, *start;             // as for the factors' gradients
    uint32_t tokens, rp;
};
constexpr uint32_t THIN_CTAS = 8, THIN_THREADS = 512;
constexpr float THIN_LOWER = 1.0f / 2048;      // of a lower half
static __global__ void __launch_bounds__(THIN_THREADS) k_thin(const __grid_constant__ ThinArgs a)
{
    __shared__ uint32_t s_most;
    const ThinJob &job = a.job[blockIdx.z];
    const uint32_t tid = threadIdx.x, i = blockIdx.y, rank = cluster_rank(), parts = a.rp / 8;
    wait_for_previous();
    const uint32_t begin = a.start ? a.start[i] : 0, end = a.start ? a.start[i + 1] : i ? 0 : a.tokens;
    const uint64_t units = static_cast<uint64_t>(end - begin) * parts;
    auto at = [&](uint64_t u, uint64_t &row, uint32_t &c) {
        const uint32_t n = static_cast<uint32_t>(u / parts);
        row = a.order ? a.order[begin + n] : n, c = static_cast<uint32_t>(u - static_cast<uint64_t>(n) * parts) * 8;
    };
    auto load = [&](uint64_t row, uint32_t c, float *v) {
        const float4 *p = reinterpret_cast<const float4 *>(job.from + row * a.rp + c);
        *reinterpret_cast<float4 *>(v) = p[0], *reinterpret_cast<float4 *>(v + 4) = p[1];
    };
    uint32_t most = 0;
    for (uint64_t u = rank * THIN_THREADS + tid; u < units; u += THIN_CTAS * THIN_THREADS) {
        uint64_t row;
        uint32_t c;
        float v[8];
        at(u, row, c);
        load(row, c, v);
#pragma unroll
        for (uint32_t e = 0; e < 8; e++)
            if (isfinite(v[e])) most = max(most, __float_as_uint(v[e]) & 0x7FFFFFFF);
    }
    if (tid == 0) s_most = 0;
    __syncthreads();
    most = __reduce_max_sync(~0u, most);
    if ((tid & 31) == 0) atomicMax(&s_most, most);
    __syncwarp();
    cluster_barrier();
    for (uint32_t q = 0; q < THIN_CTAS; q++) {
        uint32_t other;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(other) : "r"(peer_addr(&s_most, q)) : "memory");
        most = max(most, other);
    }
    const int e2 = most ? max(-100, min(113, static_cast<int>(most >> 23) - 127 - 14)) : 0;
    const float down = __uint_as_float(static_cast<uint32_t>(127 - e2) << 23);
    if (rank == 0 && tid == 0) job.scale[i] = __uint_as_float(static_cast<uint32_t>(127 + e2) << 23);
    for (uint64_t u = rank * THIN_THREADS + tid; u < units; u += THIN_CTAS * THIN_THREADS) {
        uint64_t row;
        uint32_t c;
        float v[8];
        at(u, row, c);
        load(row, c, v);
        Vec<__half, 16> upper, lower;
#pragma unroll
        for (uint32_t e = 0; e < 8; e++) {
            const float w = v[e] * down;
            __half hi = narrow<__half>(w);
            if (v[e] != 0 && __heq(hi, __ushort_as_half(0))) hi = __ushort_as_half(w < 0 || (w == 0 && v[e] < 0) ? 0x8001 : 1);
            upper.e[e] = hi;
            lower.e[e] = narrow<__half>(isfinite(v[e]) ? (w - widen(hi)) * (1 / THIN_LOWER) : 0.0f);
        }
        __half *to = job.to + row * 2 * a.rp + c;
        *reinterpret_cast<uint4 *>(to) = upper.raw;
        *reinterpret_cast<uint4 *>(to + a.rp) = lower.raw;
    }
    __syncwarp();
    cluster_barrier();                                           // nobody leaves while another reads its largest
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
