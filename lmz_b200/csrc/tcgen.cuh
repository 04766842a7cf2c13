// Fifth-generation tensor cores, TMA and mbarriers of sm_100a, as the projection kernels use them.
//
// Operand tiles lie in shared memory in 128-byte rows whose 16-byte parts are swizzled by the row's number (what TMA's 128-byte
// swizzle writes): either a row per M or N index with 64 consecutive K elements (K-major), or a row per K index with 64
// consecutive M or N elements, further 64 of them in a block of their own (MN-major).  Tiles start on 1024 bytes.
#pragma once
#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>

namespace lmz {

constexpr uint32_t ROW_BYTES = 128, ATOM_BYTES = 1024, STEP_K = 64;

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// ---- mbarriers

__device__ __forceinline__ void bar_init(uint64_t *b, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t *b)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t *b, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t *b, uint32_t parity)
{
    uint32_t done;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done) : "r"(smem_addr(b)), "r"(parity) : "memory");
    return done;
}

// Set once a wait has run out (no wait does unless the hardware loses a copy): lmz_gpu_ops_gave_up() tells the host.
static __device__ uint32_t g_gave_up;

// Wait for a phase, but not for ever: after WAIT_NS the block's waits are all over, and with them its work; `over` is the
// block's flag.
constexpr uint64_t WAIT_NS = 4000000000ull;
__device__ __forceinline__ uint64_t nanoseconds()
{
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ bool bar_wait(uint64_t *b, uint32_t parity, volatile uint32_t *over)
{
    uint64_t since = 0;
    for (uint32_t i = 1; !bar_try(b, parity); i++) {
        if (i & 255) continue;
        if (*over) return false;
        const uint64_t now = nanoseconds();
        if (!since) since = now;
        if (now - since > WAIT_NS) {
            *over = 1;
            g_gave_up = 1;
            return false;
        }
    }
    return true;
}
// The same behind a wait that was over: for a copy or a product that must end before its memory goes.
__device__ __forceinline__ void bar_drain(uint64_t *b, uint32_t parity)
{
    const uint64_t since = nanoseconds();
    while (!bar_try(b, parity) && nanoseconds() - since < WAIT_NS) {}
}

// The address, in the cluster's window, of a word that another CTA has where this one has `p`.
__device__ __forceinline__ uint32_t peer_addr(const void *p, uint32_t rank)
{
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
    return at;
}
__device__ __forceinline__ void peer_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// (Relaxed: nothing of this thread's is handed over, and a release would wait a microsecond for nothing.)
__device__ __forceinline__ void peer_expect(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// One lane of the warp, always the same: what one thread issues stands in a loop that all lanes run, so that the compiler
// knows addresses and descriptors to be the warp's (a loop of lane 0's alone took twice as long to issue a step).
__device__ __forceinline__ bool elected()
{
    uint32_t p;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p;
}

// Where a role stands in a ring of stages, counted up without divisions (the threads that issue copies and products run alone:
// every instruction of their loops counts).
struct RingPlace {
    uint32_t stage = 0, turn = 0;              // turn: bit 0 is the parity of this use's phase
    __device__ __forceinline__ void next(uint32_t stages)
    {
        if (++stage == stages) stage = 0, turn++;
    }
    __device__ __forceinline__ void skip(uint32_t n, uint32_t stages)
    {
        stage += n;
        turn += stage / stages;
        stage %= stages;
    }
};

// ---- asynchronous copies

// Tiles; the barrier by its address.  PAIR: that of the pair's first CTA (in the cluster's window).
template <bool PAIR = false>
__device__ __forceinline__ void tma_load_2d(const CUtensorMap *map, uint32_t bar, uint32_t dst, int32_t x, int32_t y)
{
    if constexpr (PAIR)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
template <bool PAIR = false>
__device__ __forceinline__ void tma_load_3d(const CUtensorMap *map, uint32_t bar, uint32_t dst, int32_t x, int32_t y, int32_t z)
{
    if constexpr (PAIR)
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                     ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                     ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
// Four rows, by their numbers, of a map whose tiles are one row high (a row behind the tensor's last reads as zeros).
__device__ __forceinline__ void tma_gather4(const CUtensorMap *map, uint64_t *bar, uint32_t dst, int32_t x, const uint32_t *row)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
                 ::"r"(dst), "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(row[0]), "r"(row[1]), "r"(row[2]), "r"(row[3]) : "memory");
}
// 16 bytes from global to shared memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool on)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// What this thread has written to shared memory becomes visible to the tensor core.
__device__ __forceinline__ void publish_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Where 16-byte part c of row r of a tile lies.
__device__ __forceinline__ uint32_t swizzled(uint32_t r, uint32_t c) { return r * ROW_BYTES + ((c ^ (r & 7)) << 4); }

__device__ __forceinline__ void sync_threads(uint32_t barrier, uint32_t threads)
{
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
}

// Whether `ok` holds for all threads that come to a barrier.
__device__ __forceinline__ bool sync_all(uint32_t barrier, uint32_t threads, bool ok)
{
    uint32_t all;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %3, 0;\nbarrier.cta.red.and.pred q, %1, %2, p;\nselp.u32 %0, 1, 0, q;\n}\n"
                 : "=r"(all) : "r"(barrier), "r"(threads), "r"(static_cast<uint32_t>(ok)) : "memory");
    return all;
}

// ---- tensor cores

// PAIR: two CTAs of a cluster as one, each with half of the M rows of A, half of the N rows of B and its M rows of D.  Both
// allocate; the first one's thread issues.
template <bool PAIR = false>
__device__ __forceinline__ void tmem_alloc(uint32_t *at, uint32_t columns)
{
    if constexpr (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(at)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(at)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
}
template <bool PAIR = false>
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns)
{
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// A tile's descriptor.  K-major: eight rows of 128 bytes, 1024 bytes to the next eight.  MN-major: eight K indices, 1024 bytes to
// the next eight; `block` bytes to the next 64 M or N elements.  The upper word is the same for all tiles; 16 more bytes of address are one more in the lower word.
constexpr uint32_t DESC_HI = ATOM_BYTES >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t block) { return (addr & 0x3FFFF) >> 4 | (block >> 4) << 16; }
// 16-bit operands of one type, sums in 32 bits.
__device__ __forceinline__ uint32_t mma_desc(bool bf16, bool a_mn, bool b_mn, uint32_t m, uint32_t n)
{
    return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | (n >> 3) << 17 | (m >> 4) << 24;
}
// D (+)= A B^T over 16 K elements; the tiles by their descriptors' lower words.
template <bool PAIR = false>
__device__ __forceinline__ void mma16(uint32_t d, uint32_t a, uint32_t b, uint32_t desc, bool add)
{
    if constexpr (PAIR)
        asm volatile("{\n.reg .pred p;\n.reg .b64 x, y;\nsetp.ne.u32 p, %4, 0;\nmov.b64 x, {%1, %5};\nmov.b64 y, {%2, %5};\n"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], x, y, %3, p;\n}\n"
                     ::"r"(d), "r"(a), "r"(b), "r"(desc), "r"(static_cast<uint32_t>(add)), "r"(DESC_HI) : "memory");
    else
        asm volatile("{\n.reg .pred p;\n.reg .b64 x, y;\nsetp.ne.u32 p, %4, 0;\nmov.b64 x, {%1, %5};\nmov.b64 y, {%2, %5};\n"
                     "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n"
                     ::"r"(d), "r"(a), "r"(b), "r"(desc), "r"(static_cast<uint32_t>(add)), "r"(DESC_HI) : "memory");
}
// The barrier (of a pair: both CTAs') gets an arrival when all MMAs issued so far have ended.
template <bool PAIR = false>
__device__ __forceinline__ void mma_commit(uint64_t *bar)
{
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(smem_addr(bar)), "h"(static_cast<uint16_t>(3)) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// Sixteen columns of the warp's 32 lanes.
__device__ __forceinline__ void tmem_load16(uint32_t at, float *v)
{
    uint32_t r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(at));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}

// Eight of them.
__device__ __forceinline__ void tmem_load8(uint32_t at, float *v)
{
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(at));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = __uint_as_float(r[i]);
}

// The same for a warp whose lanes stay together.  (All of them ask: one lane alone, and the others told by a vote, took 350
// cycles where the phase was over already.)
__device__ __forceinline__ bool warp_wait(uint64_t *b, uint32_t parity, volatile uint32_t *over)
{
    bool ok = bar_try(b, parity);
    if (!ok) ok = bar_wait(b, parity, over);
    __syncwarp();
    return __all_sync(~0u, ok);
}

// ---- a kernel and the one launched behind it

// From here on the next kernel's blocks may start where there is room.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// The kernel before has ended and its results can be read.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- clusters

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_barrier()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Sums over a cluster's CTAs (at most eight), in their order, of words that each has at the same address; all loads are under
// way together.
struct Peers {
    uint32_t at[8], ctas;                      // where the others' words lie that this CTA has at `base`
    __device__ __forceinline__ Peers(uint32_t base, uint32_t n) : ctas(n)
    {
#pragma unroll
        for (uint32_t q = 0; q < 8; q++) asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at[q]) : "r"(base), "r"(q < n ? q : 0));
    }
    __device__ __forceinline__ float sum(uint32_t offset) const
    {
        float v[8];
#pragma unroll
        for (uint32_t q = 0; q < 8; q++) {
            v[q] = 0;
            if (q < ctas) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[q]) : "r"(at[q] + offset) : "memory");
        }
        float all = v[0];
#pragma unroll
        for (uint32_t q = 1; q < 8; q++) all += v[q];
        return all;
    }
    // Eight of them, `step` bytes apart.
    __device__ __forceinline__ void sum8(uint32_t offset, uint32_t step, float *to) const
    {
#pragma unroll
        for (uint32_t e = 0; e < 8; e++) to[e] = 0;
#pragma unroll
        for (uint32_t q = 0; q < 8; q++) {
            if (q >= ctas) break;
            float v[8];
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[e]) : "r"(at[q] + offset + e * step) : "memory");
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) to[e] += v[e];
        }
    }
};

}  // namespace lmz
