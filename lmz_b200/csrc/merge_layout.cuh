// What k_merge's block keeps in shared memory: plain arithmetic, for the kernel, its launcher and the checks that run without a
// GPU.
#pragma once
#include <cstdint>

#include "geometry.cuh"

namespace lmz {

constexpr uint32_t M_ROWS = 128, M_COLS = 128, M_MAX_PLACES = 256;
constexpr uint32_t M_ROW_BYTES = 128;                  // 64 elements, swizzled as operands are
constexpr uint32_t M_BLOCK = M_ROWS * M_ROW_BYTES;     // 64 columns of the weight's tile
constexpr uint32_t M_SHARED = 16;                      // what the block's threads share (MergeShared)

// `places`: the rank up to a multiple of 16.  Stages of the weight's and A's tiles (as many as have room), a tile of B.
LMZ_HD constexpr uint32_t merge_stage(uint32_t places) { return M_COLS / 64 * (M_BLOCK + places * M_ROW_BYTES); }
LMZ_HD constexpr uint32_t merge_stages(uint32_t places) { return places <= 192 ? 2 : 1; }
LMZ_HD constexpr uint32_t merge_smem(uint32_t places)
{
    return merge_stages(places) * merge_stage(places) + (places + 63) / 64 * M_BLOCK + M_SHARED;
}
// The most that any rank takes: not the highest one, which has a stage less.
LMZ_HD constexpr uint32_t merge_smem_most()
{
    uint32_t most = 0;
    for (uint32_t places = 16; places <= M_MAX_PLACES; places += 16) most = merge_smem(places) > most ? merge_smem(places) : most;
    return most;
}
static_assert(merge_smem_most() <= F_SMEM_DYN, "a block has room for every rank");

}  // namespace lmz
