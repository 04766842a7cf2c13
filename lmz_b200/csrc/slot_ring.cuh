// Who makes which of a tile's mixed groups, and what the maker waits for: plain rules, for k_project and the check that runs
// without a GPU.
//
// Slots are a ring that groups use in their order; four warps (the epilogue's) take every group's sums out again, in that order.
// Of a tile's mixed groups the feeding warps make every other one, from its first, and the epilogue's warps the others before
// they take out any of that tile; a pair's feeding warps make all.
//
// A wait by parity can tell a slot's use only from its neighbours', so a maker may be neither two uses ahead of the slot's
// barrier nor two behind.  The feeding warps wait for the groups that they make, and for no others: the use that they are about
// to fill cannot be taken out before that, so the barrier is not ahead.  It is not behind either: their own group before (at most
// two groups back, and then there are two slots or more) waited until the groups up to one ring before it were out.  Had they
// waited for the epilogue's groups too, the epilogue could have made one and taken it out before they looked, and its barrier
// would have been two uses on: they would have waited for a phase that needs themselves.
#pragma once
#include <cstdint>

#include "geometry.cuh"

namespace lmz {

// `order`: the group's number among its tile's mixed ones.
LMZ_HD constexpr bool slot_by_feed(bool pair, uint32_t order) { return pair || order % 2 == 0; }
// Whether the feeding warps wait for the slot's use before; `turn`: the ring's.
LMZ_HD constexpr bool slot_feed_waits(bool pair, uint32_t order, uint32_t turn) { return turn != 0 && slot_by_feed(pair, order); }

}  // namespace lmz
