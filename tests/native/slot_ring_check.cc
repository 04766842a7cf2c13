// The slots between a projection's warps (csrc/slot_ring.cuh) under random schedules: barriers with the parity semantics of an
// mbarrier.  Exit status 0 = every schedule ended, and no slot was filled before it was empty or read before it was full.
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <random>
#include <vector>

#include "../../lmz_b200/csrc/slot_ring.cuh"

using namespace lmz;

namespace {

constexpr uint32_t WARPS = 4;                         // that take sums out

struct Bar {
    uint32_t count, pending, phase = 0;
    explicit Bar(uint32_t n) : count(n), pending(n) {}
    void arrive()
    {
        if (--pending == 0) phase++, pending = count;
    }
    bool over(uint32_t parity) const { return (phase & 1) != parity; }      // the phase of that parity has ended
};

struct Op {
    enum { WAIT_EMPTY, WAIT_FULL, FILL, FULL, TAKE, MEET } what;
    uint32_t slot, value;                             // a parity, or which use of all slots it is
};

struct Place {
    uint32_t stage = 0, turn = 0;
    void next(uint32_t n)
    {
        if (++stage == n) stage = 0, turn++;
    }
};

bool schedule(uint32_t seed)
{
    std::mt19937 rng(seed);
    auto any = [&](uint32_t n) { return static_cast<uint32_t>(rng() % n); };
    const bool pair = any(4) == 0;
    const uint32_t slots = pair ? 3 : 1 + any(8), tiles = 1 + any(12);
    std::vector<Op> agent[1 + WARPS];                 // the feeding warps, and the others
    Place feed, take[WARPS];
    uint32_t use = 0;
    for (uint32_t t = 0; t < tiles; t++) {
        const uint32_t most = pair ? 16 : slots, groups = any(3) ? any(most + 1) : most, first = use;
        for (uint32_t g = 0; g < groups; g++, use++) {
            if (slot_feed_waits(pair, g, feed.turn)) agent[0].push_back({Op::WAIT_EMPTY, feed.stage, (feed.turn - 1) & 1});
            if (slot_by_feed(pair, g)) {
                agent[0].push_back({Op::FILL, feed.stage, use});
                agent[0].push_back({Op::FULL, feed.stage, use});
            }
            feed.next(slots);
        }
        for (uint32_t w = 0; w < WARPS; w++) {
            Place at = take[w];
            for (uint32_t g = 0; !pair && g < groups; g++, at.next(slots)) {
                if (slot_by_feed(pair, g)) continue;
                agent[1 + w].push_back({Op::MEET, 0, 0});
                if (w == 0) agent[1].push_back({Op::FILL, at.stage, first + g});
                agent[1 + w].push_back({Op::MEET, 0, 0});
                if (w == 0) agent[1].push_back({Op::FULL, at.stage, first + g});
            }
            for (uint32_t g = 0; g < groups; g++, take[w].next(slots)) {
                agent[1 + w].push_back({Op::WAIT_FULL, take[w].stage, take[w].turn & 1});
                agent[1 + w].push_back({Op::TAKE, take[w].stage, first + g});
            }
        }
    }
    std::vector<Bar> full(slots, Bar(1)), empty(slots, Bar(WARPS));
    std::vector<int64_t> holds(slots, -1);
    std::vector<uint32_t> left(slots, 0);             // warps that have not taken what it holds
    size_t at[1 + WARPS] = {}, met[1 + WARPS] = {};   // met: how often the warp has come to a meeting
    bool waits[1 + WARPS] = {};
    uint32_t weight[1 + WARPS];
    for (uint32_t &w : weight) w = any(3) ? 1 + any(40) : 1;
    for (uint32_t idle = 0; idle < 4000;) {
        uint32_t sum = 0, i = 0;
        for (uint32_t w : weight) sum += w;
        for (uint32_t r = any(sum); r >= weight[i]; i++) r -= weight[i];
        if (any(500) == 0) weight[any(1 + WARPS)] = 1 + any(40);
        idle++;
        if (at[i] == agent[i].size()) {
            bool done = true;
            for (uint32_t a = 0; a <= WARPS; a++) done = done && at[a] == agent[a].size();
            if (done) return true;
            continue;
        }
        const Op op = agent[i][at[i]];
        if (op.what == Op::WAIT_EMPTY && !empty[op.slot].over(op.value)) continue;
        if (op.what == Op::WAIT_FULL && !full[op.slot].over(op.value)) continue;
        if (op.what == Op::MEET) {
            if (!waits[i]) waits[i] = true, met[i]++;
            if (*std::min_element(met + 1, met + 1 + WARPS) < met[i]) continue;
            waits[i] = false;
        }
        if (op.what == Op::FILL) {
            if (left[op.slot]) return fprintf(stderr, "seed %u: use %u fills a slot that still holds %lld\n", seed, op.value, (long long)holds[op.slot]), false;
            holds[op.slot] = op.value, left[op.slot] = WARPS;
        }
        if (op.what == Op::FULL) full[op.slot].arrive();
        if (op.what == Op::TAKE) {
            if (holds[op.slot] != op.value) return fprintf(stderr, "seed %u: use %u is taken where %lld is\n", seed, op.value, (long long)holds[op.slot]), false;
            left[op.slot]--;
            empty[op.slot].arrive();
        }
        at[i]++, idle = 0;
    }
    return fprintf(stderr, "seed %u: nobody goes on (%zu of %zu of the feeding warps' steps done)\n", seed, at[0], agent[0].size()), false;
}

}  // namespace

int main()
{
    for (uint32_t seed = 0; seed < 20000; seed++)
        if (!schedule(seed)) return 1;
    return 0;
}
