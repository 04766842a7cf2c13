// Checks of csrc/merge_layout.cuh.  Exit status 0 = they held.
#include <cstdint>
#include <cstdio>

#include "../../lmz_b200/csrc/merge_layout.cuh"

using namespace lmz;

int main()
{
    bool found = false;
    for (uint32_t rank = 1; rank <= M_MAX_PLACES; rank++) {
        const uint32_t places = (rank + 15) & ~15u, bytes = merge_smem(places);
        if (bytes > merge_smem_most() || bytes > F_SMEM_DYN) return fprintf(stderr, "rank %u takes %u bytes\n", rank, bytes), 1;
        // its parts: stages, B's tile, the shared words on a boundary of their own
        if (bytes != merge_stages(places) * (2 * 16384 + 2 * places * 128) + (places + 63) / 64 * 16384 + 16 || (bytes - M_SHARED) % 1024)
            return fprintf(stderr, "rank %u: parts\n", rank), 1;
        found = found || bytes == merge_smem_most();
    }
    return found && merge_smem_most() > merge_smem(M_MAX_PLACES) ? 0 : 1;
}
