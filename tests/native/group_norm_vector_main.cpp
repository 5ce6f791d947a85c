// The number of groups that a vector of channels may touch, and with it the passes over the lanes' sums, against counting
// them: every vector of a row, whose groups and vectors start together.
#include <cstdio>

#include "../../l2_torch_alloc_amd/csrc/group_norm.h"

using namespace sideaware;

int main() {
    int cases = 0;
    for (int vec = 1; vec <= 8; vec *= 2) {
        for (int gc = 1; gc <= 80; gc++, cases++) {
            int most = 0;
            for (int v = 0; v < gc; v++) {                        // vec rows of a vector: all ways to start
                const int touched = (v * vec + vec - 1) / gc - v * vec / gc + 1;
                if (touched > most) most = touched;
            }
            if (gn_groups_of_vector(vec, gc) != most || 2 * gn_sum_passes(vec, gc) < most || 2 * (gn_sum_passes(vec, gc) - 1) >= most) {
                std::printf("FAIL vec=%d gc=%d: %d groups, %d passes, %d counted\n", vec, gc, gn_groups_of_vector(vec, gc), gn_sum_passes(vec, gc), most);
                return 1;
            }
        }
    }
    std::printf("cases=%d ok\n", cases);
    return 0;
}
