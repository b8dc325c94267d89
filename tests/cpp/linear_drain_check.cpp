// Tiles under way when linear attention's chunked form gives up: the chunks that are waited for are those whose copies may not have landed, each by a parity that tells
// its phase from the one before.
#include <cstdio>
#include <vector>

#include "kvb_linear_plan.hpp"

using namespace kvb;

int main() {
    int bad = 0;
    for (int chunks = 0; chunks <= 40; ++chunks)
        for (int issued = 0; issued <= chunks; ++issued) {  // where the load warp gave up, or all of them
            // chunk c is asked for when c - kLinearStages is done with, so all before issued - kLinearStages have landed; any of the others may have
            const int sure = issued - kLinearStages > 0 ? issued - kLinearStages : 0;
            for (int landed = sure; landed <= issued; ++landed) {
                std::vector<int> phase(kLinearStages, 0);  // completed phases of a stage's barrier
                for (int c = 0; c < landed; ++c) ++phase[c % kLinearStages];
                std::vector<bool> waited(issued, false);
                for (int c = linear_first_in_flight(issued); c < issued; ++c) {
                    waited[c] = true;
                    const int stage = c % kLinearStages, parity = (c / kLinearStages) & 1, done = phase[stage];
                    const bool passes = ((done - 1) & 1) == parity && done > 0;  // the barrier's last completed phase has this parity
                    if (passes != (c < landed)) ++bad;
                    if (!passes && done != c / kLinearStages) ++bad;  // it is the phase that is under way
                }
                for (int c = landed; c < issued; ++c) bad += !waited[c];
            }
        }
    std::printf(bad ? "linear drain: %d wrong\n" : "linear drain: ok\n", bad);
    return bad != 0;
}
