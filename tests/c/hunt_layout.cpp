// For launches over splits of `runs` runs and a last split of any fewer steps: whether the words that its workgroup
// addresses in shared memory are within the launch's bytes.  Prints the number that are not and that of all.
#include <algorithm>
#include <cstdio>

#include "gefenx_hunt.h"

using namespace gx;

int main() {
    long bad = 0, checked = 0;
    constexpr int kLanes = 256, kOfStep = kStep * kLanes;
    for (int64_t steps = 1; steps <= 3000; ++steps) {
        for (const int64_t runs : {steps * kOfStep, (steps - 1) * kOfStep + 1}) {
            const HuntPlan plan = plan_hunt(runs, kLanes);
            const int64_t words = (int64_t)(plan.bytes / sizeof(uint64_t));
            if (slots_of(runs, kLanes, plan.steps_of_slot) > kSlots) ++bad;
            for (int64_t own = 0; own <= steps; own += steps > 100 ? 7 : 1) {
                const int slots = slots_of(std::min(own * kOfStep, runs), kLanes, plan.steps_of_slot);
                const int64_t at = maxima_words(kLanes, slots);  // of the candidates
                // the candidates, which their ranks read in pairs; before them a word of 4 bytes of each lane
                const int64_t end = at + std::max((plan.room + 2) / 2 * 2, kLanes / 2);
                const int64_t bins = 256 / 2 + 8, likeliest = 128 + 2;
                if (std::max(end, std::max(bins, likeliest)) > words) {
                    if (bad++ < 5)
                        std::fprintf(stderr, "runs %ld, last split of %ld steps: %ld of %ld words\n", (long)runs, (long)own, (long)end,
                                     (long)words);
                }
                ++checked;
            }
        }
    }
    std::printf("%ld %ld\n", bad, checked);
    return 0;
}
