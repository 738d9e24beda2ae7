// gefenx_hunt.h -- shared memory of the search for a row's likeliest tokens: maxima of a lane's steps, then
// candidates, in words of 8 bytes.
#pragma once

#include <cstddef>
#include <cstdint>

namespace gx {

constexpr int kStep = 4;    // runs of a lane in flight
constexpr int kSlots = 20;  // maxima of a lane's steps that are kept, at most

constexpr int maxima_words(int lanes, int slots) { return lanes / 2 * slots; }

// Candidates that there is room for, beside so many maxima of a lane: short rows may have all of their logits among them.
// A launch has one room for all of its splits, by the slots of a whole one: the last split of a row may have fewer.
constexpr int candidates_room(int lanes, int slots) { return lanes < 256 ? 256 : slots > 4 ? 384 : 1024; }
constexpr int hunt_words(int lanes, int slots) { return maxima_words(lanes, slots) + candidates_room(lanes, slots) + 2; }

// Of a workgroup of `lanes` over splits of up to `runs` runs: steps that share a maximum, room, bytes.
struct HuntPlan {
    int steps_of_slot, room;
    size_t bytes;
};
constexpr int slots_of(int64_t runs, int lanes, int steps_of_slot) {
    return (int)(((runs + kStep * lanes - 1) / (kStep * lanes) + steps_of_slot - 1) / steps_of_slot);
}
constexpr HuntPlan plan_hunt(int64_t runs, int lanes) {
    const int steps = slots_of(runs, lanes, 1), per = (steps + kSlots - 1) / kSlots, slots = slots_of(runs, lanes, per);
    return {per, candidates_room(lanes, slots), sizeof(uint64_t) * (size_t)hunt_words(lanes, slots)};
}

}  // namespace gx
