// Runs of work of the attention over a cache in pages (paged.hip): the steps of
// all units, one behind the other, in equal runs, and the runs that hold a unit.
#pragma once
#include <cstdint>

namespace qh {

constexpr uint32_t kRunMin = 2;    // steps of a run at least
constexpr uint32_t kUnitCost = 2;  // steps in front of a unit's own that are not work

__host__ __device__ inline uint64_t div64(uint64_t a, uint64_t b) {
    return (a | b) >> 32 ? a / b : (uint32_t)a / (uint32_t)b;
}
// Run i of `total` steps in all holds the steps [total i / runs, total (i + 1) /
// runs); fewer than `most` runs where they would be too short.
__host__ __device__ inline uint64_t runs_of(uint64_t total, uint32_t most) {
    const uint64_t n = (total + kRunMin - 1) / kRunMin;
    return n < most ? n : most;
}
__host__ __device__ inline uint64_t run_begin(uint64_t total, uint64_t runs, uint64_t i) { return div64(total * i, runs); }
__host__ __device__ inline uint64_t run_with(uint64_t total, uint64_t runs, uint64_t x) {  // the run of step x
    return div64((x + 1) * runs + total - 1, total) - 1;
}

// The runs that hold a unit's own steps: unit u of a sequence whose `units` units
// lie at the steps [begin, end) of `total`.  Whatever begin and end are, they are
// runs of runs_of(total, most).
struct Parts {
    uint64_t first;
    uint32_t count;
};
__host__ __device__ inline Parts parts_of(uint64_t total, uint32_t most, uint64_t begin, uint64_t end, uint32_t units,
                                          uint32_t u) {
    end = end < total ? end : total;
    begin = begin < end ? begin : end;
    const uint64_t runs = runs_of(total, most), steps = div64(end - begin, units), x = begin + u * steps;
    if (steps <= kUnitCost) return {0, 0};
    const uint64_t first = run_with(total, runs, x + kUnitCost), last = run_with(total, runs, x + steps - 1);
    return {first, (uint32_t)(last - first) + 1};
}

}  // namespace qh
