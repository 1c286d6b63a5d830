// The order in which the fp8 x fp8 kernels for few rows take the K tiles of a slice (plain C++: host and device).
#pragma once

namespace wq {

// A slice of `ntiles` K tiles, walked from tile `turn` on.  Trailing slices of a k_batch may be empty (ntiles <= 0): they have
// no tile to load and no scale to read, and store zeros.
struct F8F8Walk
{
    int ntiles, turn;
    constexpr F8F8Walk(int tiles, unsigned start) : ntiles(tiles), turn(tiles > 0 ? (int)(start % (unsigned)tiles) : 0) {}
    constexpr bool empty() const { return ntiles <= 0; }
    // tile of a step; inside the slice for steps below ntiles
    constexpr int tile(int step) const { return step + turn < ntiles ? step + turn : step + turn - ntiles; }
    // tile whose scales a fetch for `step` reads, of a slice that is not empty: steps behind the last one repeat its
    constexpr int scales(int step) const { return tile(step < ntiles ? step : ntiles - 1); }
};

} // namespace wq
