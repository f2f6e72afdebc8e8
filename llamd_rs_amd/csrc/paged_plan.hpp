// paged_plan.hpp -- arithmetic of the paged attention that both sides or a test on the CPU share: plain integers, no device.
#pragma once

namespace llamd {

// The positions that a group of sequences shares, whole pages, from what the device says: inside a table of max_page pages
// (2^30 positions at most), so that a position behind them can be stepped on without passing 32 bits.
constexpr int shared_positions(int shared, int page_log, int max_page) {
    const int top = max_page << page_log;
    return (shared < 0 ? 0 : shared < top ? shared : top) & ~((1 << page_log) - 1);
}

// Tiles of shared prefixes counted so far, and `more` of the next group: no more than there are slots for (starts of groups
// that descend claim more, up to 2^22 per group; the sum over the lanes of a wave stays inside 32 bits this way).
constexpr int add_tiles(int so_far, int more, int tiles) { return more < tiles - so_far ? so_far + more : tiles; }

// The tile that row number `row` of a group lies in, tiles of R rows, `before` of them in front of the group; inside the slots.
constexpr long long tile_of_row(long long before, long long row, int R, int tiles) {
    const long long tile = before + row / R;
    return tile < tiles ? tile : tiles - 1;
}

}  // namespace llamd
