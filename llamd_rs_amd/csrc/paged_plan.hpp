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

// How many there are of something: `want`, but no more than `most` nor `cap`, and one at least.
constexpr int at_least_one(long long want, long long most, long long cap) {
    const long long n = want < most ? want : most, x = n < cap ? n : cap;
    return x < 1 ? 1 : (int)x;
}

// The tiles of R rows that there can be where `rows` rows lie in up to `pieces` pieces (sequences, groups) that each begin a
// tile of their own, and the parts of a tile's positions that make about `want` workgroups, `most` and `cap` at the most. How
// many pieces have rows is known on the device only: parts are for tiles that the rows fill, or for a tile per four pieces
// if that is more, so that tiles times parts stays within a few times `want` whatever the pieces. 64 sequences of 32 heads
// in 32 pairs: 2 parts, 166 us and 130 MB of slots, where parts for full tiles are 16, 192 us and 1 GB, and a tile per piece
// gives one part, 164 us; but one group in a list of 32 places (64 sequences behind 15000 positions, 32 / 4 heads) takes 53
// us this way, 98 with a tile per piece. A prompt batch of one token in 64 sequences' places (200 positions, tables of 16384):
// 12.7 us, 36 with slots for 64 tiles of 128 parts; 8 tokens of one sequence in 256 places, 32 heads: 27 us, a part per tile
// of each place 54, slots for them all 368 us and 1.5 GB; 64 single tokens of 12 heads 35.5, 27.8, 39.2.
struct TilePlan {
    long long tiles;
    int parts;
};
constexpr TilePlan plan_tiles(long long rows, long long pieces, int R, int n_kv_head, long long want, long long most, int cap) {
    const long long full = (rows + R - 1) / R, some = (pieces + 3) / 4, least = full > some ? full : some;
    return {rows / R + pieces, at_least_one(want / (least * n_kv_head), most, cap)};
}

}  // namespace llamd
