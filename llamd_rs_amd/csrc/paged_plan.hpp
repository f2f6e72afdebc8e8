// paged_plan.hpp -- arithmetic of the paged attention that both sides or a test on the CPU share: plain integers, no device.
#pragma once

namespace llamd {

// The positions that a group of sequences shares, whole pages, from what the device says: inside a table of max_page pages
// (2^30 positions at most), so that a position behind them can be stepped on without passing 32 bits.
constexpr int shared_positions(int shared, int page_log, int max_page) {
    const int top = max_page << page_log;
    return (shared < 0 ? 0 : shared < top ? shared : top) & ~((1 << page_log) - 1);
}

}  // namespace llamd
