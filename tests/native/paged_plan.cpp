// The arithmetic of llamd_rs_amd/csrc/paged_plan.hpp by name, for tests/test_paged_plan.py: a line of numbers in, a line out.
#include <cstdio>
#include <cstring>

#include "paged_plan.hpp"

int main() {
    char name[32];
    long long a[8];
    while (scanf("%31s", name) == 1) {
        const auto read = [&](int n) {
            for (int i = 0; i < n; ++i)
                if (scanf("%lld", &a[i]) != 1) return false;
            return true;
        };
        if (!strcmp(name, "shared") && read(3)) printf("%d\n", llamd::shared_positions((int)a[0], (int)a[1], (int)a[2]));
        else if (!strcmp(name, "join") && read(6)) {
            // a wave counts the tiles of `groups` groups, 64 at a time, every other one of `more` tiles, and looks for a row
            const int groups = (int)a[0], more = (int)a[1], tiles = (int)a[2], R = (int)a[3];
            int sum = 0;
            for (int lane = 0; lane < 64; ++lane) {
                int mine = 0;
                for (int i = lane; i < groups; i += 64) mine = llamd::add_tiles(mine, i % 2 ? 0 : more, tiles);
                sum += mine;
            }
            printf("%d %lld\n", sum, llamd::tile_of_row(a[5] ? a[5] : sum, a[4], R, tiles));
        } else if (!strcmp(name, "tiles") && read(7)) {
            const llamd::TilePlan x = llamd::plan_tiles(a[0], a[1], (int)a[2], (int)a[3], a[4], a[5], (int)a[6]);
            printf("%lld %d\n", x.tiles, x.parts);
        } else return 1;
    }
    return 0;
}
