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
        else return 1;
    }
    return 0;
}
