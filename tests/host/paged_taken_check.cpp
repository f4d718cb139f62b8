// Host check of what a run's prefix is read for (csrc/paged_index.h): with the rows that the sequences behind the first one take
// in place of all that it shares, every one of those takes the same rows as before, and the first one takes all that is read.
#include <limits.h>
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <random>
#include <vector>

#include "paged_index.h"

using namespace moss;

#define REQUIRE(c)                                              \
    do {                                                        \
        if (!(c)) {                                             \
            printf("line %d: %s\n", __LINE__, #c);              \
            exit(1);                                            \
        }                                                       \
    } while (0)

int main() {
    std::mt19937 rng(7);
    long long less = 0, none = 0;
    for (int round = 0; round < 200000; ++round) {
        const int n = 2 + rng() % 8, top = 1 << (rng() % 31);
        std::vector<int> want(n), length(n);
        for (int i = 0; i < n; ++i) {
            want[i] = rng() % 6 ? (int)(rng() % top) : rng() % 2 ? INT_MAX : 0;
            length[i] = clamp_length(rng() % 6 ? (int)(rng() % top) : rng() % 2 ? INT_MAX : 0, 1 << 26, 4);
        }
        const int rows = shared_rows(want[0], length[0]);
        int most = 0;
        for (int i = 1; i < n; ++i) most = std::max(most, shared_from(rows, want[i], length[i]));
        const int read = taken_rows(most);
        REQUIRE(read % 16 == 0 && read >= 0 && read <= rows);
        for (int i = 1; i < n; ++i) {
            const int from = shared_from(rows, want[i], length[i]);
            REQUIRE(shared_from(read, want[i], length[i]) == from && from <= read);
        }
        REQUIRE(shared_from(read, want[0], length[0]) == read);
        less += read < rows, none += read == 0 && rows > 0;
    }
    REQUIRE(less > 10000 && none > 100);
    printf("ok\n");
    return 0;
}
