// Host check of the shared prefixes' part of csrc/paged_index.h: whatever groups, shared rows and lengths hold, a sequence's rows
// are its run's first ones and its own, whole; the parts of all runs cover their tiles' keys and fit what the workspace and the
// grid are sized for.
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
    std::mt19937 rng(5);
    auto any = [&](std::vector<int> v) { return v[rng() % v.size()]; };
    long long shared_runs = 0;
    for (int round = 0; round < 20000; ++round) {
        const int B = 1 + rng() % (rng() % 4 ? 70 : 300), group = any({1, 2, 3, 4, 7, 16, 40}), height = any({64, 128}), shift = 4 + rng() % 4;
        const int W = 1 + rng() % 60, shares = 1 + rng() % 300, kinds = 1 + rng() % 6;
        std::vector<int> id(B), want(B), length(B);
        for (int b = 0; b < B; ++b) {
            id[b] = b && rng() % 3 ? id[b - 1] : (int)(rng() % kinds) - 1;
            want[b] = rng() % 8 ? (int)(rng() % 2000) : any({INT_MIN, -1, 0, INT_MAX});
            length[b] = clamp_length(rng() % 8 ? (int)(rng() % 2500) : any({INT_MIN, -1, 0, INT_MAX}), W, shift);
        }
        struct Run { int size, rows; };
        std::vector<Run> runs;
        for (int b = 0; b < B;) {
            int e = b + 1;
            while (e < B && e % 64 && id[e] >= 0 && id[e] == id[b]) ++e;
            const int rows = e - b > 1 ? shared_rows(std::max(want[b], 0), length[b]) : 0;
            REQUIRE(rows >= 0 && rows % 16 == 0 && rows <= length[b]);
            for (int i = b; i < e; ++i) {
                const int from = shared_from(rows, std::max(want[i], 0), length[i]);
                REQUIRE(from >= 0 && from <= rows && from <= length[i]);
                REQUIRE(from % 16 == 0 || from == length[i]);
            }
            if (rows) runs.push_back({e - b, rows}), ++shared_runs;
            b = e;
        }
        long long total = 0, items = 0, rows = 0, most_items, most_rows;
        for (const Run& r : runs) total += (long long)((r.size * group + height - 1) / height) * ((r.rows + kPromptBlock - 1) / kPromptBlock);
        const int share = prefix_share_of(total, shares);
        REQUIRE(share >= kPrefixShare);
        for (const Run& r : runs) {
            const int blocks = (r.rows + kPromptBlock - 1) / kPromptBlock, parts = shares_of(blocks, share);
            REQUIRE(parts >= 1 && (parts - 1) * (long long)share < blocks && parts * (long long)share >= blocks);
            items += (long long)((r.size * group + height - 1) / height) * parts;
            rows += (long long)r.size * group * parts;
        }
        prefix_bounds(B, group, height, shares, most_items, most_rows);
        REQUIRE(items <= most_items && rows <= most_rows);
    }
    REQUIRE(shared_runs > 1000);
    REQUIRE(prefix_share_of(1ll << 50, 1) == 1 << 24);
    printf("ok\n");
    return 0;
}
