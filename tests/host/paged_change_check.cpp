// Host check of csrc/paged_index.h for starts and lengths that change while the kernels run: an item's number that was
// counted from one batch and is looked up in another either stands for a part of a tile there, whose rows and blocks exist,
// or is told apart; and partial results outside the workspace are told apart.
#include <limits.h>
#include <stdio.h>
#include <stdlib.h>

#include <random>

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
    std::mt19937 rng(11);
    const int groups[] = {1, 2, 3, 4, 7, 16, 40}, heights[] = {64, 128};
    long long real = 0, told = 0;
    for (int round = 0; round < 20000; ++round) {
        const int group = groups[rng() % 7], height = heights[rng() % 2];
        auto tiles = [&]() {
            return PromptTiles{rng() % 4 ? (int)(rng() % 700) : 0, group, rng() % 3 ? (int)(rng() % 3000) : (int)(rng() % 40) - 700, height};
        };
        const PromptTiles counted = tiles(), t = tiles();
        const int share = prompt_share(counted.blocks_bound() / (1 + rng() % 4), 1 + rng() % 64), n = counted.items(share);
        if (!n) continue;
        const int index = (int)(rng() % n);
        const PromptItem it = prompt_item(t, share, index);
        REQUIRE(it.slot >= 0 && it.part >= 0);
        if (!is_item(t, share, it)) {
            REQUIRE(index >= t.items(share));
            ++told;
            continue;
        }
        REQUIRE(index < t.items(share));
        REQUIRE(it.tile < t.tiles() && it.tile * height < t.rows());
        REQUIRE(it.part == 0 || it.part * share < t.blocks(it.tile));
        ++real;
    }
    REQUIRE(real > 1000 && told > 1000);
    REQUIRE(in_slots(0, 0, 0) && in_slots(0, 1, 1) && in_slots(3, 4, 7));
    REQUIRE(!in_slots(3, 5, 7) && !in_slots(-1, 1, 7) && !in_slots(7, 1, 7) && !in_slots(1, -1, 7) && !in_slots(0, 1, 0));
    REQUIRE(!in_slots(INT_MAX, INT_MAX, 1ll << 31) && !in_slots(INT_MIN, 1, 7));
    printf("ok\n");
    return 0;
}
