// Host check of the shared prefixes' part of csrc/paged_index.h: whatever groups, shared rows and lengths hold, a sequence's rows
// are its run's first ones and its own, whole; the pieces of the lines of work cover them, each part's results have a
// place of their own within the workspace, and the places are those where the join looks for them.
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
    for (int round = 0; round < 4000; ++round) {
        const int B = 1 + rng() % (rng() % 4 ? 70 : 200), group = any({1, 2, 3, 4, 7, 16, 40}), height = any({64, 128}), shift = 4 + rng() % 4;
        const int W = 1 + rng() % 60, shares = 1 + rng() % 300, kinds = 1 + rng() % 6;
        std::vector<int> id(B), want(B), length(B);
        for (int b = 0; b < B; ++b) {
            id[b] = b && rng() % 3 ? id[b - 1] : (int)(rng() % kinds) - 1;
            want[b] = rng() % 8 ? (int)(rng() % 2000) : any({INT_MIN, -1, 0, INT_MAX});
            length[b] = clamp_length(rng() % 8 ? (int)(rng() % 2500) : any({INT_MIN, -1, 0, INT_MAX}), W, shift);
        }
        const int G = group, workgroups = 1 + shares, head_tiles = (G + 15) / 16;
        struct Tile { long long start; int blocks, rows_before, rows; };
        struct Own { long long start; int units, b, tile; };
        std::vector<Tile> tiles;
        std::vector<Own> owns;
        std::vector<int> from(B);
        long long blocks_all = 0, units_all = 0;
        int rows_before = 0;
        for (int b = 0; b < B;) {
            int e = b + 1;
            while (e < B && e % 64 && id[e] >= 0 && id[e] == id[b]) ++e;
            const int rows = e - b > 1 ? shared_rows(std::max(want[b], 0), length[b]) : 0;
            REQUIRE(rows >= 0 && rows % 16 == 0 && rows <= length[b]);
            for (int i = b; i < e; ++i) {
                from[i] = shared_from(rows, std::max(want[i], 0), length[i]);
                REQUIRE(from[i] >= 0 && from[i] <= rows && from[i] <= length[i]);
                REQUIRE(from[i] % 16 == 0 || from[i] == length[i]);
            }
            if (rows) {
                const int all = (e - b) * G, blocks = (rows + kPromptBlock - 1) / kPromptBlock;
                for (int r = 0; r < all; r += height) {
                    tiles.push_back({blocks_all, blocks, rows_before + r, std::min(height, all - r)});
                    blocks_all += blocks;
                }
                rows_before += all;
                ++shared_runs;
            }
            b = e;
        }
        for (int b = 0; b < B; ++b)
            for (int t = 0; t < head_tiles; ++t) {
                owns.push_back({units_all, own_units(length[b] - from[b]), b, t});
                units_all += owns.back().units;
            }
        const int takers = prefix_takers((float)blocks_all, (float)units_all, workgroups);
        REQUIRE(takers >= (blocks_all > 0) && workgroups - takers >= (units_all > 0));
        const int blocks_each = piece_of(blocks_all, std::max(takers, 1)), units_each = piece_of(units_all, 4 * std::max(workgroups - takers, 1));
        REQUIRE(blocks_each >= 1 && (long long)blocks_each * std::max(takers, 1) >= blocks_all);
        REQUIRE(units_each >= 1 && (long long)units_each * 4 * std::max(workgroups - takers, 1) >= units_all);
        std::vector<char> row_taken((long long)B * G + (long long)workgroups * height), slot_taken((size_t)(4 * workgroups + B) * head_tiles);
        for (const Tile& t : tiles) {
            const long long w0 = quotient(t.start, blocks_each), w1 = quotient(t.start + t.blocks - 1, blocks_each);
            REQUIRE(w1 < takers);
            for (long long w = w0; w <= w1; ++w)
                for (int r = 0; r < t.rows; ++r) {
                    const long long place = t.rows_before + r + w * height;
                    REQUIRE(place < (long long)row_taken.size() && !row_taken[place]);
                    row_taken[place] = 1;
                }
        }
        for (const Own& o : owns) {
            if (!o.units) continue;
            const long long w0 = quotient(o.start, units_each), w1 = quotient(o.start + o.units - 1, units_each);
            REQUIRE(w1 < 4 * (workgroups - takers));
            for (long long w = w0; w <= w1; ++w) {
                const long long place = (w + o.b) * head_tiles + o.tile;
                REQUIRE(place < (long long)slot_taken.size() && !slot_taken[place]);
                slot_taken[place] = 1;
            }
        }
    }
    REQUIRE(shared_runs > 1000);
    REQUIRE(piece_of(0, 7) == 1 && piece_of(28, 7) == 4 && piece_of(29, 7) == 5 && piece_of(1ll << 60, 1) == 1 << 30);
    REQUIRE(piece_of((1ll << 31) - 1, 512) == 1 << 22 && piece_of(1ll << 40, 512) == 1 << 30);
    REQUIRE(quotient((1ll << 32) - 1, 3) == ((1ll << 32) - 1) / 3 && quotient(1ll << 40, 3) == (1ll << 40) / 3);
    printf("ok\n");
    return 0;
}
