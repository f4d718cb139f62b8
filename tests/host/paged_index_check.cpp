// Host check of csrc/paged_index.h: whatever a table, lengths and starts hold, offsets stay inside the cache, and the
// decode shares cover every row once and fit the slots that the workspace is sized for.
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
    auto any = [&](std::vector<int> v) { return v[rng() % v.size()]; };
    const std::vector<int> odd = {INT_MIN, INT_MIN + 1, -65536, -2, -1, 0, 1, 2, 3, 16, 100, 1 << 20, 1 << 30, INT_MAX - 1, INT_MAX};
    // pages and rows
    for (int round = 0; round < 20000; ++round) {
        const int shift = 4 + rng() % 9, pages = 1 + rng() % 5, kh = 1 + rng() % 4, D = rng() % 2 ? 64 : 128, W = 1 + rng() % 6;
        const long long page = ((long long)kh << shift) * D, stride = page + 8 * (rng() % 3);
        const size_t elements = (size_t)(pages - 1) * stride + page;
        std::vector<int> table(W);
        for (int& t : table) t = rng() % 2 ? any(odd) : (int)(rng() % pages);
        const int length = clamp_length(rng() % 2 ? any(odd) : (int)(rng() % ((W << shift) + 9)), W, shift);
        REQUIRE(length >= 0 && length <= W << shift);
        const int row = rng() % 2 ? any(odd) : (int)(rng() % ((W + 1) << shift));
        const int p = page_of_row(table.data(), row, W, shift, pages);
        REQUIRE(p >= -1 && p < pages);
        REQUIRE((p >= 0) == (row >= 0 && row < W << shift && table[row >> shift] >= 0 && table[row >> shift] < pages));
        const int kvh = rng() % kh;
        // the attention kernels read 16 rows from a multiple of 16 on, from page 0 where there is none
        const size_t at = row_offset(p, stride, kvh, row & ~15, shift, D);
        REQUIRE(at + (size_t)16 * D <= elements);
        REQUIRE(row_offset(p, stride, kvh, row, shift, D) + D <= elements);
        int first, count;
        const int T = 1 + rng() % 50, s0 = rng() % 2 ? any(odd) : (int)(rng() % (T + 3)), s1 = rng() % 2 ? any(odd) : (int)(rng() % (T + 3));
        clamp_tokens(s0, s1, T, first, count);
        REQUIRE(first >= 0 && count >= 0 && first + count <= T);
        if (0 <= s0 && s0 <= s1 && s1 <= T) REQUIRE(first == s0 && count == s1 - s0);
    }
    // shares
    for (int round = 0; round < 4000; ++round) {
        const int shift = 4 + rng() % 5, B = 1 + rng() % 70, W = 1 + rng() % 200, shares = 1 + rng() % (rng() % 2 ? 3 : 2048);
        std::vector<int> rows(B);
        long long total = 0;
        for (int& r : rows) {
            r = clamp_length(rng() % 4 ? (int)(rng() % ((W << shift) + 1)) : any(odd), W, shift);
            total += units_of(r);
        }
        const int share = share_of_units(total, shares);
        REQUIRE(share >= 1);
        long long slots = 0;
        for (int r : rows) {
            const int count = shares_of(units_of(r), share);
            REQUIRE((count == 0) == (r == 0));
            slots += count;
            int next = 0;
            for (int i = 0; i < count; ++i) {
                int r0, r1;
                share_rows(r, count, i, r0, r1);
                REQUIRE(r0 == next && r1 >= r0 && r1 <= r && (r0 % 16 == 0 || r0 == r));
                next = r1;
            }
            REQUIRE(next == r);
        }
        REQUIRE(slots <= decode_slots(B, W, shift, shares));
    }
    // tiles of prompts and their parts
    for (int round = 0; round < 4000; ++round) {
        const int B = 1 + rng() % 12, group = any({1, 2, 3, 4, 7, 8, 16, 40, 128, 200}), shares = any({1, 2, 64, 512}), height = any({64, 128});
        std::vector<PromptTiles> seqs(B);
        long long bound = 0, blocks = 0;
        for (auto& t : seqs) {
            t = PromptTiles{rng() % 4 ? (int)(rng() % 900) : 0, group, (rng() % 3 ? (int)(rng() % 3000) : (int)(rng() % 40) - 700), height};
            long long sum = 0;
            for (int i = 0; i < t.tiles(); ++i) sum += t.blocks(i);
            REQUIRE(sum <= t.blocks_bound());
            for (int x : {1, 2, 5, 8, 13, 40}) {
                int over = 0;
                for (int i = 0; i < t.tiles(); ++i) over += t.blocks(i) > x;
                REQUIRE(over == t.tiles_over(x));
            }
            bound += t.blocks_bound();
            blocks += sum;
        }
        const int share = prompt_share(bound, shares);
        long long items = 0, tiles = 0, parts = 0, cut = 0;
        for (const auto& t : seqs) {
            std::vector<int> seen(t.tiles(), 0), slot(t.parts(share) + 1, 0);
            for (int i = 0; i < t.items(share); ++i) {
                const PromptItem it = prompt_item(t, share, i);
                REQUIRE(it.tile >= 0 && it.tile < t.tiles());
                REQUIRE(it.part == 0 || it.part * share < t.blocks(it.tile));
                seen[it.tile] |= 1 << it.part;
                if (t.blocks(it.tile) > share) {
                    REQUIRE(it.slot >= 0 && it.slot < t.parts(share) && !slot[it.slot]);
                    slot[it.slot] = 1;
                }
            }
            for (int i = 0; i < t.tiles(); ++i) {
                const int n = std::max(1, (t.blocks(i) + share - 1) / share);
                REQUIRE(n < 31 && seen[i] == (1 << n) - 1);
            }
            items += t.items(share);
            tiles += t.tiles();
            if (t.tiles_over(share)) parts += t.parts(share);
            else REQUIRE(t.parts(share) == 0);
            cut += t.tiles_over(share);
        }
        REQUIRE(items <= tiles + shares && parts <= 2 * shares && cut <= shares);
    }
    REQUIRE(share_of_units(65535ll << 23, 1) == 1 << 24 && shares_of(1 << 23, 1 << 24) == 1);
    printf("ok\n");
    return 0;
}
