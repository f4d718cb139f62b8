// Where the rows of a paged cache are and how decode work is shared out: the arithmetic of every index that the kernels
// of the paged operators take from device data, in one place and free of the device, so that it also runs on a host.
#pragma once

#include <stddef.h>

#if defined(__HIP__)
#define MOSS_HD __host__ __device__ __forceinline__
#else
#define MOSS_HD inline
#endif

namespace moss {

MOSS_HD int clamp_int(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// Rows of a sequence that the table can hold, whatever the length says (W << shift <= 2^30).
MOSS_HD int clamp_length(int length, int W, int shift) { return clamp_int(length, 0, W << shift); }

// A table entry as a page, or -1 for none.
MOSS_HD int page_or_none(int entry, int pages) { return entry >= 0 && entry < pages ? entry : -1; }

// The page of row `row` of a sequence with table row `trow`, or -1: no such row, or no page.
MOSS_HD int page_of_row(const int* trow, int row, int W, int shift, int pages) {
    if (row < 0 || (row >> shift) >= W) return -1;
    return page_or_none(trow[row >> shift], pages);
}

// Elements from the cache's start to row `row` of a KV head in a page (-1 reads as page 0: its values are not used).
MOSS_HD size_t row_offset(int page, long long page_stride, int kvh, int row, int shift, int D) {
    return (size_t)(page < 0 ? 0 : page) * (size_t)page_stride +
           (((size_t)kvh << shift) + (size_t)(row & ((1 << shift) - 1))) * (size_t)D;
}

// First packed token and number of tokens of a sequence, inside [0, T] whatever `starts` holds.
MOSS_HD void clamp_tokens(int s0, int s1, int T, int& first, int& count) {
    first = clamp_int(s0, 0, T);
    count = clamp_int(s1, first, T) - first;
}

// Decode work: rows in units, the units of all sequences in shares of `share` units, at most `shares` of them and one
// more per sequence; a sequence's units are spread evenly over its own shares.
constexpr int kUnit = 128;
MOSS_HD int units_of(int rows) { return (rows + kUnit - 1) / kUnit; }
template <typename N>  // of int (totals up to 2^30) or long long
MOSS_HD int share_of_units(N total, int shares) {
    const N share = total <= shares ? 1 : (total + shares - 1) / shares;
    return share < (1 << 24) ? (int)share : 1 << 24;  // no sequence has more units
}
MOSS_HD int shares_of(int units, int share) { return (units + share - 1) / share; }
MOSS_HD void share_rows(int rows, int count, int index, int& r0, int& r1) {
    const int per = (units_of(rows) + count - 1) / count;
    const long long from = (long long)index * per * kUnit, to = from + (long long)per * kUnit;
    r0 = from < rows ? (int)from : rows;
    r1 = to < rows ? (int)to : rows;
}

// Prompt work: tiles of `height` (128 or 64) (token, head) rows, which see keys up to their last row's position, in blocks of
// kPromptBlock keys; a tile of more than `share` blocks is cut into parts of that many.  The sum of all tiles' blocks is
// at most `shares` times the share, so at most `shares` parts come on top of the tiles and the parts of the cut tiles are at
// most twice as many.
constexpr int kPromptBlock = 64, kPromptShare = 8;
struct PromptTiles {
    int tokens, group, pos0, height;  // new tokens of a sequence, query heads per KV head, position of the first one
    MOSS_HD int rows() const { return tokens * group; }
    MOSS_HD int tiles() const { return (rows() + height - 1) / height; }
    MOSS_HD int token_of(int row) const { return (int)((unsigned)row / (unsigned)group); }
    MOSS_HD int last_key(int tile) const {  // -1 and below: none
        const int row = (tile + 1) * height - 1;
        return pos0 + token_of(row < rows() - 1 ? row : rows() - 1);
    }
    MOSS_HD int blocks(int tile) const {
        const int last = last_key(tile);
        return last < 0 ? 0 : last / kPromptBlock + 1;
    }
    // tiles, the last ones, of more than `blocks` (> 0) blocks
    MOSS_HD int tiles_over(int blocks) const {
        const long long y = (long long)blocks * kPromptBlock - pos0;  // tokens before the first that sees so many
        const int n = tiles();
        if (y <= 0) return n;
        if (y > tokens - 1) return 0;
        const int first = ((int)y * group + height) / height - 1;  // ceil((y group + 1) / rows) - 1
        return (first < n - 1 ? n - 1 - first : 0) + 1;
    }
    // no less than the sum of blocks() over the tiles: they rise no faster than a line (rows are at most 2^30)
    MOSS_HD long long blocks_bound() const {
        const int n = tiles();
        if (n == 0) return 0;
        const int end = pos0 + token_of(n * height - 1);
        return ((long long)n * (blocks(0) + (end < 0 ? 0 : end / kPromptBlock + 1) + 2) + 1) / 2;
    }
    MOSS_HD int items(int share) const {
        int n = tiles();
        for (int k = 1, c = 1; c > 0; ++k) n += c = tiles_over(k * share);
        return n;
    }
    MOSS_HD int parts(int share) const {
        int n = tiles_over(share);
        for (int k = 1, c = 1; c > 0; ++k) n += c = tiles_over(k * share);
        return n;
    }
};
MOSS_HD int prompt_share(long long blocks, int shares) {
    const long long share = (blocks + shares - 1) / shares;
    return share < kPromptShare ? kPromptShare : share < (1 << 24) ? (int)share : 1 << 24;
}
// A sequence's item: part `part` of `count` of tile `tile`, whose first partial result is number `slot` (of the
// sequence's; its parts are tiles_over(share) apart at part 0 and then as the parts are listed).
struct PromptItem {
    int tile, part, slot;
};
MOSS_HD PromptItem prompt_item(const PromptTiles& t, int share, int index) {
    const int n = t.tiles();
    if (index < n) return PromptItem{n - 1 - index, 0, index};  // parts 0: of the cut tiles the first numbers
    int slot = t.tiles_over(share);
    index -= n;
    for (int k = 1;; ++k) {
        const int c = t.tiles_over(k * share);
        if (index < c || c == 0) return PromptItem{n - 1 - index, k, slot + index};
        index -= c;
        slot += c;
    }
}
// The item stands for a part of a tile: false for a number behind the sequence's items, as starts or lengths that change
// under the kernel can lead to (its tile is -1 or less, or the part lies behind the tile's blocks).
MOSS_HD bool is_item(const PromptTiles& t, int share, const PromptItem& it) {
    return it.tile >= 0 && (it.part == 0 || (long long)it.part * share < t.blocks(it.tile));
}
// Partial results first .. first + count - 1 lie in a workspace of `slots` (lengths that change between the launches can name
// others).
MOSS_HD bool in_slots(int first, int count, long long slots) { return first >= 0 && count >= 0 && (long long)first + count <= slots; }
// Shared prefixes (paged_shared.hip).  The rows that a run of sequences shares, whose first one has `length` and shares `want`; where
// a sequence's own rows begin: behind those, in whole 16 rows (which a page holds all of), or nowhere.
MOSS_HD int shared_rows(int want, int length) { return (want < length ? want : length) & ~15; }
MOSS_HD int shared_from(int rows, int want, int length) {
    const int most = want < rows ? want : rows;
    return length <= most ? length : most & ~15;
}
// The rows of a run that its prefix is read for: what the sequences behind the first one take of them, `most` the largest of their
// shared_from (whose values stay the same with these rows in place of all that the first one shares).
MOSS_HD int taken_rows(int most) { return (most + 15) & ~15; }
// Own rows of a unit.  32 / 64 / 128: four sequences of 700 11.9 / 12.4 / 14.6 us, 64 over 4096 shared rows 41.9 / 37.8 / 42.6.
constexpr int kOwnUnit = 64;
MOSS_HD int own_units(int rows) { return (rows + kOwnUnit - 1) / kOwnUnit; }
// A line of work, `all` long, in `pieces` equal pieces.  Part (piece w, thing k) of what the line holds in order has the number
// w + k: either grows along the line, and from a part to the next one of them does.
MOSS_HD int piece_of(long long all, int pieces) {
    const long long piece = all < 1ll << 31 ? (long long)(((unsigned)all + (unsigned)pieces - 1) / (unsigned)pieces) : (all + pieces - 1) / pieces;
    return piece < 1 ? 1 : piece < (1ll << 30) ? (int)piece : 1 << 30;
}
// Of `workgroups` (2 at least), how many take the prefixes' blocks and not the units of own rows.
// (1 : 1 / 3 : 2 / 2 : 1 / 3 : 1: 64 sequences over 4096 shared rows 40.5 / 37.8 / 42.1 / 41.5 us, 40 in five runs over 8 bits 28.8 / 28.9 /
// 28.0 / 29.5, 64 over 16384 74 / 73 / 77 / 90.  One ratio for all forms: 8 bits alone would take 2 : 1.)
constexpr float kBlockCost = 3.f, kUnitCost = 2.f;
MOSS_HD int prefix_takers(float blocks, float units, int workgroups) {
    if (blocks <= 0.f) return 0;
    if (units <= 0.f) return workgroups;
    const float share = blocks * kBlockCost / (blocks * kBlockCost + units * kUnitCost);
    return clamp_int((int)(share * (float)workgroups + 0.5f), 1, workgroups - 1);
}
MOSS_HD long long quotient(long long a, int b) {  // of what is not negative; in 32 bits where that is enough
    return a < 1ll << 32 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}
inline long long decode_slots(int B, int W, int shift, int shares) {
    const long long most = (long long)B * ((((long long)W << shift) + kUnit - 1) / kUnit);
    return (long long)B + shares < most ? (long long)B + shares : most;
}

}  // namespace moss
