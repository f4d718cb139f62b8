// What the operators over a paged key-value cache share: the cache and batch descriptions, element types, and the
// search for the sequence that a token or a workgroup belongs to.
//
// A cache holds pages of P rows (P = 1 << shift >= 16) per KV head: K and V [pages, KH, P, D], the page stride free.
// Row r of sequence b lies in page table[b][r >> shift]; an entry outside [0, pages) names no page, and its rows take
// no part.  Everything that says where rows are lives on the device, so a captured graph follows growing sequences:
// the kernels clamp lengths to what the table holds and starts to the packed rows, and no entry can lead an access
// outside the cache.
#pragma once

#include "wave_scan.h"
#include "paged_index.h"

namespace moss {

struct PagedCache {
    uint16_t* k;
    uint16_t* v;
    long long k_stride, v_stride;  // elements from a page to the next
    int pages, kh, shift;
};

struct PagedBatch {
    const int* table;    // [B, W], rows table_stride apart
    const int* lengths;  // [B]: rows of each sequence, new tokens included
    const int* starts;   // [B + 1]: first packed token of each sequence (NULL: one token a sequence)
    int B, W;
    long long table_stride;
};

// ---------------------------------------------------------------- element types (16 bits)
typedef __bf16 bf16x8_v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_v __attribute__((ext_vector_type(2)));
typedef float f32x4_v __attribute__((ext_vector_type(4)));
typedef float f32x16_v __attribute__((ext_vector_type(16)));
typedef unsigned int u32x2_v __attribute__((ext_vector_type(2)));

struct Bf16 {
    static __device__ __forceinline__ float lo(uint32_t w) { return bf16_lo(w); }
    static __device__ __forceinline__ float hi(uint32_t w) { return bf16_hi(w); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
    static __device__ __forceinline__ f32x4_v mfma16(u32x4_t a, u32x4_t b, f32x4_v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c,
                                                       0, 0, 0);
    }
    static __device__ __forceinline__ f32x16_v mfma32(u32x4_t a, u32x4_t b, f32x16_v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c,
                                                       0, 0, 0);
    }
};

struct F16 {
    static __device__ __forceinline__ float lo(uint32_t w) { return (float)__builtin_bit_cast(f16x2_v, w)[0]; }
    static __device__ __forceinline__ float hi(uint32_t w) { return (float)__builtin_bit_cast(f16x2_v, w)[1]; }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {  // round to nearest even, one value at a time
        const f16x2_v v = {(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(uint32_t, v);
    }
    static __device__ __forceinline__ f32x4_v mfma16(u32x4_t a, u32x4_t b, f32x4_v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_v, a), __builtin_bit_cast(f16x8_v, b), c, 0,
                                                      0, 0);
    }
    static __device__ __forceinline__ f32x16_v mfma32(u32x4_t a, u32x4_t b, f32x16_v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_v, a), __builtin_bit_cast(f16x8_v, b), c, 0,
                                                      0, 0);
    }
};

// ---------------------------------------------------------------- where things are
__device__ __forceinline__ int paged_length(const PagedBatch& bt, int b, int shift) {
    return clamp_length(bt.lengths[b], bt.W, shift);
}

// First packed token (x) and number of tokens (y) of sequence b.
__device__ __forceinline__ int2 paged_tokens(const PagedBatch& bt, int b, int T) {
    int2 r;
    clamp_tokens(bt.starts[b], bt.starts[b + 1], T, r.x, r.y);
    return r;
}

// A sequence of the batch and what the caller looks for in it.
struct Place {
    int b;      // -1: the index lies behind the last item
    int index;  // the item's number within the sequence
    int count;  // the sequence's items
};

// The sequences' items counted in order (count(b) of sequence b): whose the item `item` is.  Every wave finds it by
// itself, 64 sequences at a time; the result is uniform.
template <typename Count>
__device__ __forceinline__ Place find_item(int B, int item, int lane, Count count) {
    int before = 0;
    for (int b0 = 0; b0 < B; b0 += kWave) {
        const int n = b0 + lane < B ? count(b0 + lane) : 0;
        const int through = wave_prefix(n);
        const unsigned long long past = __ballot(before + through > item);
        if (past) {
            const int l = __builtin_ctzll(past);
            const int c = __builtin_amdgcn_readlane(n, l), t = before + __builtin_amdgcn_readlane(through, l);
            return Place{b0 + l, item - (t - c), c};
        }
        before += __builtin_amdgcn_readlane(through, kWave - 1);
    }
    return Place{-1, 0, 0};
}

// ---------------------------------------------------------------- host checks
static inline bool paged_shape_ok(const PagedCache& c, const PagedBatch& b, int qh, int d) {
    return c.pages > 0 && c.kh > 0 && qh > 0 && qh % c.kh == 0 && qh <= 1024 && (d == 64 || d == 128) && c.shift >= 4 &&
           c.shift <= 12 && b.B > 0 && b.B <= 65535 && b.W > 0 && ((long long)b.W << c.shift) <= (1ll << 30) &&
           b.table_stride >= b.W && c.k_stride % 8 == 0 && c.v_stride % 8 == 0 &&
           c.k_stride >= ((long long)c.kh << c.shift) * d && c.v_stride >= ((long long)c.kh << c.shift) * d;
}

static inline bool paged_pointers_ok(const PagedCache& c, const PagedBatch& b) {
    return c.k && c.v && b.table && b.lengths && MOSS_ALIGNED(c.k, 16) && MOSS_ALIGNED(c.v, 16) && MOSS_ALIGNED(b.table, 4) &&
           MOSS_ALIGNED(b.lengths, 4) && MOSS_ALIGNED(b.starts, 4);
}

// log2 of a page's rows, or -1
static inline int page_shift(int rows) {
    for (int s = 4; s <= 12; ++s)
        if (rows == 1 << s) return s;
    return -1;
}

static inline PagedCache paged_cache(const void* k, const void* v, long long k_stride, long long v_stride, int pages, int kh,
                                     int page_rows) {
    return PagedCache{(uint16_t*)k, (uint16_t*)v, k_stride, v_stride, pages, kh, page_shift(page_rows)};
}

}  // namespace moss
