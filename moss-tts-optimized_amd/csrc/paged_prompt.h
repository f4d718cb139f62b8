// Rows of queries (up to 32 a wave) over a range of keys of a paged cache, on the matrix cores: the inner part of the attentions
// that have many rows for the same keys, with the running maximum m and sum l of each row.
//
//   S^T = K Q^T: 32 keys x 32 rows per matrix instruction, so a lane holds one row and 16 of its keys, and the row's
//   maximum needs one exchange with the lane 32 away; the running maximum and sum are fp32, base 2.
//   O^T += V^T P^T: P, in 16 bits, is the B operand as S^T left it.
// The prompt form rounds P to 16 bits: the one step with fewer bits before the output, as in the single request's prompt attention;
// the sum adds up the unrounded values.  (P = 2^(s scale - m) with m a rounded product: a row's largest P is 1 up to that rounding,
// which l and O share.)  Split into two 16-bit values (SPLIT), as the decode form has it, P adds nothing to the output's own
// rounding, but costs half as many matrix instructions again where they are what bounds: 8000 tokens 555 -> 724 us, from 8 bits 571
// -> 770, nine prompts 60 -> 67, from 8 bits 54 -> 67, for an error against 64 bits of 1.65 instead of 1.88 and 1.64 instead of 1.78
// 10^-3 (heads of 128, bf16; fp16 an eighth).  Shared prefixes split it, since they stand beside rows that the decode form takes, and
// which rows are whose follows from the rest of the batch: 64 sequences over 4096 rows 35.0 us either way, 40 in groups over 8 bits
// 25.4 -> 26.9, for an error of 1.66 instead of 1.75 10^-3; there each half of a tile's P is used as soon as it is formed, or its two
// values would not fit the registers (36.5 and 27.6 us).
// Blocks of 64 keys lie in LDS in one of two stages while the other is consumed, one barrier per block.  From a 16-bit cache
// they go there straight from the pages (buffer loads, 16 rows of K and of V a wave, which lie in one page;
// rows that nobody sees or that have no page are read as zeros: past the buffer's end), without registers.  From one in 8 bits
// they pass through registers, where each is converted once for all the workgroup's waves: the codes and scales of the next block
// are loaded before this one's products and written behind them.  V is read transposed (ds_read_b64_tr_b16: a lane gets one
// dim of 4 rows).  16-byte chunk c of row r lies at c ^ f(r), which spreads the rows of one read over the banks.
#pragma once

#include "paged8.h"

namespace moss {

// Where 16-byte chunk c of key row r lies in its LDS row: c ^ f(r).
template <int D>
__device__ __forceinline__ int k_swizzle(int r) { return D == 128 ? r & 15 : (r >> 1) & 7; }
template <int D>
__device__ __forceinline__ int v_swizzle(int r) {
    return D == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : ((r >> 1 & 1) << 2) | ((r >> 2) & 3);
}

// 16 bytes per lane straight to lds + 16 lane.  (In a function of its own: the host's pass drops a kernel that names a
// builtin it does not know.)
__device__ __forceinline__ void copy16(const Span& s, unsigned char* lds, uint32_t voff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(span_rsrc(s), lds, 16, voff, 0, 0, 0);
}

typedef short s16x4_v __attribute__((ext_vector_type(4)));
// 4 rows of one dim: a 16-lane group reads 4 rows of 16 dims, lane i the 8 bytes of row i / 4 from dim 4 (i % 4) on.
__device__ __forceinline__ u32x2_v read_transposed(const unsigned char* p) {
    return __builtin_bit_cast(u32x2_v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_v*)p));
}

// Blocks of keys from the pages into a stage: begin() issues what block b needs, end() leaves it in `stage` (complete() of the
// caller's wait and barrier).  row0: the wave's 16 rows of a block.
template <typename E, int D>
struct Stage16 {  // straight into LDS
    using Cache = PagedCache;
    // where chunk c of row r lies
    static __device__ __forceinline__ int k_slot(int c, int r) { return c ^ k_swizzle<D>(r); }
    static __device__ __forceinline__ int v_slot(int c, int r) { return c ^ v_swizzle<D>(r); }
    static constexpr int RB = 2 * D, NL = 16 * RB / 1024, RPL = 1024 / RB, CPR = D / 8;  // loads of 16 rows, rows of a load
    uint32_t kload[NL], vload[NL];  // LDS offsets: this lane's part of a load
    __device__ __forceinline__ explicit Stage16(int lane) {
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            const int r = j * RPL + lane / CPR, slot = lane % CPR;
            kload[j] = (uint32_t)(r * RB + 16 * (slot ^ k_swizzle<D>(r)));
            vload[j] = (uint32_t)(r * RB + 16 * (slot ^ v_swizzle<D>(r)));
        }
    }
    __device__ __forceinline__ void begin(unsigned char* stage, const Cache& c, int page, int kvh, int key, int rows, int wave) {
        const uint32_t bytes = (uint32_t)(rows * RB);
        const Span ks{c.k + row_offset(page, c.k_stride, kvh, key, c.shift, D), bytes};
        const Span vs{c.v + row_offset(page, c.v_stride, kvh, key, c.shift, D), bytes};
        unsigned char* at = stage + 16 * RB * wave;
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            copy16(ks, at + 1024 * j, kload[j]);
            copy16(vs, at + kPromptBlock * RB + 1024 * j, vload[j]);
        }
    }
    __device__ __forceinline__ void end(unsigned char*, int) {}
    // a key's rows for one query at a time, from dim d on: 8 values of K, 4 of V
    struct Key {
        const uint16_t *k, *v;
        __device__ __forceinline__ u32x4_t key8(int at) const { return *reinterpret_cast<const u32x4_t*>(k + at); }
        __device__ __forceinline__ u32x2_v value4(int at) const { return *reinterpret_cast<const u32x2_v*>(v + at); }
    };
    static __device__ __forceinline__ Key key_of(const Cache& c, int page, int kvh, int key, int dk, int dv) {
        return Key{c.k + row_offset(page, c.k_stride, kvh, key, c.shift, D) + dk, c.v + row_offset(page, c.v_stride, kvh, key, c.shift, D) + dv};
    }
};

// 16 bytes per lane, one byte, of a span.
__device__ __forceinline__ uint32_t load1(const Span& s, uint32_t voff) {
    return __builtin_amdgcn_raw_buffer_load_b8(span_rsrc(s), voff, 0, 0);
}

template <typename E, int D>
struct Stage8 {  // codes in registers until the block before is consumed
    using Cache = PagedCache8;
    static constexpr int RB = 2 * D, LPR = D / 16, RPL = kWave / LPR, NL = 16 / RPL;  // lanes of a row, rows of a load, loads of 16 rows
    // Where chunk c of row r lies: spread for the reads as Stage16's, and so that the eight lanes of a write, which hold every second
    // chunk of a row (D 128) or of two (D 64), meet all banks: with Stage16's order a write takes twice as long (8000 tokens 577 ->
    // 571 us, 40 sequences over five shared prefixes 28.2 -> 26.8).
    static __device__ __forceinline__ int k_slot(int c, int r) {
        if (D == 128) return ((c >> 1) | (c & 1) << 3) ^ (r & 15);
        return ((c >> 1) | (c & 1) << 2) ^ (((r & 1) << 2 | (r >> 1 & 3)) ^ (r >> 3 & 1) << 2);
    }
    static __device__ __forceinline__ int v_slot(int c, int r) {
        if (D == 128) return ((c >> 1) ^ (c & 1) ^ (r & 3) << 1) | (c & 1) << 3;
        return c ^ (r & 1) * 3 ^ (r & 2) << 1;
    }
    uint32_t kput, vput;  // LDS offsets of this lane's first chunk of 8 values; chunk i of load j: see end()
    uint32_t at;          // its codes in 16 rows
    int row;
    u32x4_t k[NL], v[NL];
    uint32_t ks[NL], vs[NL];
    __device__ __forceinline__ explicit Stage8(int lane) : at(16 * lane), row(lane / LPR) {
        kput = (uint32_t)(row * RB + 16 * k_slot(2 * (lane % LPR), row));
        vput = (uint32_t)(row * RB + 16 * v_slot(2 * (lane % LPR), row));
    }
    __device__ __forceinline__ void begin(unsigned char*, const Cache& c, int page, int kvh, int key, int rows, int) {
        const Span kc{c.kc() + row_offset(page, c.k_stride, kvh, key, c.shift, D), (uint32_t)(rows * D)};
        const Span vc{c.vc() + row_offset(page, c.v_stride, kvh, key, c.shift, D), (uint32_t)(rows * D)};
        const Span kb{c.ks + row_offset(page, c.ks_stride, kvh, key, c.shift, 1), (uint32_t)rows};
        const Span vb{c.vs + row_offset(page, c.vs_stride, kvh, key, c.shift, 1), (uint32_t)rows};
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            k[j] = load16(kc, at + 1024 * j, 0);
            v[j] = load16(vc, at + 1024 * j, 0);
            ks[j] = load1(kb, row + RPL * j);
            vs[j] = load1(vb, row + RPL * j);
        }
    }
    __device__ __forceinline__ void end(unsigned char* stage, int wave) {
        unsigned char* to = stage + 16 * RB * wave;
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            const float a = scale_of(ks[j]), b = scale_of(vs[j]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                // the slots of the next chunk and of the row 8 further on (D 128) are some bits away
                const uint32_t kat = (kput ^ (D == 128 ? 128 * i ^ 128 * j : 64 * i)) + RPL * RB * j;
                const uint32_t vat = (vput ^ (D == 128 ? 144 * i : 16 * i)) + RPL * RB * j;
                *reinterpret_cast<u32x4_t*>(to + kat) = widen8<E>(k[j][2 * i], k[j][2 * i + 1], a);
                *reinterpret_cast<u32x4_t*>(to + kPromptBlock * RB + vat) = widen8<E>(v[j][2 * i], v[j][2 * i + 1], b);
            }
        }
    }
    struct Key {
        const uint8_t *k, *v;
        float ks, vs;
        __device__ __forceinline__ u32x4_t key8(int at) const {
            const u32x2_v w = *reinterpret_cast<const u32x2_v*>(k + at);
            return widen8<E>(w[0], w[1], ks);
        }
        __device__ __forceinline__ u32x2_v value4(int at) const {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(v + at);
            return u32x2_v{widen<E, false>(w, vs), widen<E, true>(w, vs)};
        }
    };
    static __device__ __forceinline__ Key key_of(const Cache& c, int page, int kvh, int key, int dk, int dv) {
        return Key{c.kc() + row_offset(page, c.k_stride, kvh, key, c.shift, D) + dk,
                   c.vc() + row_offset(page, c.v_stride, kvh, key, c.shift, D) + dv,
                   scale_of(c.ks[row_offset(page, c.ks_stride, kvh, key, c.shift, 1)]),
                   scale_of(c.vs[row_offset(page, c.vs_stride, kvh, key, c.shift, 1)])};
    }
};

// A wave's rows (those of wave % (4 / KS) of the workgroup's tile) and the keys that its workgroup takes for them (all but qpos uniform over the wave, trow to last over the
// workgroup).
struct TileRows {
    const int* trow;            // the sequence's pages
    int kvh, b0, b1, last;      // KV head; blocks b0 .. b1 - 1; the last key that any row sees
    int qpos;                   // this lane's row (lane % 32) sees keys 0 .. qpos
    int wave_first, wave_last;  // the wave's rows all see keys up to the first, none a key behind the second
    bool idle;                  // no row of this wave's exists
};

// A stage of K | V in LDS.  A workgroup has two, as two variables, so that reading one does not wait for the loads into the other.
template <int D>
using Stage = unsigned char[4 * D * kPromptBlock];

// The thread's index for a function that is called in a loop: what such a function computes from it is computed in each call, and
// not kept in registers from one to the next.
__device__ __forceinline__ int fresh_thread() {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    return tid;
}

// SPLIT: P as the sum of two 16-bit values.
// o, m, l of the rows (l summed over the lane's keys and, on return, its partner's).  KS 2: two waves share the rows and halve a
// block's keys; false: this wave's part went to the other.
template <typename E, int D, int KS, bool SPLIT, typename S>
__device__ __forceinline__ bool attend_rows(const typename S::Cache& c, const TileRows& t, int W, const u32x4_t (&qf)[D / 16], float scale,
                                            int tid, Stage<D>& even, Stage<D>& odd, f32x16_v (&o_out)[D / 32], float& m_out, float& l_out) {
    constexpr int NT = 2 / KS, BK = kPromptBlock, DT = D / 32, DK = D / 16, RB = 2 * D, KB = BK * RB;  // NT: a wave's 32-key tiles
    const int lane = tid & 63, half = lane >> 5, rl = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), rw = wave % (4 / KS), kq = KS == 1 ? 0 : wave / (4 / KS);
    const int kvh = t.kvh, b0 = t.b0, b1 = t.b1, last = t.last, qpos = t.qpos, wave_first = t.wave_first, wave_last = t.wave_last;
    const bool idle = t.idle;
    const int* trow = t.trow;
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    f32x16_v o[DT];  // (the caller's own in the loop cost 28 registers, a workgroup a CU for heads of 64)
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    float m = -INFINITY, l = 0.f;  // l: this lane's keys only

    // Blocks are taken from the last one down, so that the ones that not all rows see come first.
    // pages: lane i holds that of 16-row group i % 4 of the i / 4-th of the next 16 blocks (-1: none, or behind the last key);
    // bit i of `there` says that the group's rows up to the last key exist
    int pages = -1;
    unsigned long long there = 0, there_next = 0;
    auto fetch_pages = [&](int b) {
        const int key = BK * (b - lane / 4) + 16 * (lane & 3);
        pages = key >= 0 && key <= last ? page_or_none(trow[key >> c.shift], c.pages) : -1;
        there_next = __ballot(pages >= 0 || key > last);
    };
    S source(lane);
    auto copy = [&](unsigned char* stage, int b) {  // block b's rows 16 wave .. + 15
        if (((b1 - 1 - b) & 15) == 0) fetch_pages(b);
        const int page = __builtin_amdgcn_readlane(pages, 4 * ((b1 - 1 - b) & 15) + wave), key = BK * b + 16 * wave;
        source.begin(stage, c, page, kvh, key, uniform(page < 0 ? 0 : min(max(last + 1 - key, 0), 16)), wave);
    };
    uint32_t kread[DK], vread[2][DT];
#pragma unroll
    for (int kk = 0; kk < DK; ++kk) kread[kk] = (uint32_t)((32 * kq + rl) * RB + 16 * S::k_slot(2 * kk + half, rl));
    {
        const int i = lane & 15, r = 4 * half + (i >> 2), chunk = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                vread[s2][dt] = (uint32_t)((32 * kq + r + 8 * s2) * RB + 16 * S::v_slot(4 * dt + chunk, r + 8 * s2) + 8 * (i & 1));
    }

    // O of this wave's keys from block b on, one key at a time and from memory, each row taking the keys it sees alone.
    auto again = [&](int b) {
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
        for (int j = 0; j < 32 * NT * (b1 - b); ++j) {
            const int key = uniform(BK * (b + j / (32 * NT)) + 32 * kq + j % (32 * NT));
            if (key > wave_last) break;
            const int page = uniform(page_of_row(trow, key, W, c.shift, c.pages));
            if (page < 0) continue;
            const typename S::Key row = S::key_of(c, page, kvh, key, 8 * half, 4 * half);
            float dot = 0.f;
#pragma unroll
            for (int kk = 0; kk < DK; ++kk) {
                const u32x4_t kw = row.key8(16 * kk);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    dot = fmaf(E::hi(qf[kk][i]), E::hi(kw[i]), fmaf(E::lo(qf[kk][i]), E::lo(kw[i]), dot));
            }
            dot = sum_xor32(dot);
            if (key > qpos) continue;
            const float p = __builtin_amdgcn_exp2f(fmaf(dot, scale, -(m == -INFINITY ? 0.f : m)));
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    const u32x2_v v = row.value4(32 * dt + 8 * q4);
                    o[dt][4 * q4] = fmaf(p, E::lo(v[0]), o[dt][4 * q4]);
                    o[dt][4 * q4 + 1] = fmaf(p, E::hi(v[0]), o[dt][4 * q4 + 1]);
                    o[dt][4 * q4 + 2] = fmaf(p, E::lo(v[1]), o[dt][4 * q4 + 2]);
                    o[dt][4 * q4 + 3] = fmaf(p, E::hi(v[1]), o[dt][4 * q4 + 3]);
                }
        }
    };
    auto products = [&](const unsigned char* ks, int b, unsigned int groups) {
        const int first = BK * b + 32 * kq;  // this wave's keys: 32 NT from here on, and their 16-row groups
        if (idle || first > wave_last) return;  // none of its rows sees any of its keys
        const unsigned char* vs = ks + KB;
        f32x16_v s[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) s[i] = f32x16_v{};
#pragma unroll
        for (int kk = 0; kk < DK; ++kk)
#pragma unroll
            for (int i = 0; i < NT; ++i)
                s[i] = E::mfma32(*reinterpret_cast<const u32x4_t*>(ks + kread[kk] + 32 * RB * i), qf[kk], s[i]);
        // element e of tile i: key first + 32 i + 8 (e / 4) + 4 half + e % 4, row rl
        if (groups != (1u << 2 * NT) - 1 || first + 32 * NT - 1 > wave_first) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int key = first + 32 * i + 8 * (e >> 2) + 4 * half + (e & 3);
                    s[i][e] = key <= qpos && (groups >> (2 * i + (e >> 3)) & 1) ? s[i][e] : -INFINITY;
                }
        }
        float mx = s[0][0];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 2) mx = fmaxf(fmaxf(mx, s[i][e]), s[i][e + 1]);
        mx = max_xor32(mx) * scale;
        if (__any(mx > m)) {
            const float mn = fmaxf(m, mx);
            const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= f;
        }
        const float mr = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            u32x4_t pf[2], pl[2];
            // keys 16 u + {4 half + 0..3, 8 + 4 half + 0..3} of the tile: their P, and the K step over them
            auto weights = [&](int u) {
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(s[i][8 * u + 2 * v], scale, -mr));
                    const float p1 = __builtin_amdgcn_exp2f(fmaf(s[i][8 * u + 2 * v + 1], scale, -mr));
                    l += p0 + p1;
                    pf[u][v] = E::pack(p0, p1);
                    if constexpr (SPLIT) pl[u][v] = E::pack(p0 - E::lo(pf[u][v]), p1 - E::hi(pf[u][v]));
                }
            };
            auto step = [&](int u) {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const u32x2_v a0 = read_transposed(vs + vread[0][dt] + (32 * i + 16 * u) * RB);
                    const u32x2_v a1 = read_transposed(vs + vread[1][dt] + (32 * i + 16 * u) * RB);
                    o[dt] = E::mfma32(u32x4_t{a0[0], a0[1], a1[0], a1[1]}, pf[u], o[dt]);
                    if constexpr (SPLIT) o[dt] = E::mfma32(u32x4_t{a0[0], a0[1], a1[0], a1[1]}, pl[u], o[dt]);
                }
            };
            weights(0);
            if constexpr (SPLIT) step(0);  // at once: both halves' P in two values would not fit the registers
            weights(1);
            if constexpr (!SPLIT) step(0);
            step(1);
        }
        if (first + 32 * NT - 1 > wave_first) {
            // A P of 0 times a NaN or infinity in V of a key that a row does not see is a NaN all the same.
            float z = 0.f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) z = fmaf(o[dt][e], 0.f, z);
            if (__any(z != z)) again(b);
        }
    };
    auto block = [&](const unsigned char* ks, unsigned char* next, int b) {
        // this wave's rows of block b are there, then everyone's; and everyone is done with block b + 1's stage
        __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));  // vmcnt(0)
        __syncthreads();
        if (((b1 - 1 - b) & 15) == 0) there = there_next;
        const unsigned int groups = (unsigned int)(there >> (4 * ((b1 - 1 - b) & 15) + 2 * kq)) & ((1u << 2 * NT) - 1);
        if (b > b0) copy(next, b - 1);
        products(ks, b, groups);
        if (b > b0) source.end(next, wave);
    };
    if (b0 < b1) {
        copy(even, b1 - 1);
        source.end(even, wave);
    }
    for (int b = b1 - 1; b >= b0; b -= 2) {
        block(even, odd, b);
        if (b > b0) block(odd, even, b - 1);
    }
    l = sum_xor32(l);
    if constexpr (KS > 1) {
        // the second wave of the same rows hands over m, l and O in LDS; both scale to the larger m
        __syncthreads();
        float4* ox = reinterpret_cast<float4*>(rw ? odd : even);  // [dt][e / 4][lane], then m and l
        float* ml = reinterpret_cast<float*>(ox + DT * 4 * 64);
        if (kq == 1) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    ox[(4 * dt + j) * 64 + lane] = make_float4(o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]);
            ml[lane] = m;
            ml[64 + lane] = l;
        }
        __syncthreads();
        if (kq == 1) return false;
        const float m1 = ml[lane], mn = fmaxf(m, m1);
        const float f0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        const float f1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - mn);
        m = mn;
        l = fmaf(l, f0, ml[64 + lane] * f1);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 v = ox[(4 * dt + j) * 64 + lane];
                o[dt][4 * j] = fmaf(v.x, f1, o[dt][4 * j] * f0);
                o[dt][4 * j + 1] = fmaf(v.y, f1, o[dt][4 * j + 1] * f0);
                o[dt][4 * j + 2] = fmaf(v.z, f1, o[dt][4 * j + 2] * f0);
                o[dt][4 * j + 3] = fmaf(v.w, f1, o[dt][4 * j + 3] * f0);
            }
    }
#pragma unroll
    for (int i = 0; i < DT; ++i) o_out[i] = o[i];
    m_out = m, l_out = l;
    return true;
}

}  // namespace moss
