// The work of one workgroup of a decode attention over a paged cache: one query token's heads of a KV head over some rows of its
// sequence, with the running maximum m and sum l of each head, from a cache in 16 or 8 bits.
//
// A wave takes every fourth 32-row tile of the rows and reads it from the pages straight into registers
// (K of the next tile once the scores are formed, V of it once this one's is used: half the registers of two whole
// tiles, three workgroups a CU for two; 16 sequences of 17 to 8000 rows 23.5 -> 17.0 us with the join's loads together):
// K as the A operand of the 16x16x32 matrix instruction (S^T[row][head], up to 16 heads of a KV head in one tile), V
// with a full row over 16 lanes, so a lane holds 8 rows x D / 16 dims.  S^T leaves lane (g, head) with rows 4 g + i and
// 16 + 4 g + i, which is the K order that the V rows are loaded in: P goes from the softmax into the B operand of
// O^T += V^T P^T without leaving the lane, and V^T is one byte permute per register pair.  P is split into the
// sum of two 16-bit values (the second holds what rounding the first left): it costs D / 16 matrix instructions that
// the memory hides and keeps P's rounding out of the result.
//
// In 8 bits the tile's registers hold the codes, and the conversion to the 16-bit type, which takes the row's scale as
// an operand, stands between them and the matrix instructions: half the bytes and nothing else to do for a scale.
#pragma once

#include "paged8.h"

namespace moss {

// Workgroups that the work is shared out over.  512 / 1024 / 1536 / 2048: 273 / 265 / 261 / 263 us for 64 sequences of 4 to 8
// thousand rows of 8 heads, 25.9 / 24.3 / 24.1 / 24.1 for 48 of up to 2000 rows of 12 heads of 64 (six caches in turn), 109 / 99 /
// 97 / 98 for 128 of 300 to 2000 rows, no difference for 16 sequences.
constexpr int kTarget = 1536;
// Pages of more than the last-level cache (256 MB) are read past it.  The pages that the call can name decide, since the host
// does not know the lengths: with a server's pool that is nearly every call, of few rows too, and right for it, as what one
// layer's call reads is gone by the time of the next step's.  To / past the cache: 287 / 261 us for those 64 sequences (1.6 GB),
// 103 / 96 for 128 and 192 / 183 for 256 of 300 to 2000 rows; 16 sequences with 58 MB, 36 layers' caches in turn, 19.8 / 19.3, one
// of 509 rows 9.0 / 8.8; but one cache read again and again, which stays: 16.7 / 17.5, four such 17.0 / 18.6.
constexpr long long kCached = 256ll << 20;

struct DecodeArgs {
    const uint16_t* q;
    long long q_stride;
    uint16_t* out;
    float* part;   // [slots, QH, D]: O of each share
    float2* stat;  // [slots, QH]: its m and l
    int qh, group, xdim, shares;  // xdim: head tiles; shares: workgroups per head tile that the units are shared out over
    long long slots;
    float scale;            // scale log2(e)
    uint32_t flip;          // its sign where `scale` is without one, for the two values of a word of q
};

// K or V of a row: 16 bytes or 8, past the last-level cache (NT) or through it.
template <bool NT, typename V>
__device__ __forceinline__ V load_row(const void* p) {
    if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
    return *reinterpret_cast<const V*>(p);
}

// 32 rows of a cache, lane (g, r = lane % 16), half tile h the rows 16 h .. + 15, which lie in one page (-1: of some page,
// unused).  key(h, i): dims q_dim(i, g) .. + 7 of row 16 h + r.  pair(j): of V, dims (D / 16) r + 2 j and + 1, the lane's 8
// rows (16 (e / 4) + 4 g + e % 4) as K.
template <typename E, int D>
struct Tile16 {
    using Cache = PagedCache;
    static constexpr int NC = D / 32, VW = D / 32;  // K chunks of 32 dims; words of a lane's D / 16 values of a V row
    u32x4_t k[2][NC];
    uint32_t v[8][VW];
    static __device__ __forceinline__ int q_dim(int i, int g) { return 32 * i + 8 * g; }
    template <bool NT>
    __device__ __forceinline__ void load_k(int h, const Cache& c, int page, int kvh, int row, int g, int r) {
        const uint16_t* kr = c.k + row_offset(page, c.k_stride, kvh, row, c.shift, D);
#pragma unroll
        for (int i = 0; i < NC; ++i) k[h][i] = load_row<NT, u32x4_t>(kr + r * D + 32 * i + 8 * g);
    }
    template <bool NT>
    __device__ __forceinline__ void load_v(int h, const Cache& c, int page, int kvh, int row, int g, int r) {
        const uint16_t* vr = c.v + row_offset(page, c.v_stride, kvh, row, c.shift, D);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint16_t* p = vr + (4 * g + e) * D + (D / 16) * r;
            if constexpr (VW == 4) {
                const u32x4_t w = load_row<NT, u32x4_t>(p);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * h + e][i] = w[i];
            } else {
                const u32x2_v w = load_row<NT, u32x2_v>(p);
                v[4 * h + e][0] = w[0];
                v[4 * h + e][1] = w[1];
            }
        }
    }
    __device__ __forceinline__ u32x4_t key(int h, int i) const { return k[h][i]; }
    __device__ __forceinline__ void drop(int e, bool live) {  // V of a row without a part, which may hold anything
#pragma unroll
        for (int i = 0; i < VW; ++i) v[e][i] = live ? v[e][i] : 0u;
    }
    template <int J>
    __device__ __forceinline__ uint32_t value(int e) const { return v[e][J]; }
};

template <typename E, int D>
struct Tile8 {
    using Cache = PagedCache8;
    static constexpr int NC = D / 32, VW = D / 32, NL = D / 64;  // NL: 16-byte loads of a lane's codes of a K row
    u32x4_t k[2][NL];      // row 16 h + r, dims 64 i + 16 g ..: two chunks
    uint32_t v[8][NL];     // dims (D / 16) r ..
    uint32_t ks[2], vs[2];  // the scale bytes of row 16 h + r, of rows 16 h + 4 g ..
    static __device__ __forceinline__ int q_dim(int i, int g) { return 64 * (i >> 1) + 16 * g + 8 * (i & 1); }
    template <bool NT>
    __device__ __forceinline__ void load_k(int h, const Cache& c, int page, int kvh, int row, int g, int r) {
        const uint8_t* kr = c.kc() + row_offset(page, c.k_stride, kvh, row, c.shift, D);
#pragma unroll
        for (int i = 0; i < NL; ++i) k[h][i] = load_row<NT, u32x4_t>(kr + r * D + 64 * i + 16 * g);
        ks[h] = c.ks[row_offset(page, c.ks_stride, kvh, row, c.shift, 1) + r];
    }
    template <bool NT>
    __device__ __forceinline__ void load_v(int h, const Cache& c, int page, int kvh, int row, int g, int r) {
        const uint8_t* vr = c.vc() + row_offset(page, c.v_stride, kvh, row, c.shift, D);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint8_t* p = vr + (4 * g + e) * D + (D / 16) * r;
            if constexpr (NL == 2) {
                const u32x2_v w = load_row<NT, u32x2_v>(p);
                v[4 * h + e][0] = w[0];
                v[4 * h + e][1] = w[1];
            } else {
                v[4 * h + e][0] = load_row<NT, uint32_t>(p);
            }
        }
        vs[h] = *reinterpret_cast<const uint32_t*>(c.vs + row_offset(page, c.vs_stride, kvh, row, c.shift, 1) + 4 * g);
    }
    __device__ __forceinline__ u32x4_t key(int h, int i) const {
        return widen8<E>(k[h][i >> 1][2 * (i & 1)], k[h][i >> 1][2 * (i & 1) + 1], scale_of(ks[h]));
    }
    __device__ __forceinline__ void drop(int e, bool live) {
        const uint32_t at = 0xffu << (8 * (e & 3));  // a scale of any byte times 0 is not 0: of 1
#pragma unroll
        for (int i = 0; i < NL; ++i) v[e][i] = live ? v[e][i] : 0u;
        vs[e >> 2] = live ? vs[e >> 2] : (vs[e >> 2] & ~at) | (0x7f7f7f7fu & at);
    }
    template <int J>
    __device__ __forceinline__ uint32_t value(int e) const {
        const uint32_t byte = (vs[e >> 2] >> (8 * (e & 3))) & 0xffu;
        return widen<E, (J & 1) != 0>(v[e][J >> 1], scale_of(byte));
    }
};

template <int N>
struct Int {
    static constexpr int value = N;
};

// Where a workgroup's result goes: the output itself (its rows are all there is), or (m, l, O) in slot `slot`.
struct ShareOf {
    int b, kvh, h0, heads;  // sequence, KV head, the first of the heads (within the KV head's) and how many, up to 16
    int r0, r1;             // rows (may be empty); r0 a multiple of 16
    bool alone;
    long long slot;
};

// WAVES: 4, a workgroup's, or 1, each by itself and without LDS.  ow, mw, lw: LDS for the waves' parts (16-byte aligned).
template <typename E, int D, typename T, bool NT, int WAVES>
__device__ __forceinline__ void decode_share(const DecodeArgs& a, const typename T::Cache& c, const PagedBatch& bt,
                                             const ShareOf& sh, int tid, float (&ow)[4][16][D], float (&mw)[4][16], float (&lw)[4][16]) {
    constexpr int NJ = D / 16;
    const int lane = tid & (kWave - 1), w = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int g = lane >> 4, r = lane & 15;
    const int kvh = sh.kvh, h0 = sh.h0, heads = sh.heads, r0 = sh.r0, r1 = sh.r1;
    const int qhead = kvh * a.group + h0;

    // q as the B operand: lane (g, head r)
    u32x4_t qf[T::NC];
    const uint16_t* qr = a.q + (size_t)sh.b * a.q_stride + (size_t)(qhead + min(r, heads - 1)) * D;
#pragma unroll
    for (int i = 0; i < T::NC; ++i) {
        qf[i] = *reinterpret_cast<const u32x4_t*>(qr + T::q_dim(i, g));
        qf[i] = r < heads ? qf[i] ^ a.flip : u32x4_t{0u, 0u, 0u, 0u};
    }
    f32x4_v o[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j] = f32x4_v{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;  // l: this lane's rows only

    const int* trow = bt.table + (size_t)sh.b * bt.table_stride;
    const int w0 = WAVES == 1 ? 0 : w;
    const int ntile = r1 > r0 ? ((r1 - r0 + 31) / 32 - w0 + WAVES - 1) / WAVES : 0;  // this wave's tiles w0, w0 + WAVES, ..
    // lane i: the page of half tile i of 32 tiles; those of the next 32 replace them when tile 32 k is loaded
    auto row_of = [&](int i, int h) { return r0 + 32 * (w0 + WAVES * i) + 16 * h; };
    int pages = -1;
    auto fetch_pages = [&](int first) {
        const int row = row_of(first + lane / 2, lane & 1);
        int p = -1;
        if (row < r1) p = page_or_none(trow[row >> c.shift], c.pages);
        pages = p;
    };
    // K of tile i + 1 is loaded as soon as the scores of tile i are formed, V of it once tile i's is consumed: one set
    // of registers for each, and loads on their way all the time
    T t;
    int p0 = -1, p1 = -1;  // the pages of the tile whose K was loaded last
    auto next_k = [&](int i) {
        if ((i & 31) == 0) fetch_pages(i);
        p0 = __builtin_amdgcn_readlane(pages, 2 * (i & 31));
        p1 = __builtin_amdgcn_readlane(pages, 2 * (i & 31) + 1);
        t.template load_k<NT>(0, c, p0, kvh, row_of(i, 0), g, r);
        t.template load_k<NT>(1, c, p1, kvh, row_of(i, 1), g, r);
    };
    auto next_v = [&](int i) {
        t.template load_v<NT>(0, c, p0, kvh, row_of(i, 0), g, r);
        t.template load_v<NT>(1, c, p1, kvh, row_of(i, 1), g, r);
    };
    if (ntile > 0) {
        next_k(0);
        next_v(0);
    }
    for (int i = 0; i < ntile; ++i) {
        // rows of the halves that take part: 16, fewer at the end, none without a page
        const int n0 = p0 < 0 ? 0 : min(16, max(0, r1 - row_of(i, 0))), n1 = p1 < 0 ? 0 : min(16, max(0, r1 - row_of(i, 1)));
        f32x4_v s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s[h] = f32x4_v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < T::NC; ++k) s[h] = E::mfma16(t.key(h, k), qf[k], s[h]);
        }
        if (i + 1 < ntile) next_k(i + 1);
        float sv[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) sv[e] = s[e >> 2][e & 3] * a.scale;
        if (n0 + n1 < 32) {  // uniform: rows without a part, whose K and V may hold anything
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool live = 4 * g + (e & 3) < (e < 4 ? n0 : n1);
                sv[e] = live ? sv[e] : -INFINITY;
                t.drop(e, live);
            }
        }
        float mx = sv[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) mx = fmaxf(mx, sv[e]);
        mx = max_xor32(max_xor16(mx));
        if (__any(mx > m)) {
            const float mn = fmaxf(m, mx);
            const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[j][k] *= f;
        }
        const float mr = m == -INFINITY ? 0.f : m;
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            p[e] = __builtin_amdgcn_exp2f(sv[e] - mr);
            l += p[e];
        }
        u32x4_t ph, plo;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            ph[k] = E::pack(p[2 * k], p[2 * k + 1]);
            plo[k] = E::pack(p[2 * k] - E::lo(ph[k]), p[2 * k + 1] - E::hi(ph[k]));
        }
        // V^T rows (D / 16) r + 2 J and + 1
        auto multiply = [&](auto j) {
            constexpr int J = decltype(j)::value;
            u32x4_t even, odd;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t v0 = t.template value<J>(2 * k), v1 = t.template value<J>(2 * k + 1);
                even[k] = __builtin_amdgcn_perm(v1, v0, 0x05040100u);
                odd[k] = __builtin_amdgcn_perm(v1, v0, 0x07060302u);
            }
            o[2 * J] = E::mfma16(even, ph, o[2 * J]);
            o[2 * J + 1] = E::mfma16(odd, ph, o[2 * J + 1]);
            o[2 * J] = E::mfma16(even, plo, o[2 * J]);
            o[2 * J + 1] = E::mfma16(odd, plo, o[2 * J + 1]);
        };
        multiply(Int<0>{});
        multiply(Int<1>{});
        if constexpr (T::VW == 4) {
            multiply(Int<2>{});
            multiply(Int<3>{});
        }
        if (i + 1 < ntile) next_v(i + 1);
    }

    l = sum_xor32(sum_xor16(l));
    if constexpr (WAVES == 1) {
        if (r >= heads) return;
        const float inv = sh.alone ? (l == 0.f ? 0.f : 1.0f / l) : 1.f;
        const size_t at = (sh.alone ? (size_t)sh.b : (size_t)sh.slot) * a.qh + qhead + r;
#pragma unroll
        for (int i = 0; i < 4; ++i)  // dims (D / 16) (4 g + i) + j
#pragma unroll
            for (int j = 0; j < NJ; j += 4) {
                const int d = NJ * (4 * g + i) + j;
                if (sh.alone)
                    *reinterpret_cast<uint2*>(a.out + at * D + d) =
                        make_uint2(E::pack(o[j][i] * inv, o[j + 1][i] * inv), E::pack(o[j + 2][i] * inv, o[j + 3][i] * inv));
                else
                    *reinterpret_cast<float4*>(a.part + at * D + d) = make_float4(o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]);
            }
        if (!sh.alone && g == 0) a.stat[at] = make_float2(m, l);
        return;
    }
    // the waves' parts, each against its own m, meet in LDS
    if (g == 0) {
        mw[w][r] = m;
        lw[w][r] = l;
    }
    if (r < heads) {
#pragma unroll
        for (int i = 0; i < 4; ++i)  // lane (g, head r): dims (D / 16) (4 g + i) + j
#pragma unroll
            for (int j = 0; j < NJ; j += 4)
                *reinterpret_cast<float4*>(&ow[w][r][NJ * (4 * g + i) + j]) =
                    make_float4(o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]);
    }
    __syncthreads();
    for (int e = tid; e < heads * (D / 2); e += 256) {
        const int h = e / (D / 2), d = 2 * (e % (D / 2));
        float mx = -INFINITY, den = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int v = 0; v < 4; ++v) mx = fmaxf(mx, mw[v][h]);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const float f = mw[v][h] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw[v][h] - mx);
            const float2 ov = *reinterpret_cast<const float2*>(&ow[v][h][d]);
            den = fmaf(f, lw[v][h], den);
            x = fmaf(f, ov.x, x);
            y = fmaf(f, ov.y, y);
        }
        if (sh.alone) {
            const float inv = den == 0.f ? 0.f : 1.0f / den;  // every row without a page: zeros
            *reinterpret_cast<uint32_t*>(a.out + ((size_t)sh.b * a.qh + qhead + h) * D + d) = E::pack(x * inv, y * inv);
        } else {
            const size_t at = (size_t)sh.slot * a.qh + qhead + h;
            *reinterpret_cast<float2*>(a.part + at * D + d) = make_float2(x, y);
            if (d == 0) a.stat[at] = make_float2(mx, den);
        }
    }
}

}  // namespace moss
