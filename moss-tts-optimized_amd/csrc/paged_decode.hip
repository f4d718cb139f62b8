// Attention of one new token per sequence over a paged cache, split over the cache's length and joined.
//
// o_h = sum_t softmax_t(scale q_h . k_t) v_t over the rows t < length of the sequence (query head h reads KV head
// h / (QH / KH)); a sequence without rows gives zeros.  One pass with the running maximum m and sum l of each head:
// scores in the base-2 domain (scale log2(e) in one multiplication), O = sum 2^(s - m) v, rescaled when m grows.
//
// What bounds it: the cache's bytes (64 sequences of 4 to 8 thousand rows, 32 / 8 heads of 128: 261 us, 6.2 TB/s; 256 of 300 to
// 2000: 175 to 187 us, 5.2 TB/s; 16 of up to 8000, 58 MB: 16.7 us from the last-level cache, 19.5 from memory; one of 509: two
// launches and the chain of a share, 8.2 us).  Work is laid out on the device from the lengths, so that it is even whatever
// they are and a captured graph follows them: rows are counted in units of kUnit, every KV head's units of all
// sequences are shared out over about kTarget workgroups, and a workgroup takes an even share of one sequence.  A
// sequence of one share writes its output; the others write (m, l, O) per share and a second launch joins them, which
// also writes the zeros of the empty ones.
//
// A wave takes every fourth 32-row tile of its workgroup's share and reads it from the pages straight into registers
// (K of the next tile once the scores are formed, V of it once this one's is used: half the registers of two whole
// tiles, three workgroups a CU for two; 16 sequences of 17 to 8000 rows 23.5 -> 17.0 us with the join's loads together):
// K as the A operand of the 16x16x32 matrix instruction (S^T[row][head], up to 16 heads of a KV head in one tile), V
// with a full row over 16 lanes, so a lane holds 8 rows x D / 16 dims.  S^T leaves lane (g, head) with rows 4 g + i and
// 16 + 4 g + i, which is the K order that the V rows are loaded in: P goes from the softmax into the B operand of
// O^T += V^T P^T without leaving the lane, and V^T is one byte permute per register pair.  P is split into the
// sum of two 16-bit values (the second holds what rounding the first left): it costs D / 16 matrix instructions that
// the memory hides and keeps P's rounding out of the result.
#include "paged.h"

namespace moss {
namespace {

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
};

// A share's size in units (at most 65535 sequences of 2^23 units).
__device__ __forceinline__ int share_units(const PagedBatch& bt, int shift, int shares, int lane) {
    long long total = 0;
    for (int b = lane; b < bt.B; b += kWave) total += units_of(paged_length(bt, b, shift));
    return share_of_units(wave_total(total), shares);
}

// The sequence and share of a slot.  A batch of up to 64 is one load and two sums over the wave.
__device__ __forceinline__ Place find_share(const PagedBatch& bt, int shift, int shares, int slot, int lane) {
    if (bt.B <= kWave) {
        const int units = lane < bt.B ? units_of(paged_length(bt, lane, shift)) : 0;
        const int share = share_of_units(wave_total((long long)units), shares), n = shares_of(units, share);
        const int through = wave_prefix(n);
        const unsigned long long past = __ballot(through > slot);
        if (!past) return Place{-1, 0, 0};
        const int l = __builtin_ctzll(past), c = __builtin_amdgcn_readlane(n, l);
        const int first = __builtin_amdgcn_readlane(through, l) - c;
        return Place{l, slot - first, c};
    }
    const int share = share_units(bt, shift, shares, lane);
    return find_item(bt.B, slot, lane, [&](int b) { return shares_of(units_of(paged_length(bt, b, shift)), share); });
}

template <int D>
struct KvTile {  // 32 rows: lane (g, r = lane % 16)
    static constexpr int NC = D / 32, VW = D / 32;  // K chunks of 32 dims; words of a lane's D / 16 values of a V row
    u32x4_t k[2][NC];   // row 16 h + r, dims 32 c + 8 g ..
    uint32_t v[8][VW];  // row 16 (e / 4) + 4 g + e % 4, dims (D / 16) r ..
};

// K or V of one half tile: from row `row` (a multiple of 16) of page `page` (-1: of some page, unused) on.
template <bool NT, typename V>
__device__ __forceinline__ V load_row(const uint16_t* p) {
    if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
    return *reinterpret_cast<const V*>(p);
}
template <bool NT, int D>
__device__ __forceinline__ void load_k(KvTile<D>& t, int h, const PagedCache& c, int page, int kvh, int row, int g, int r) {
    const uint16_t* kr = c.k + row_offset(page, c.k_stride, kvh, row, c.shift, D);
#pragma unroll
    for (int i = 0; i < KvTile<D>::NC; ++i) t.k[h][i] = load_row<NT, u32x4_t>(kr + r * D + 32 * i + 8 * g);
}
template <bool NT, int D>
__device__ __forceinline__ void load_v(KvTile<D>& t, int h, const PagedCache& c, int page, int kvh, int row, int g, int r) {
    const uint16_t* vr = c.v + row_offset(page, c.v_stride, kvh, row, c.shift, D);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint16_t* p = vr + (4 * g + e) * D + (D / 16) * r;
        if constexpr (KvTile<D>::VW == 4) {
            const u32x4_t w = load_row<NT, u32x4_t>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) t.v[4 * h + e][i] = w[i];
        } else {
            const u32x2_v w = load_row<NT, u32x2_v>(p);
            t.v[4 * h + e][0] = w[0];
            t.v[4 * h + e][1] = w[1];
        }
    }
}

template <typename E, int D, bool NT>
__global__ __launch_bounds__(256, 3) void paged_decode_split(DecodeArgs a, PagedCache c, PagedBatch bt) {
    using T = KvTile<D>;
    constexpr int NJ = D / 16;
    __shared__ __attribute__((aligned(16))) float ow[4][16][D];
    __shared__ float mw[4][16], lw[4][16];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), w = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int g = lane >> 4, r = lane & 15;
    const int tiles = (a.group + 15) / 16;  // head tiles of a KV head
    const int slot = blockIdx.x / a.xdim, x = blockIdx.x % a.xdim;
    const int kvh = x / tiles, h0 = 16 * (x % tiles), heads = min(16, a.group - h0);
    const Place pl = find_share(bt, c.shift, a.shares, slot, lane);
    if (pl.b < 0) return;
    int r0, r1;  // may be empty
    share_rows(paged_length(bt, pl.b, c.shift), pl.count, pl.index, r0, r1);
    const int qhead = kvh * a.group + h0;

    // q as the B operand: lane (g, head r), dims 32 c + 8 g ..
    u32x4_t qf[T::NC];
    const uint16_t* qr = a.q + (size_t)pl.b * a.q_stride + (size_t)(qhead + min(r, heads - 1)) * D + 8 * g;
#pragma unroll
    for (int i = 0; i < T::NC; ++i) {
        qf[i] = *reinterpret_cast<const u32x4_t*>(qr + 32 * i);
        if (r >= heads) qf[i] = u32x4_t{0u, 0u, 0u, 0u};
    }
    f32x4_v o[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) o[j] = f32x4_v{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;  // l: this lane's rows only

    const int* trow = bt.table + (size_t)pl.b * bt.table_stride;
    const int ntile = r1 > r0 ? ((r1 - r0 + 31) / 32 - w + 3) / 4 : 0;  // this wave's tiles w, w + 4, ..
    // lane i: the page of half tile i of 32 tiles; those of the next 32 replace them when tile 32 k is loaded
    auto row_of = [&](int i, int h) { return r0 + 32 * (w + 4 * i) + 16 * h; };
    int pages = -1;
    auto fetch_pages = [&](int first) {
        const int row = row_of(first + lane / 2, lane & 1);
        int p = -1;
        if (row < r1) p = page_or_none(trow[row >> c.shift], c.pages);
        pages = p;
    };
    // K of tile i + 1 is loaded as soon as the scores of tile i are formed, V of it once tile i's is consumed: one set
    // of registers for each, and loads on their way all the time
    KvTile<D> t;
    int p0 = -1, p1 = -1;  // the pages of the tile whose K was loaded last
    auto next_k = [&](int i) {
        if ((i & 31) == 0) fetch_pages(i);
        p0 = __builtin_amdgcn_readlane(pages, 2 * (i & 31));
        p1 = __builtin_amdgcn_readlane(pages, 2 * (i & 31) + 1);
        load_k<NT, D>(t, 0, c, p0, kvh, row_of(i, 0), g, r);
        load_k<NT, D>(t, 1, c, p1, kvh, row_of(i, 1), g, r);
    };
    auto next_v = [&](int i) {
        load_v<NT, D>(t, 0, c, p0, kvh, row_of(i, 0), g, r);
        load_v<NT, D>(t, 1, c, p1, kvh, row_of(i, 1), g, r);
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
            for (int k = 0; k < T::NC; ++k) s[h] = E::mfma16(t.k[h][k], qf[k], s[h]);
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
#pragma unroll
                for (int k = 0; k < T::VW; ++k) t.v[e][k] = live ? t.v[e][k] : 0u;
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
#pragma unroll
        for (int jw = 0; jw < T::VW; ++jw) {
            u32x4_t even, odd;  // V^T rows (D / 16) r + 2 jw and + 1, the lane's 8 rows as K
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                even[k] = __builtin_amdgcn_perm(t.v[2 * k + 1][jw], t.v[2 * k][jw], 0x05040100u);
                odd[k] = __builtin_amdgcn_perm(t.v[2 * k + 1][jw], t.v[2 * k][jw], 0x07060302u);
            }
            o[2 * jw] = E::mfma16(even, ph, o[2 * jw]);
            o[2 * jw + 1] = E::mfma16(odd, ph, o[2 * jw + 1]);
            o[2 * jw] = E::mfma16(even, plo, o[2 * jw]);
            o[2 * jw + 1] = E::mfma16(odd, plo, o[2 * jw + 1]);
        }
        if (i + 1 < ntile) next_v(i + 1);
    }

    // the waves' parts, each against its own m, meet in LDS
    l = sum_xor32(sum_xor16(l));
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
        if (pl.count == 1) {
            const float inv = den == 0.f ? 0.f : 1.0f / den;  // every row without a page: zeros
            *reinterpret_cast<uint32_t*>(a.out + ((size_t)pl.b * a.qh + qhead + h) * D + d) = E::pack(x * inv, y * inv);
        } else {
            const size_t at = (size_t)slot * a.qh + qhead + h;
            *reinterpret_cast<float2*>(a.part + at * D + d) = make_float2(x, y);
            if (d == 0) a.stat[at] = make_float2(mx, den);
        }
    }
}

// grid (QH, B), 256 threads: the shares of one head of a sequence, wave w taking w, w + 4, ..; the four waves' sums meet
// in LDS.
template <typename E, int D>
__global__ __launch_bounds__(256) void paged_decode_join(DecodeArgs a, PagedCache c, PagedBatch bt) {
    constexpr int VPL = D / kWave;
    __shared__ float acc_s[4][D];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & (kWave - 1), w = tid / kWave;
    const int su = share_units(bt, c.shift, a.shares, lane);
    const int count = shares_of(units_of(paged_length(bt, b, c.shift)), su);
    if (count == 1) return;  // written by its workgroup
    uint16_t* dst = a.out + ((size_t)b * a.qh + h) * D;
    if (count == 0) {
        for (int d = tid; d < D; d += 256) dst[d] = 0;
        return;
    }
    int first = 0;
    for (int s = lane; s < b; s += kWave) first += shares_of(units_of(paged_length(bt, s, c.shift)), su);
    first = wave_total(first);
    if (!in_slots(first, count, a.slots)) return;  // only when the lengths change between the launches
    // m and l of share 64 i + lane; a share's weight is 2^(m - largest m)
    const float2* st = a.stat + (size_t)first * a.qh + h;
    const float2 own = lane < count ? st[(size_t)lane * a.qh] : make_float2(-INFINITY, 0.f);
    const float* part = a.part + ((size_t)first * a.qh + h) * D + VPL * lane;
    const size_t step = (size_t)a.qh * D;
    float mx = own.x;
    for (int s = kWave + lane; s < count; s += kWave) mx = fmaxf(mx, st[(size_t)s * a.qh].x);
    mx = wave_max(mx);
    auto weight = [&](float m) { return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mx); };
    const float f0 = weight(own.x);
    float den = f0 * own.y;
    for (int s = kWave + lane; s < count; s += kWave) {
        const float2 v = st[(size_t)s * a.qh];
        den += weight(v.x) * v.y;
    }
    den = wave_sum(den);
    float acc[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) acc[i] = 0.f;
    constexpr int N = 8;  // parts on their way together: shares w, w + 4, ..
    for (int s0 = w; s0 < count; s0 += 4 * N) {
        float x[N][VPL], f[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int s = min(s0 + 4 * n, count - 1);
#pragma unroll
            for (int i = 0; i < VPL; ++i) x[n][i] = part[s * step + i];
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int s = min(s0 + 4 * n, count - 1);
            f[n] = s < kWave ? __uint_as_float(lane_value(__float_as_uint(f0), s)) : weight(st[(size_t)s * a.qh].x);
            if (s0 + 4 * n >= count) f[n] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < VPL; ++i) acc[i] = f[n] == 0.f ? acc[i] : fmaf(f[n], x[n][i], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) acc_s[w][VPL * lane + i] = acc[i];
    __syncthreads();
    if (tid < D / 2) {
        const float inv = den == 0.f ? 0.f : 1.0f / den;
        float x = 0.f, y = 0.f;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            x += acc_s[v][2 * tid];
            y += acc_s[v][2 * tid + 1];
        }
        reinterpret_cast<uint32_t*>(dst)[tid] = E::pack(x * inv, y * inv);
    }
}

struct DecodePlan {
    int xdim, shares;
    long long slots;
};

DecodePlan decode_plan(int B, int W, int shift, int qh, int kh) {
    DecodePlan p;
    p.xdim = kh * ((qh / kh + 15) / 16);
    p.shares = kTarget / p.xdim > 1 ? kTarget / p.xdim : 1;
    p.slots = decode_slots(B, W, shift, p.shares);
    return p;
}

template <typename E, int D>
void launch_decode(const DecodeArgs& a, const PagedCache& c, const PagedBatch& bt, const DecodePlan& p, hipStream_t st) {
    const long long page = ((long long)c.kh << c.shift) * D * 2, named = (long long)bt.B * bt.W;
    const dim3 grid((unsigned)(p.xdim * p.slots));
    if ((named < c.pages ? named : c.pages) * page * 2 > kCached)
        hipLaunchKernelGGL((paged_decode_split<E, D, true>), grid, dim3(256), 0, st, a, c, bt);
    else
        hipLaunchKernelGGL((paged_decode_split<E, D, false>), grid, dim3(256), 0, st, a, c, bt);
    hipLaunchKernelGGL((paged_decode_join<E, D>), dim3((unsigned)a.qh, (unsigned)bt.B), dim3(256), 0, st, a, c, bt);
}

}  // namespace
}  // namespace moss

using namespace moss;

MOSS_API long long moss_paged_decode_workspace_bytes(int B, int W, int page_rows, int qh, int kh, int d) {
    const int shift = page_shift(page_rows);
    if (B <= 0 || W <= 0 || shift < 0 || ((long long)W << shift) > (1ll << 30) || kh <= 0 || qh <= 0 || qh % kh ||
        (d != 64 && d != 128))
        return 0;
    return decode_plan(B, W, shift, qh, kh).slots * qh * (d + 2) * 4;
}

MOSS_API int moss_paged_decode_attention(const void* q, long long q_stride, const void* k, const void* v,
                                         long long k_stride, long long v_stride, int pages, int page_rows,
                                         const void* table, long long table_stride, const void* lengths, int B, int W,
                                         int qh, int kh, int d, float scale, void* out, void* workspace,
                                         long long workspace_bytes, int dtype, void* stream) {
    const PagedCache c = paged_cache(k, v, k_stride, v_stride, pages, kh, page_rows);
    const PagedBatch bt{(const int*)table, (const int*)lengths, nullptr, B, W, table_stride};
    MOSS_CHECK_ARG(q && out && workspace && paged_pointers_ok(c, bt) && paged_shape_ok(c, bt, qh, d));
    MOSS_CHECK_ARG((dtype == 0 || dtype == 1) && q_stride % 8 == 0 && q_stride >= (long long)qh * d && scale == scale);
    MOSS_CHECK_ARG(MOSS_ALIGNED(q, 16) && MOSS_ALIGNED(out, 16) && MOSS_ALIGNED(workspace, 16));
    const DecodePlan p = decode_plan(B, W, c.shift, qh, kh);
    MOSS_CHECK_ARG(workspace_bytes >= p.slots * qh * (d + 2) * 4 && p.slots * p.xdim * 256 < (1ll << 32));
    DecodeArgs a{(const uint16_t*)q, q_stride, (uint16_t*)out, (float*)workspace,
                 reinterpret_cast<float2*>((float*)workspace + p.slots * qh * d), qh, qh / kh, p.xdim, p.shares, p.slots,
                 scale * 1.4426950408889634f};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0)
        d == 128 ? launch_decode<Bf16, 128>(a, c, bt, p, st) : launch_decode<Bf16, 64>(a, c, bt, p, st);
    else
        d == 128 ? launch_decode<F16, 128>(a, c, bt, p, st) : launch_decode<F16, 64>(a, c, bt, p, st);
    return moss_launch_status();
}
