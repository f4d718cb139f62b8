// Attention of one new token per sequence over a paged cache, split over the cache's length and joined.
//
// o_h = sum_t softmax_t(scale q_h . k_t) v_t over the rows t < length of the sequence (query head h reads KV head
// h / (QH / KH)); a sequence without rows gives zeros.  One pass with the running maximum m and sum l of each head:
// scores in the base-2 domain (scale log2(e) in one multiplication), O = sum 2^(s - m) v, rescaled when m grows.
//
// What bounds it: the cache's bytes.  Work is laid out on the device from the lengths, so that it is even whatever
// they are and a captured graph follows them: rows are counted in units of kUnit, every KV head's units of all
// sequences are shared out over about kTarget workgroups, and a workgroup takes an even share of one sequence.  A
// sequence of one share writes its output; the others write (m, l, O) per share and a second launch joins them, which
// also writes the zeros of the empty ones.
//
// A wave takes every fourth 32-row tile of its workgroup's share and reads it from the pages straight into registers:
// K as the A operand of the 16x16x32 matrix instruction (S^T[row][head], up to 16 heads of a KV head in one tile), V
// with a full row over 16 lanes, so a lane holds 8 rows x D / 16 dims.  S^T leaves lane (g, head) with rows 4 g + i and
// 16 + 4 g + i, which is the K order that the V rows are loaded in: P goes from the softmax into the B operand of
// O^T += V^T P^T without leaving the lane, and V^T is one byte permute per register pair.  P is split into the
// sum of two 16-bit values (the second holds what rounding the first left): it costs D / 16 matrix instructions that
// the memory hides and keeps P's rounding out of the result.
#include "paged.h"

namespace moss {
namespace {

constexpr int kTarget = 2048;  // workgroups that the work is shared out over

struct DecodeArgs {
    const uint16_t* q;
    long long q_stride;
    uint16_t* out;
    float* part;   // [slots, QH, D]: O of each share
    float2* stat;  // [slots, QH]: its m and l
    int qh, group, xdim, shares;  // xdim: head tiles; shares: workgroups per head tile that the units are shared out over
    float scale;            // scale log2(e)
};

// A share's size in units (at most 65535 sequences of 2^23 units).
__device__ __forceinline__ int share_units(const PagedBatch& bt, int shift, int shares, int lane) {
    long long total = 0;
    for (int b = lane; b < bt.B; b += kWave) total += units_of(paged_length(bt, b, shift));
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) total += __shfl_xor(total, m);
    return __builtin_amdgcn_readfirstlane(share_of_units(total, shares));
}

template <int D>
struct KvTile {  // 32 rows: lane (g, r = lane % 16)
    static constexpr int NC = D / 32, VW = D / 32;  // K chunks of 32 dims; words of a lane's D / 16 values of a V row
    u32x4_t k[2][NC];    // row 16 h + r, dims 32 c + 8 g ..
    uint32_t v[8][VW];   // row 16 (e / 4) + 4 g + e % 4, dims (D / 16) r ..
};

// One half tile's rows: from row `row` (a multiple of 16) of page `page` (-1: of some page, unused).
template <int D>
__device__ __forceinline__ void load_half(KvTile<D>& t, int h, const PagedCache& c, int page, int kvh, int row, int g, int r) {
    using T = KvTile<D>;
    const uint16_t* kr = c.k + row_offset(page, c.k_stride, kvh, row, c.shift, D);
    const uint16_t* vr = c.v + row_offset(page, c.v_stride, kvh, row, c.shift, D);
#pragma unroll
    for (int i = 0; i < T::NC; ++i) t.k[h][i] = *reinterpret_cast<const u32x4_t*>(kr + (size_t)r * D + 32 * i + 8 * g);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint16_t* p = vr + (size_t)(4 * g + e) * D + (D / 16) * r;
        if constexpr (T::VW == 4) {
            const u32x4_t w = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) t.v[4 * h + e][i] = w[i];
        } else {
            const u32x2_v w = *reinterpret_cast<const u32x2_v*>(p);
            t.v[4 * h + e][0] = w[0];
            t.v[4 * h + e][1] = w[1];
        }
    }
}

template <typename E, int D>
__global__ __launch_bounds__(256, 2) void paged_decode_split(DecodeArgs a, PagedCache c, PagedBatch bt) {
    using T = KvTile<D>;
    constexpr int NJ = D / 16;
    __shared__ __attribute__((aligned(16))) float ow[4][16][D];
    __shared__ float mw[4][16], lw[4][16];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), w = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int g = lane >> 4, r = lane & 15;
    const int tiles = (a.group + 15) / 16;  // head tiles of a KV head
    const int slot = blockIdx.x / a.xdim, x = blockIdx.x % a.xdim;
    const int kvh = x / tiles, h0 = 16 * (x % tiles), heads = min(16, a.group - h0);
    const int su = share_units(bt, c.shift, a.shares, lane);
    const Place pl = find_item(bt.B, slot, lane, [&](int b) { return shares_of(units_of(paged_length(bt, b, c.shift)), su); });
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
    int pages = -1;  // lane i: the page of half tile i of the 32 tiles from `fetched` on
    auto fetch_pages = [&](int first) {
        const int row = r0 + 32 * (w + 4 * (first + lane / 2)) + 16 * (lane & 1);
        int p = -1;
        if (row < r1) p = page_or_none(trow[row >> c.shift], c.pages);
        pages = p;
    };
    auto load = [&](KvTile<D>& t, int i) {
        if ((i & 31) == 0) fetch_pages(i);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = r0 + 32 * (w + 4 * i) + 16 * h;
            const int page = __builtin_amdgcn_readlane(pages, 2 * (i & 31) + h);
            load_half<D>(t, h, c, page, kvh, row, g, r);
        }
    };
    // rows of half tile h of tile i that take part: 16, fewer at the end, none without a page
    auto rows_of = [&](int i, int h, int page) { return page < 0 ? 0 : min(16, max(0, r1 - (r0 + 32 * (w + 4 * i) + 16 * h))); };
    auto compute = [&](KvTile<D>& t, int n0, int n1) {
        f32x4_v s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s[h] = f32x4_v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < T::NC; ++i) s[h] = E::mfma16(t.k[h][i], qf[i], s[h]);
        }
        float sv[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) sv[e] = s[e >> 2][e & 3] * a.scale;
        if (n0 + n1 < 32) {  // uniform: rows without a part, whose K and V may hold anything
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool live = 4 * g + (e & 3) < (e < 4 ? n0 : n1);
                sv[e] = live ? sv[e] : -INFINITY;
#pragma unroll
                for (int i = 0; i < T::VW; ++i) t.v[e][i] = live ? t.v[e][i] : 0u;
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
                for (int i = 0; i < 4; ++i) o[j][i] *= f;
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
        for (int i = 0; i < 4; ++i) {
            ph[i] = E::pack(p[2 * i], p[2 * i + 1]);
            plo[i] = E::pack(p[2 * i] - E::lo(ph[i]), p[2 * i + 1] - E::hi(ph[i]));
        }
#pragma unroll
        for (int jw = 0; jw < T::VW; ++jw) {
            u32x4_t even, odd;  // V^T rows (D / 16) r + 2 jw and + 1, the lane's 8 rows as K
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                even[i] = __builtin_amdgcn_perm(t.v[2 * i + 1][jw], t.v[2 * i][jw], 0x05040100u);
                odd[i] = __builtin_amdgcn_perm(t.v[2 * i + 1][jw], t.v[2 * i][jw], 0x07060302u);
            }
            o[2 * jw] = E::mfma16(even, ph, o[2 * jw]);
            o[2 * jw + 1] = E::mfma16(odd, ph, o[2 * jw + 1]);
            o[2 * jw] = E::mfma16(even, plo, o[2 * jw]);
            o[2 * jw + 1] = E::mfma16(odd, plo, o[2 * jw + 1]);
        }
    };
    // tile i + 1 is on its way while tile i is consumed
    KvTile<D> ta, tb;
    int na0 = 0, na1 = 0, nb0 = 0, nb1 = 0;
    auto load_counted = [&](KvTile<D>& t, int i, int& n0, int& n1) {
        load(t, i);
        n0 = rows_of(i, 0, __builtin_amdgcn_readlane(pages, 2 * (i & 31)));
        n1 = rows_of(i, 1, __builtin_amdgcn_readlane(pages, 2 * (i & 31) + 1));
    };
    if (ntile > 0) load_counted(ta, 0, na0, na1);
    for (int i = 0; i < ntile; i += 2) {
        if (i + 1 < ntile) load_counted(tb, i + 1, nb0, nb1);
        compute(ta, na0, na1);
        if (i + 1 < ntile) {
            if (i + 2 < ntile) load_counted(ta, i + 2, na0, na1);
            compute(tb, nb0, nb1);
        }
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
#pragma unroll
    for (int k = 1; k < kWave; k <<= 1) first += __shfl_xor(first, k);
    const float2* st = a.stat + (size_t)first * a.qh + h;
    float mx = -INFINITY;
    for (int s = lane; s < count; s += kWave) mx = fmaxf(mx, st[(size_t)s * a.qh].x);
    mx = wave_max(mx);
    float den = 0.f;
    for (int s = lane; s < count; s += kWave) {
        const float2 v = st[(size_t)s * a.qh];
        den += v.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v.x - mx) * v.y;
    }
    den = wave_sum(den);
    float acc[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) acc[i] = 0.f;
    for (int s = w; s < count; s += 4) {
        const size_t at = (size_t)(first + s) * a.qh + h;
        const float ms = a.stat[at].x;
        const float f = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - mx);
#pragma unroll
        for (int i = 0; i < VPL; ++i) acc[i] = fmaf(f, a.part[at * D + VPL * lane + i], acc[i]);
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
    hipLaunchKernelGGL((paged_decode_split<E, D>), dim3((unsigned)(p.xdim * p.slots)), dim3(256), 0, st, a, c, bt);
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
                 reinterpret_cast<float2*>((float*)workspace + p.slots * qh * d), qh, qh / kh, p.xdim, p.shares,
                 scale * 1.4426950408889634f};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0)
        d == 128 ? launch_decode<Bf16, 128>(a, c, bt, p, st) : launch_decode<Bf16, 64>(a, c, bt, p, st);
    else
        d == 128 ? launch_decode<F16, 128>(a, c, bt, p, st) : launch_decode<F16, 64>(a, c, bt, p, st);
    return moss_launch_status();
}
