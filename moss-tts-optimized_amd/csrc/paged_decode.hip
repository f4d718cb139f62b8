// Attention of one new token per sequence over a paged cache, split over the cache's length and joined.
//
// o_h = sum_t softmax_t(scale q_h . k_t) v_t over the rows t < length of the sequence (query head h reads KV head
// h / (QH / KH)); a sequence without rows gives zeros.  One pass with the running maximum m and sum l of each head:
// scores in the base-2 domain (scale log2(e) in one multiplication), O = sum 2^(s - m) v, rescaled when m grows.
//
// What bounds it: the cache's bytes (64 sequences of 4 to 8 thousand rows, 32 / 8 heads of 128: 261 us, 6.2 TB/s; 256 of 300 to
// 2000: 175 to 187 us, 5.2 TB/s; 16 of up to 8000, 58 MB: 16.7 us from the last-level cache, 19.5 from memory; one of 509: two
// launches and the chain of a share, 8.2 us).  From 8 bits the same: 64 sequences 147 us, 5.5 TB/s, 16 of up to 3128 15, one of
// 509 8.8; the conversions (27.3 million vector instructions for 19.5 without them) hide behind the loads, and a fourth
// workgroup a CU, which spills eight registers, takes 195.
//
// Work is laid out on the device from the lengths, so that it is even whatever
// they are and a captured graph follows them: rows are counted in units of kUnit, every KV head's units of all
// sequences are shared out over about kTarget workgroups, and a workgroup takes an even share of one sequence.  A
// sequence of one share writes its output; the others write (m, l, O) per share and a second launch joins them, which
// also writes the zeros of the empty ones.
//
// A workgroup's part of it is in paged_decode.h.
#include "paged_decode.h"

namespace moss {
namespace {

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
        const int share = share_of_units(wave_total(units), shares), n = shares_of(units, share);  // (at most 2^23 units each)
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

template <typename E, int D, typename T, bool NT>
__global__ __launch_bounds__(256, 3) void paged_decode_split(DecodeArgs a, typename T::Cache c, PagedBatch bt) {
    __shared__ __attribute__((aligned(16))) float ow[4][16][D];
    __shared__ float mw[4][16], lw[4][16];
    const int tiles = (a.group + 15) / 16;  // head tiles of a KV head
    const int slot = blockIdx.x / a.xdim, x = blockIdx.x % a.xdim;
    const Place pl = find_share(bt, c.shift, a.shares, slot, threadIdx.x & (kWave - 1));
    if (pl.b < 0) return;
    ShareOf sh;
    sh.b = pl.b, sh.kvh = x / tiles, sh.h0 = 16 * (x % tiles), sh.heads = min(16, a.group - sh.h0);
    share_rows(paged_length(bt, pl.b, c.shift), pl.count, pl.index, sh.r0, sh.r1);
    sh.alone = pl.count == 1, sh.slot = slot;
    decode_share<E, D, T, NT, 4>(a, c, bt, sh, threadIdx.x, ow, mw, lw);
}

// grid (QH, B), 256 threads: the shares of one head of a sequence, wave w taking w, w + 4, ..; the four waves' sums meet
// in LDS.
template <typename E, int D>
__global__ __launch_bounds__(256) void paged_decode_join(DecodeArgs a, int shift, PagedBatch bt) {
    constexpr int VPL = D / kWave;
    __shared__ float acc_s[4][D];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & (kWave - 1), w = tid / kWave;
    const int su = share_units(bt, shift, a.shares, lane);
    const int count = shares_of(units_of(paged_length(bt, b, shift)), su);
    if (count == 1) return;  // written by its workgroup
    uint16_t* dst = a.out + ((size_t)b * a.qh + h) * D;
    if (count == 0) {
        for (int d = tid; d < D; d += 256) dst[d] = 0;
        return;
    }
    int first = 0;
    for (int s = lane; s < b; s += kWave) first += shares_of(units_of(paged_length(bt, s, shift)), su);
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

template <typename E, int D, typename T>
void launch_decode(const DecodeArgs& a, const typename T::Cache& c, const PagedBatch& bt, const DecodePlan& p, hipStream_t st) {
    const long long page = ((long long)c.kh << c.shift) * D * (std::is_same<typename T::Cache, PagedCache>::value ? 2 : 1);
    const long long named = (long long)bt.B * bt.W;
    const dim3 grid((unsigned)(p.xdim * p.slots));
    if ((named < c.pages ? named : c.pages) * page * 2 > kCached)
        hipLaunchKernelGGL((paged_decode_split<E, D, T, true>), grid, dim3(256), 0, st, a, c, bt);
    else
        hipLaunchKernelGGL((paged_decode_split<E, D, T, false>), grid, dim3(256), 0, st, a, c, bt);
    hipLaunchKernelGGL((paged_decode_join<E, D>), dim3((unsigned)a.qh, (unsigned)bt.B), dim3(256), 0, st, a, c.shift, bt);
}

template <template <typename, int> class T, typename Cache>
int decode(const void* q, long long q_stride, const Cache& c, const PagedBatch& bt, int qh, int d, float scale, void* out,
           void* workspace, long long workspace_bytes, int dtype, void* stream) {
    MOSS_CHECK_ARG(q && out && workspace && paged_pointers_ok(c, bt) && paged_shape_ok(c, bt, qh, d));
    MOSS_CHECK_ARG((dtype == 0 || dtype == 1) && q_stride % 8 == 0 && q_stride >= (long long)qh * d && paged_scale_ok(scale));
    MOSS_CHECK_ARG(MOSS_ALIGNED(q, 16) && MOSS_ALIGNED(out, 16) && MOSS_ALIGNED(workspace, 16));
    const DecodePlan p = decode_plan(bt.B, bt.W, c.shift, qh, c.kh);
    MOSS_CHECK_ARG(workspace_bytes >= p.slots * qh * (d + 2) * 4 && p.slots * p.xdim * 256 < (1ll << 32));
    DecodeArgs a{(const uint16_t*)q, q_stride, (uint16_t*)out, (float*)workspace,
                 reinterpret_cast<float2*>((float*)workspace + p.slots * qh * d), qh, qh / c.kh, p.xdim, p.shares, p.slots,
                 scale * 1.4426950408889634f, 0u};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0)
        d == 128 ? launch_decode<Bf16, 128, T<Bf16, 128>>(a, c, bt, p, st) : launch_decode<Bf16, 64, T<Bf16, 64>>(a, c, bt, p, st);
    else
        d == 128 ? launch_decode<F16, 128, T<F16, 128>>(a, c, bt, p, st) : launch_decode<F16, 64, T<F16, 64>>(a, c, bt, p, st);
    return moss_launch_status();
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
    return decode<Tile16>(q, q_stride, c, bt, qh, d, scale, out, workspace, workspace_bytes, dtype, stream);
}

MOSS_API int moss_paged_decode_attention_fp8(const void* q, long long q_stride, const void* k, const void* v, const void* k_scales,
                                             const void* v_scales, long long k_stride, long long v_stride,
                                             long long k_scale_stride, long long v_scale_stride, int pages, int page_rows,
                                             const void* table, long long table_stride, const void* lengths, int B, int W,
                                             int qh, int kh, int d, float scale, void* out, void* workspace,
                                             long long workspace_bytes, int dtype, void* stream) {
    const PagedCache8 c = paged_cache8(k, v, k_scales, v_scales, k_stride, v_stride, k_scale_stride, v_scale_stride, pages, kh, page_rows);
    const PagedBatch bt{(const int*)table, (const int*)lengths, nullptr, B, W, table_stride};
    MOSS_CHECK_ARG(paged8_ok(c));
    return decode<Tile8>(q, q_stride, c, bt, qh, d, scale, out, workspace, workspace_bytes, dtype, stream);
}
