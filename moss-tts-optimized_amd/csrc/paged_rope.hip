// q/k head RMSNorm, rotary embedding and the page write of new tokens, for a batch over a paged cache.
//
// Per head x of D values (weight w, or none: then no norm), in fp32 from the 16-bit input to one rounding at the end:
//   y = x rsqrt(mean(x^2) + eps) w;   out_l = y_l cos_l - y_{l + D/2} sin_l,
//   out_{l + D/2} = y_{l + D/2} cos_{l + D/2} + y_l sin_{l + D/2}   (l < D / 2)
// with row p of the cos / sin tables (bf16 / fp16 / fp32 as given) for the token's position p = length - n + i, token i
// of the sequence's n, the length cut to what the page table's row holds as the attentions cut it.  The single-request form (norm_rope.hip) rounds after every step, as the modules it stands in
// for do; here the steps are kept in fp32, which halves the error of q and k.
//
// What bounds it: memory (2549 tokens of 32 / 8 heads of 128: 13.8 us, 4.6 TB/s, where a large copy reaches 4.9; one token:
// the launch, 2.8 us).  A head is D / 16 lanes, each with 8 values of either half, so every load and store is 16
// bytes; one workgroup takes 256 / (D / 16) heads of one token, and a wave finds the token's sequence with one ballot
// per 64 sequences.
#include "paged.h"

namespace moss {
namespace {

struct RopeArgs {
    const uint16_t* qkv;
    long long qkv_stride;
    const uint16_t* qw;
    const uint16_t* kw;
    const void* cos_t;
    const void* sin_t;
    uint16_t* q_out;
    int T, qh, table_rows;
    float eps;
};

// 8 values from the table, as floats
template <typename E, bool F32>
__device__ __forceinline__ void table8(const void* t, size_t at, float (&v)[8]) {
    if constexpr (F32) {
        const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(t) + at);
        const float4 a = p[0], b = p[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint16_t*>(t) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = E::lo(w[i]), v[2 * i + 1] = E::hi(w[i]);
    }
}

template <typename E>
__device__ __forceinline__ void unpack8(u32x4_t w, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = E::lo(w[i]), v[2 * i + 1] = E::hi(w[i]);
}

template <typename E, int D, bool F32>
__global__ __launch_bounds__(256) void paged_rope_kernel(RopeArgs a, PagedCache c, PagedBatch bt) {
    constexpr int LPH = D / 16, HPB = 256 / LPH;  // lanes per head, heads per workgroup
    const int t = blockIdx.x, lane = threadIdx.x & (kWave - 1);
    // the token's sequence: with packed tokens the last one that starts at or before it (empty ones end there too)
    int b = t, position;
    if (bt.starts) {
        int at_or_before = 0;
        for (int b0 = 0; b0 < bt.B; b0 += kWave)
            at_or_before += __popcll(__ballot(b0 + lane < bt.B && bt.starts[min(b0 + lane, bt.B - 1)] <= t));
        b = at_or_before - 1;
        if (b < 0) return;
        const int end = min(bt.starts[b + 1], a.T);  // as the attention reads it
        if (t >= end) return;  // padding behind the last sequence
        position = paged_length(bt, b, c.shift) - end + t;
    } else {
        position = paged_length(bt, b, c.shift) - 1;
    }
    const int h = blockIdx.y * HPB + threadIdx.x / LPH, j = threadIdx.x % LPH;
    if (h >= a.qh + 2 * c.kh) return;  // whole groups of lanes
    const uint16_t* src = a.qkv + (size_t)t * a.qkv_stride + (size_t)h * D + 8 * j;
    const u32x4_t wa = *reinterpret_cast<const u32x4_t*>(src), wb = *reinterpret_cast<const u32x4_t*>(src + D / 2);
    // the row's place in the cache; a token without a position (more tokens than the length says) or a page has none
    uint16_t* dst = nullptr;
    if (h >= a.qh) {
        const bool is_k = h < a.qh + c.kh;
        const int page = page_of_row(bt.table + (size_t)b * bt.table_stride, position, bt.W, c.shift, c.pages);
        if (page >= 0)
            dst = (is_k ? c.k : c.v) + 8 * j +
                  row_offset(page, is_k ? c.k_stride : c.v_stride, h - a.qh - (is_k ? 0 : c.kh), position, c.shift, D);
        if (h >= a.qh + c.kh) {  // values go as they are
            if (dst) {
                *reinterpret_cast<u32x4_t*>(dst) = wa;
                *reinterpret_cast<u32x4_t*>(dst + D / 2) = wb;
            }
            return;
        }
    } else {
        dst = a.q_out + ((size_t)t * a.qh + h) * D + 8 * j;
    }
    float x[8], y[8];
    unpack8<E>(wa, x);
    unpack8<E>(wb, y);
    const uint16_t* wt = h < a.qh ? a.qw : a.kw;
    if (wt) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(x[i], x[i], fmaf(y[i], y[i], s));
#pragma unroll
        for (int m = 1; m < LPH; m <<= 1) s += __shfl_xor(s, m, LPH);
        const float r = rsqrtf(s / (float)D + a.eps);
        float u[8], v[8];
        unpack8<E>(*reinterpret_cast<const u32x4_t*>(wt + 8 * j), u);
        unpack8<E>(*reinterpret_cast<const u32x4_t*>(wt + D / 2 + 8 * j), v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = x[i] * r * u[i];
            y[i] = y[i] * r * v[i];
        }
    }
    const size_t row = (size_t)min(max(position, 0), a.table_rows - 1) * D + 8 * j;
    float cx[8], cy[8], sx[8], sy[8];
    table8<E, F32>(a.cos_t, row, cx);
    table8<E, F32>(a.cos_t, row + D / 2, cy);
    table8<E, F32>(a.sin_t, row, sx);
    table8<E, F32>(a.sin_t, row + D / 2, sy);
    if (!dst) return;
    u32x4_t lo, hi;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        lo[i] = E::pack(x[2 * i] * cx[2 * i] - y[2 * i] * sx[2 * i],
                        x[2 * i + 1] * cx[2 * i + 1] - y[2 * i + 1] * sx[2 * i + 1]);
        hi[i] = E::pack(y[2 * i] * cy[2 * i] + x[2 * i] * sy[2 * i],
                        y[2 * i + 1] * cy[2 * i + 1] + x[2 * i + 1] * sy[2 * i + 1]);
    }
    *reinterpret_cast<u32x4_t*>(dst) = lo;
    *reinterpret_cast<u32x4_t*>(dst + D / 2) = hi;
}

template <typename E, int D>
void launch_rope(const RopeArgs& a, const PagedCache& c, const PagedBatch& bt, bool f32, hipStream_t st) {
    constexpr int HPB = 256 / (D / 16);
    const dim3 grid((unsigned)a.T, (unsigned)((a.qh + 2 * c.kh + HPB - 1) / HPB));
    if (f32)
        hipLaunchKernelGGL((paged_rope_kernel<E, D, true>), grid, dim3(256), 0, st, a, c, bt);
    else
        hipLaunchKernelGGL((paged_rope_kernel<E, D, false>), grid, dim3(256), 0, st, a, c, bt);
}

}  // namespace
}  // namespace moss

using namespace moss;

MOSS_API int moss_paged_qk_rope(const void* qkv, long long qkv_stride, const void* q_weight, const void* k_weight,
                                const void* cos, const void* sin, int table_f32, int table_rows, void* q_out, void* k,
                                void* v, long long k_stride, long long v_stride, int pages, int page_rows,
                                const void* table, long long table_stride, const void* lengths, const void* starts, int B,
                                int W, int T, int qh, int kh, int d, float eps, int dtype, void* stream) {
    const PagedCache c = paged_cache(k, v, k_stride, v_stride, pages, kh, page_rows);
    const PagedBatch bt{(const int*)table, (const int*)lengths, (const int*)starts, B, W, table_stride};
    MOSS_CHECK_ARG(qkv && cos && sin && q_out && paged_pointers_ok(c, bt) && paged_shape_ok(c, bt, qh, d));
    // 256 threads a token: from 2^24 tokens on the grid would have more than 2^32 - 1
    MOSS_CHECK_ARG(T > 0 && T < (1 << 24) && (starts || T == B) && table_rows > 0 && eps >= 0.f && (dtype == 0 || dtype == 1));
    MOSS_CHECK_ARG((q_weight == nullptr) == (k_weight == nullptr) && qkv_stride % 8 == 0 &&
                   qkv_stride >= (long long)(qh + 2 * kh) * d);
    MOSS_CHECK_ARG(MOSS_ALIGNED(qkv, 16) && MOSS_ALIGNED(q_weight, 16) && MOSS_ALIGNED(k_weight, 16) && MOSS_ALIGNED(cos, 16) &&
                   MOSS_ALIGNED(sin, 16) && MOSS_ALIGNED(q_out, 16));
    const RopeArgs a{(const uint16_t*)qkv, qkv_stride, (const uint16_t*)q_weight, (const uint16_t*)k_weight, cos, sin,
                     (uint16_t*)q_out, T, qh, table_rows, eps};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0)
        d == 128 ? launch_rope<Bf16, 128>(a, c, bt, table_f32 != 0, st) : launch_rope<Bf16, 64>(a, c, bt, table_f32 != 0, st);
    else
        d == 128 ? launch_rope<F16, 128>(a, c, bt, table_f32 != 0, st) : launch_rope<F16, 64>(a, c, bt, table_f32 != 0, st);
    return moss_launch_status();
}
