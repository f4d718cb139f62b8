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
//
// Into a cache of 8 bits (paged8.h) go the row's largest value over its lanes as its scale byte, and the codes.  K is rounded
// once there too, and not to 16 bits before.  Its arithmetic is in 64 bits: a value on the wrong side of a border between two
// codes is off by 2^-3 of itself, and fp32 sends one in a million there.  The heads with more to do go first, so that
// the others fill the end: write and gather of 2549 tokens take 20.8 us with fp32, 23.0 in 64 bits, 21.1 in this order
// (one token 6.4, 6.8, 6.5); the write alone 15.5, 4.0 TB/s.
#include "paged8.h"

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

// To fp32 so that rounding again, to fewer bits, gives what one rounding would have given: towards zero, with the last bit set
// where that left something out.
__device__ __forceinline__ float to_odd(double x) {
    const float f = (float)x;
    uint32_t w = __float_as_uint(f);
    if ((double)f != x && x == x) {
        if (fabs((double)f) > fabs(x)) w -= 1;
        w |= 1u;
    }
    return __uint_as_float(w);
}

// The row of an 8-bit cache that D / 16 lanes hold, 8 values of either half each (all of a row's lanes come here).
template <typename E, int D>
__device__ __forceinline__ void store_row8(uint8_t* codes, uint8_t* scale, int j, const float (&x)[8], const float (&y)[8]) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        top = fmaxf(top, x[i] - x[i] == 0.f ? fabsf(x[i]) : 0.f);
        top = fmaxf(top, y[i] - y[i] == 0.f ? fabsf(y[i]) : 0.f);
    }
#pragma unroll
    for (int m = 1; m < D / 16; m <<= 1) top = fmaxf(top, __shfl_xor(top, m, D / 16));
    const uint32_t byte = scale_byte<E>(top);
    const float inverse = scale_of(254 - byte), most = most_of<E>(byte);
    *reinterpret_cast<uint2*>(codes + 8 * j) = make_uint2(codes4<E>(x[0], x[1], x[2], x[3], inverse, most),
                                                          codes4<E>(x[4], x[5], x[6], x[7], inverse, most));
    *reinterpret_cast<uint2*>(codes + D / 2 + 8 * j) = make_uint2(codes4<E>(y[0], y[1], y[2], y[3], inverse, most),
                                                                  codes4<E>(y[4], y[5], y[6], y[7], inverse, most));
    if (j == 0) *scale = (uint8_t)byte;
}

template <typename E, int D, bool F32, typename Cache>
__global__ __launch_bounds__(256) void paged_rope_kernel(RopeArgs a, Cache c, PagedBatch bt) {
    constexpr bool EIGHT = std::is_same<Cache, PagedCache8>::value;
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
    const int h = (EIGHT ? gridDim.y - 1 - blockIdx.y : blockIdx.y) * HPB + threadIdx.x / LPH, j = threadIdx.x % LPH;
    if (h >= a.qh + 2 * c.kh) return;  // whole groups of lanes
    const uint16_t* src = a.qkv + (size_t)t * a.qkv_stride + (size_t)h * D + 8 * j;
    const u32x4_t wa = *reinterpret_cast<const u32x4_t*>(src), wb = *reinterpret_cast<const u32x4_t*>(src + D / 2);
    // the row's place in the cache; a token without a position (more tokens than the length says) or a page has none
    uint16_t* dst = nullptr;
    uint8_t *codes = nullptr, *scale = nullptr;
    if (h >= a.qh) {
        const bool is_k = h < a.qh + c.kh;
        const int page = page_of_row(bt.table + (size_t)b * bt.table_stride, position, bt.W, c.shift, c.pages);
        const int head = h - a.qh - (is_k ? 0 : c.kh);
        if constexpr (EIGHT) {
            if (page < 0) return;
            codes = reinterpret_cast<uint8_t*>(is_k ? c.k : c.v) +
                    row_offset(page, is_k ? c.k_stride : c.v_stride, head, position, c.shift, D);
            scale = (is_k ? c.ks : c.vs) + row_offset(page, is_k ? c.ks_stride : c.vs_stride, head, position, c.shift, 1);
            if (!is_k) {
                float x[8], y[8];
                unpack8<E>(wa, x);
                unpack8<E>(wb, y);
                store_row8<E, D>(codes, scale, j, x, y);
                return;
            }
        } else if (page >= 0) {
            dst = (is_k ? c.k : c.v) + 8 * j + row_offset(page, is_k ? c.k_stride : c.v_stride, head, position, c.shift, D);
        }
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
    const size_t row = (size_t)min(max(position, 0), a.table_rows - 1) * D + 8 * j;
    if constexpr (EIGHT) {
        if (h >= a.qh) {
            double r = 1.;
            u32x4_t wx = {}, wy = {};
            if (a.kw) {
                double s = 0.;
#pragma unroll
                for (int i = 0; i < 8; ++i) s = fma((double)x[i], (double)x[i], fma((double)y[i], (double)y[i], s));
#pragma unroll
                for (int m = 1; m < LPH; m <<= 1) s += __shfl_xor(s, m, LPH);
                s = s / (double)D + (double)a.eps;
                r = __builtin_amdgcn_rsq(s);  // about 2^-24 off: one step of Newton's
                if (s < INFINITY) r = fma(0.5 * r, fma(-s * r, r, 1.), r);
                wx = *reinterpret_cast<const u32x4_t*>(a.kw + 8 * j), wy = *reinterpret_cast<const u32x4_t*>(a.kw + D / 2 + 8 * j);
            }
            float cx[8], cy[8], sx[8], sy[8];
            table8<E, F32>(a.cos_t, row, cx);
            table8<E, F32>(a.sin_t, row, sx);
            table8<E, F32>(a.cos_t, row + D / 2, cy);
            table8<E, F32>(a.sin_t, row + D / 2, sy);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                double p = x[i], q = y[i];
                if (a.kw) {
                    p *= r * (i & 1 ? E::hi(wx[i / 2]) : E::lo(wx[i / 2]));
                    q *= r * (i & 1 ? E::hi(wy[i / 2]) : E::lo(wy[i / 2]));
                }
                x[i] = to_odd(p * cx[i] - q * sx[i]);
                y[i] = to_odd(q * cy[i] + p * sy[i]);
            }
            store_row8<E, D>(codes, scale, j, x, y);
            return;
        }
    }
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

template <typename E, int D, typename Cache>
void launch_rope(const RopeArgs& a, const Cache& c, const PagedBatch& bt, bool f32, hipStream_t st) {
    constexpr int HPB = 256 / (D / 16);
    const dim3 grid((unsigned)a.T, (unsigned)((a.qh + 2 * c.kh + HPB - 1) / HPB));
    if (f32)
        hipLaunchKernelGGL((paged_rope_kernel<E, D, true, Cache>), grid, dim3(256), 0, st, a, c, bt);
    else
        hipLaunchKernelGGL((paged_rope_kernel<E, D, false, Cache>), grid, dim3(256), 0, st, a, c, bt);
}

template <typename Cache>
int rope(const RopeArgs& a, const Cache& c, const PagedBatch& bt, int d, int table_f32, int dtype, hipStream_t st) {
    MOSS_CHECK_ARG(a.qkv && a.cos_t && a.sin_t && a.q_out && paged_pointers_ok(c, bt) && paged_shape_ok(c, bt, a.qh, d));
    // 256 threads a token: from 2^24 tokens on the grid would have more than 2^32 - 1
    MOSS_CHECK_ARG(a.T > 0 && a.T < (1 << 24) && (bt.starts || a.T == bt.B) && a.table_rows > 0 && a.eps >= 0.f &&
                   (dtype == 0 || dtype == 1));
    MOSS_CHECK_ARG((a.qw == nullptr) == (a.kw == nullptr) && a.qkv_stride % 8 == 0 &&
                   a.qkv_stride >= (long long)(a.qh + 2 * c.kh) * d);
    MOSS_CHECK_ARG(MOSS_ALIGNED(a.qkv, 16) && MOSS_ALIGNED(a.qw, 16) && MOSS_ALIGNED(a.kw, 16) && MOSS_ALIGNED(a.cos_t, 16) &&
                   MOSS_ALIGNED(a.sin_t, 16) && MOSS_ALIGNED(a.q_out, 16));
    if (dtype == 0)
        d == 128 ? launch_rope<Bf16, 128>(a, c, bt, table_f32 != 0, st) : launch_rope<Bf16, 64>(a, c, bt, table_f32 != 0, st);
    else
        d == 128 ? launch_rope<F16, 128>(a, c, bt, table_f32 != 0, st) : launch_rope<F16, 64>(a, c, bt, table_f32 != 0, st);
    return moss_launch_status();
}

// ---------------------------------------------------------------- the rows back, in order
// Token t of a sequence's n newest: the K and V rows at its position, as the 16-bit type; a token without a position or a page
// gives zeros.  What bounds it: memory and the launch (2549 tokens from 8 bits 5.5 us, 2.9 TB/s; one 2.4).  A row is D / 16 lanes with 8 values of either half, a wave takes 1024 / D rows of one
// token (K heads, then V heads), so the token's sequence is found with one ballot per 64 sequences.
struct GatherArgs {
    uint16_t* k_out;
    uint16_t* v_out;
    int T, t0, t1, waves;  // tokens in all, those of the launch; waves a token
};

template <typename E, int D, typename Cache>
__global__ __launch_bounds__(256) void paged_gather_kernel(GatherArgs a, Cache c, PagedBatch bt) {
    constexpr int LPH = D / 16, RPW = kWave / LPH;
    const int lane = threadIdx.x & (kWave - 1);
    const long long wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + threadIdx.x / kWave));
    const int t = a.t0 + (int)(wave / a.waves), part = (int)(wave % a.waves);
    if (t >= a.t1) return;
    int at_or_before = 0;
    for (int b0 = 0; b0 < bt.B; b0 += kWave)
        at_or_before += __popcll(__ballot(b0 + lane < bt.B && bt.starts[min(b0 + lane, bt.B - 1)] <= t));
    const int b = at_or_before - 1;
    if (b < 0) return;
    const int end = min(bt.starts[b + 1], a.T);
    if (t >= end) return;  // padding behind the last sequence
    const int position = paged_length(bt, b, c.shift) - end + t;
    const int row = part * RPW + lane / LPH, j = lane % LPH;
    if (row >= 2 * c.kh) return;
    const bool is_k = row < c.kh;
    const int head = row - (is_k ? 0 : c.kh);
    const int page = page_of_row(bt.table + (size_t)b * bt.table_stride, position, bt.W, c.shift, c.pages);
    u32x4_t lo = {0u, 0u, 0u, 0u}, hi = lo;
    if (page >= 0) {
        const size_t at = row_offset(page, is_k ? c.k_stride : c.v_stride, head, position, c.shift, D) + 8 * j;
        if constexpr (std::is_same<Cache, PagedCache8>::value) {
            const uint8_t* src = (is_k ? c.kc() : c.vc()) + at;
            const float scale =
                scale_of((is_k ? c.ks : c.vs)[row_offset(page, is_k ? c.ks_stride : c.vs_stride, head, position, c.shift, 1)]);
            const uint2 p = *reinterpret_cast<const uint2*>(src), q = *reinterpret_cast<const uint2*>(src + D / 2);
            lo = widen8<E>(p.x, p.y, scale);
            hi = widen8<E>(q.x, q.y, scale);
        } else {
            const uint16_t* src = (is_k ? c.k : c.v) + at;
            lo = *reinterpret_cast<const u32x4_t*>(src);
            hi = *reinterpret_cast<const u32x4_t*>(src + D / 2);
        }
    }
    uint16_t* dst = (is_k ? a.k_out : a.v_out) + ((size_t)t * c.kh + head) * D + 8 * j;
    *reinterpret_cast<u32x4_t*>(dst) = lo;
    *reinterpret_cast<u32x4_t*>(dst + D / 2) = hi;
}

template <typename E, int D, typename Cache>
void launch_gather(GatherArgs a, const Cache& c, const PagedBatch& bt, hipStream_t st) {
    // a grid has fewer than 2^32 threads: all tokens, or the first of outputs of 137 GB and more
    const int most = ((1 << 26) - 4) / a.waves;
    for (; a.t0 < a.T; a.t0 = a.t1) {
        a.t1 = a.T - a.t0 < most ? a.T : a.t0 + most;
        hipLaunchKernelGGL((paged_gather_kernel<E, D, Cache>), dim3((unsigned)(((long long)(a.t1 - a.t0) * a.waves + 3) / 4)), dim3(256),
                           0, st, a, c, bt);
    }
}

template <typename Cache>
int gather(void* k_out, void* v_out, const Cache& c, const PagedBatch& bt, int T, int d, int dtype, hipStream_t st) {
    MOSS_CHECK_ARG(k_out && v_out && bt.starts && paged_pointers_ok(c, bt) && paged_shape_ok(c, bt, c.kh, d));
    MOSS_CHECK_ARG(MOSS_ALIGNED(k_out, 16) && MOSS_ALIGNED(v_out, 16) && (dtype == 0 || dtype == 1) && T > 0 && T < (1 << 24));
    const int rows = 1024 / d;  // of a wave
    const GatherArgs a{(uint16_t*)k_out, (uint16_t*)v_out, T, 0, 0, (2 * c.kh + rows - 1) / rows};
    if (dtype == 0)
        d == 128 ? launch_gather<Bf16, 128>(a, c, bt, st) : launch_gather<Bf16, 64>(a, c, bt, st);
    else
        d == 128 ? launch_gather<F16, 128>(a, c, bt, st) : launch_gather<F16, 64>(a, c, bt, st);
    return moss_launch_status();
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
    const RopeArgs a{(const uint16_t*)qkv, qkv_stride, (const uint16_t*)q_weight, (const uint16_t*)k_weight, cos, sin,
                     (uint16_t*)q_out, T, qh, table_rows, eps};
    return rope(a, c, bt, d, table_f32, dtype, (hipStream_t)stream);
}

MOSS_API int moss_paged_qk_rope_fp8(const void* qkv, long long qkv_stride, const void* q_weight, const void* k_weight,
                                    const void* cos, const void* sin, int table_f32, int table_rows, void* q_out, void* k,
                                    void* v, void* k_scales, void* v_scales, long long k_stride, long long v_stride,
                                    long long k_scale_stride, long long v_scale_stride, int pages, int page_rows,
                                    const void* table, long long table_stride, const void* lengths, const void* starts, int B,
                                    int W, int T, int qh, int kh, int d, float eps, int dtype, void* stream) {
    const PagedCache8 c = paged_cache8(k, v, k_scales, v_scales, k_stride, v_stride, k_scale_stride, v_scale_stride, pages, kh, page_rows);
    const PagedBatch bt{(const int*)table, (const int*)lengths, (const int*)starts, B, W, table_stride};
    const RopeArgs a{(const uint16_t*)qkv, qkv_stride, (const uint16_t*)q_weight, (const uint16_t*)k_weight, cos, sin,
                     (uint16_t*)q_out, T, qh, table_rows, eps};
    MOSS_CHECK_ARG(paged8_ok(c));
    return rope(a, c, bt, d, table_f32, dtype, (hipStream_t)stream);
}

MOSS_API int moss_paged_gather(const void* k, const void* v, long long k_stride, long long v_stride, int pages, int page_rows,
                               const void* table, long long table_stride, const void* lengths, const void* starts, int B, int W,
                               int T, int kh, int d, void* k_out, void* v_out, int dtype, void* stream) {
    const PagedCache c = paged_cache(k, v, k_stride, v_stride, pages, kh, page_rows);
    const PagedBatch bt{(const int*)table, (const int*)lengths, (const int*)starts, B, W, table_stride};
    return gather(k_out, v_out, c, bt, T, d, dtype, (hipStream_t)stream);
}

MOSS_API int moss_paged_gather_fp8(const void* k, const void* v, const void* k_scales, const void* v_scales, long long k_stride,
                                   long long v_stride, long long k_scale_stride, long long v_scale_stride, int pages,
                                   int page_rows, const void* table, long long table_stride, const void* lengths,
                                   const void* starts, int B, int W, int T, int kh, int d, void* k_out, void* v_out, int dtype,
                                   void* stream) {
    const PagedCache8 c = paged_cache8(k, v, k_scales, v_scales, k_stride, v_stride, k_scale_stride, v_scale_stride, pages, kh, page_rows);
    const PagedBatch bt{(const int*)table, (const int*)lengths, (const int*)starts, B, W, table_stride};
    MOSS_CHECK_ARG(paged8_ok(c));
    return gather(k_out, v_out, c, bt, T, d, dtype, (hipStream_t)stream);
}
