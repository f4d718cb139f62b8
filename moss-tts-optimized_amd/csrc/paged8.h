// A paged cache in 8 bits: e4m3 codes, and for each row of a KV head one byte that says by which power of two.
//
// A row of D values x (|x| finite, A the largest) is held as codes c_i = RNE_e4m3(x_i 2^-e) and the byte e + 127, with e the least
// integer that brings the row under e4m3's largest value, A <= 448 2^e.  A code has four significant bits, so c 2^e is
// exact in bf16 and, for -15 <= e <= 8, in fp16: what the attentions multiply is what the cache holds, with no rounding of its
// own, and a power of two costs e4m3 nothing that a finer scale would keep (its steps are relative, but for the least codes,
// of 2^-9: an eighth of a step of 448's neighbours 2^-15 down).  A scale a row and not a page, since rows come one at a time
// and a row that is written must not change the others.
//
// Scales lie as k / v do: [pages, KH, P] bytes, the page stride free (a multiple of 16).
#pragma once

#include "paged.h"

namespace moss {

struct PagedCache8 : PagedCache {  // k and v are bytes, k_stride and v_stride count them
    uint8_t* ks;
    uint8_t* vs;
    long long ks_stride, vs_stride;
    __device__ __forceinline__ const uint8_t* kc() const { return reinterpret_cast<const uint8_t*>(k); }
    __device__ __forceinline__ const uint8_t* vc() const { return reinterpret_cast<const uint8_t*>(v); }
};

// 2^(byte - 127) from the byte's bits: 1 .. 254 are powers of two.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Byte i of a word, as a scale.
template <int I>
__device__ __forceinline__ float scale_at(uint32_t word) {
    return __uint_as_float((I < 3 ? (word >> (8 * I)) & 0xffu : word >> 24) << 23);
}

// Two codes of a word (its low or high half) times a scale, as a pair of the 16-bit type.
template <typename E, bool HI>
__device__ __forceinline__ uint32_t widen(uint32_t codes, float scale) {
    if constexpr (E::kHalf)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HI));
    else
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HI));
}

// Eight codes as eight values.
template <typename E>
__device__ __forceinline__ u32x4_t widen8(uint32_t a, uint32_t b, float scale) {
    return u32x4_t{widen<E, false>(a, scale), widen<E, true>(a, scale), widen<E, false>(b, scale), widen<E, true>(b, scale)};
}

// The byte of a row whose largest finite value is `top`: ceil(log2(top / 448)) from its bits (448 = 1.75 2^8), within what
// keeps every code exact in the 16-bit type.
template <typename E>
__device__ __forceinline__ uint32_t scale_byte(float top) {
    const int e = (int)((__float_as_uint(top) + 0x1fffffu) >> 23) - 8;
    return (uint32_t)min(max(e, 127 + E::kLeast), 127 + E::kMost);
}

// Four values times 2^-e (`inverse`) as codes.  What passes the type's largest code times its largest scale is held at that;
// NaN and infinities are e4m3's NaN.
template <typename E>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inverse, float most) {
    auto held = [&](float x) {
        const float y = fminf(fmaxf(x * inverse, -most), most);
        return x - x == 0.f ? y : NAN;
    };
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(held(a), held(b), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(held(c), held(d), w, true);
    return (uint32_t)w;
}
// The largest code of a row with this byte: 240 at the largest scale, where 448 would leave the 16-bit type.
template <typename E>
__device__ __forceinline__ float most_of(uint32_t byte) {
    return byte == (uint32_t)(127 + E::kMost) ? 240.f : 448.f;
}

static inline PagedCache8 paged_cache8(const void* k, const void* v, const void* ks, const void* vs, long long k_stride,
                                       long long v_stride, long long ks_stride, long long vs_stride, int pages, int kh,
                                       int page_rows) {
    PagedCache8 c;
    static_cast<PagedCache&>(c) = paged_cache(k, v, k_stride, v_stride, pages, kh, page_rows);
    c.ks = (uint8_t*)ks, c.vs = (uint8_t*)vs, c.ks_stride = ks_stride, c.vs_stride = vs_stride;
    return c;
}

// Beside paged_shape_ok and paged_pointers_ok: pages of codes and of scales begin at 16 bytes.
static inline bool paged8_ok(const PagedCache8& c) {
    return c.ks && c.vs && MOSS_ALIGNED(c.ks, 16) && MOSS_ALIGNED(c.vs, 16) && c.k_stride % 16 == 0 && c.v_stride % 16 == 0 &&
           c.ks_stride % 16 == 0 && c.vs_stride % 16 == 0 && c.ks_stride >= ((long long)c.kh << c.shift) &&
           c.vs_stride >= ((long long)c.kh << c.shift);
}

}  // namespace moss
