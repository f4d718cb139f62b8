// Sums over a wave's lanes in lane order, of 32- and 64-bit integers, and maxima.
#pragma once

#include "common.h"

namespace moss {

// Lane l - d's value within its 16 lanes, or lane 15's / 31's for the lanes behind; 0 where there is none.
template <int CTRL, int ROWS, typename V>
__device__ __forceinline__ V dpp_before(V v) {
    if constexpr (sizeof(V) == 4) {
        return (V)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
    } else {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
        return ((V)hi << 32) | lo;
    }
}
// Inclusive sum over the wave's lanes (all of them active).
template <typename V>
__device__ __forceinline__ V wave_prefix(V v) {
    v += dpp_before<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
    v += dpp_before<0x112, 0xf>(v);
    v += dpp_before<0x114, 0xf>(v);
    v += dpp_before<0x118, 0xf>(v);
    v += dpp_before<0x142, 0xa>(v);  // lane 15 of rows 0 and 2 to the rows behind them
    v += dpp_before<0x143, 0xc>(v);  // lane 31 to the upper half
    return v;
}
// Inclusive maximum over the wave's lanes (all of them active), of unsigned values.
__device__ __forceinline__ uint32_t wave_prefix_max(uint32_t v) {
    v = max(v, dpp_before<0x111, 0xf>(v));
    v = max(v, dpp_before<0x112, 0xf>(v));
    v = max(v, dpp_before<0x114, 0xf>(v));
    v = max(v, dpp_before<0x118, 0xf>(v));
    v = max(v, dpp_before<0x142, 0xa>(v));
    v = max(v, dpp_before<0x143, 0xc>(v));
    return v;
}
template <typename V>
__device__ __forceinline__ V lane_value(V v, int lane) {
    if constexpr (sizeof(V) == 4) {
        return (V)__builtin_amdgcn_readlane((int)v, lane);
    } else {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
        return ((V)hi << 32) | lo;
    }
}
template <typename V>
__device__ __forceinline__ V wave_total(V v) {  // the same value in every lane
    return lane_value(wave_prefix(v), kWave - 1);
}

}  // namespace moss
