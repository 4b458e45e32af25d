// sdpa_scan.h -- sums over the lanes of a wave by moves between registers.
#pragma once

#include <type_traits>

#include "sdpa_device.h"

namespace sdpa {
namespace {

// Inclusive sum over the lanes before and up to each (DPP moves inside rows of 16
// lanes, then the last lane of a row to the rows behind).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or_0(int x) {
    return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int x) {
    x += dpp_or_0<0x111, 0xF>(x);  // row_shr 1, 2, 4, 8
    x += dpp_or_0<0x112, 0xF>(x);
    x += dpp_or_0<0x114, 0xF>(x);
    x += dpp_or_0<0x118, 0xF>(x);
    x += dpp_or_0<0x142, 0xA>(x);  // row_bcast 15, 31
    x += dpp_or_0<0x143, 0xC>(x);
    return x;
}
__device__ __forceinline__ long long wave_scan(long long x) {
    const auto add = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
        const uint32_t lo = (uint32_t)dpp_or_0<decltype(ctrl)::value, decltype(rows)::value>((int)x);
        const int hi = dpp_or_0<decltype(ctrl)::value, decltype(rows)::value>((int)(x >> 32));
        x += ((long long)hi << 32) | lo;
    };
    add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});
    return x;
}
__device__ __forceinline__ long long readlane64(long long x, int l) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)x, l);
    return ((long long)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32) | lo;
}

}  // namespace
}  // namespace sdpa
