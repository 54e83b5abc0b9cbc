// Sums and maxima over groups of neighbouring lanes without LDS.
#pragma once

#include "kvip_device.h"

namespace kvip {

template <int CTRL>
KVIP_DEVICE float dpp_all(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xF, 0xF, true));
}

// x of all G lanes of a group put together, in every lane of it; G lanes lie side by side.
template <int G, typename F>
KVIP_DEVICE float over_group(float x, F f) {
    x = f(x, dpp_all<0xB1>(x));   // lane ^ 1
    x = f(x, dpp_all<0x4E>(x));   // lane ^ 2
    x = f(x, dpp_all<0x141>(x));  // mirrored in 8
    if constexpr (G >= 16) x = f(x, dpp_all<0x140>(x));  // mirrored in 16
    if constexpr (G >= 32) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    }
    if constexpr (G >= 64) {
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    }
    return x;
}
template <int G> KVIP_DEVICE float group_sum(float x) { return over_group<G>(x, [](float a, float b) { return a + b; }); }
template <int G> KVIP_DEVICE float group_max(float x) { return over_group<G>(x, [](float a, float b) { return fmaxf(a, b); }); }

}  // namespace kvip
