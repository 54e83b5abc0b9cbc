// Turns of rotary positions and vectors of features, shared by the kernels that turn heads.
#pragma once

#include "kvip_device.h"

namespace kvip {

// (cos, sin) times the magnitude of the angle position * frequency: its turns in 64 bits, of which only the fraction
// goes on.
KVIP_DEVICE float2 turn_of(int64_t position, double frequency, float magnitude, bool inverse) {
    const double turns = static_cast<double>(position) * frequency * 0.15915494309189533577;  // 1 / (2 pi)
    const float fraction = static_cast<float>(turns - rint(turns));
    float s, c;
    sincospif(2.0f * fraction, &s, &c);
    return make_float2(c * magnitude, (inverse ? -s : s) * magnitude);
}

}  // namespace kvip
