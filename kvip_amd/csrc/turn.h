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

// The same with whole quarter turns taken out first, so that the angle is rounded to 32 bits at an eighth of a turn at most:
// by 2.3e-8 instead of 9.4e-8, what else is rounded on a feature's way to its code being 3e-8 at a time. (Of 1.4 million
// layer-normed keys times 128 features 300 instead of 401 have another code than in 64 bits, at no cost in time. Turns without
// a norm stay with turn_of, whose results callers have.)
KVIP_DEVICE float2 fine_turn_of(int64_t position, double frequency, float magnitude) {
    const double turns = static_cast<double>(position) * frequency * 0.15915494309189533577;  // 1 / (2 pi)
    const double quarters = 4.0 * (turns - rint(turns)), whole = rint(quarters);
    const int quadrant = static_cast<int>(whole);
    float s, c;
    sincospif(0.5f * static_cast<float>(quarters - whole), &s, &c);
    const float sine = (quadrant & 1) != 0 ? c : s, cosine = (quadrant & 1) != 0 ? s : c;
    return make_float2(((quadrant + 1) & 2) != 0 ? -cosine * magnitude : cosine * magnitude, (quadrant & 2) != 0 ? -sine * magnitude : sine * magnitude);
}

}  // namespace kvip
