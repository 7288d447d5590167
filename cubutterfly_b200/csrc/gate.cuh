// gate.cuh -- sigmoids of fp32 pairs on the special-function unit.
#pragma once

#include "f32x2.cuh"

namespace cubf::gate {

using f32x2::add2;
using f32x2::fma2;
using f32x2::mul2;
using Pair = f32x2::P;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLn2Rest = static_cast<float>(0.69314718055994530942 - static_cast<double>(kLn2));

CUBF_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
CUBF_DEV float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
CUBF_DEV float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
CUBF_DEV float min_nan(float a, float b) {
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

CUBF_DEV Pair both(float v) { return f32x2::pk(v, v); }
template <typename F>
CUBF_DEV Pair each(Pair p, F f) {
    float lo, hi;
    f32x2::up(p, lo, hi);
    return f32x2::pk(f(lo), f(hi));
}

// 1/(1 + exp(-v)) to the last bits of fp32.  exp(-v) is 2^h, h = -v log2(e), by
// the special-function unit; the rounding of h, which alone would make it off by
// |v| 2^-24, leaves t = -v - h ln 2, taken into account as the factor 1 + t.  |v|
// above 88 is taken as 88: exp(88) = 1.7e38 is finite, and its reciprocal flushes
// to zero like those of all beyond.
CUBF_DEV Pair sigmoid(Pair v) {
    const Pair u = each(v, [](float x) { return min_nan(max_nan(-x, -88.f), 88.f); });
    const Pair h = mul2(u, both(kLog2e)), e = each(h, [](float x) { return ex2(x); });
    const Pair t = fma2(h, both(-kLn2Rest), fma2(h, both(-kLn2), u));
    return each(add2(fma2(e, t, e), both(1.f)), [](float x) { return rcp(x); });
}

}  // namespace cubf::gate
