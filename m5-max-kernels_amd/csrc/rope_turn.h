// Sine and cosine of a rotary position.
//
// Angles.  p f_j / 2 pi is reduced to a fraction of a turn in 64 bits: at position 10^6 an FP32 angle would be off by
// 0.06 rad, the 64-bit fraction by 10^-10.  The fraction's nearest quarter turn is taken off in 64 bits too and the
// rest, |y| <= pi / 4, goes through the Taylor series of sine and cosine in FP32 (terms left out below 2e-9).
#pragma once

#include "m5k_common.h"

namespace m5k {

constexpr double INV_TURN = 0.15915494309189533577;  // 1 / (2 pi)

__device__ __forceinline__ void turn_of(int position, double frequency, float magnitude, float& c, float& s) {
  double t = static_cast<double>(position) * (frequency * INV_TURN);
  t -= rint(t);
  const double q = rint(4.0 * t);
  const float y = static_cast<float>(t - 0.25 * q) * 6.28318530717958647692f;
  const float z = y * y;
  float a = __builtin_fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f);
  a = __builtin_fmaf(z, a, 1.0f / 120.0f);
  a = __builtin_fmaf(z, a, -1.0f / 6.0f);
  const float sine = __builtin_fmaf(y * z, a, y);
  float b = __builtin_fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  b = __builtin_fmaf(z, b, -1.0f / 720.0f);
  b = __builtin_fmaf(z, b, 1.0f / 24.0f);
  b = __builtin_fmaf(z, b, -0.5f);
  const float cosine = __builtin_fmaf(z, b, 1.0f);
  const int quarter = static_cast<int>(q) & 3;
  const bool odd = quarter & 1;
  c = (odd ? sine : cosine) * ((quarter == 1 || quarter == 2) ? -magnitude : magnitude);
  s = (odd ? cosine : sine) * (quarter >= 2 ? -magnitude : magnitude);
}

}  // namespace m5k
