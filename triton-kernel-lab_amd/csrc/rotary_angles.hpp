// Angles of rotary positions, shared by the kernels that turn queries and keys (rotary.hip,
// qk_norm_rotary.hip).
#pragma once
#include "tk_common.hpp"

namespace tk_rotary_angles {

// sin and cos of r in [-pi/4, pi/4] by their Taylor series (coefficients 1/n!).
__device__ __forceinline__ void sincos_reduced(double r, double& s, double& c) {
  const double z = r * r;
  double p = -1.0 / 39916800.0;
  p = fma(p, z, 1.0 / 362880.0);
  p = fma(p, z, -1.0 / 5040.0);
  p = fma(p, z, 1.0 / 120.0);
  p = fma(p, z, -1.0 / 6.0);
  s = fma(p * z, r, r);
  double q = 1.0 / 479001600.0;
  q = fma(q, z, -1.0 / 3628800.0);
  q = fma(q, z, 1.0 / 40320.0);
  q = fma(q, z, -1.0 / 720.0);
  q = fma(q, z, 1.0 / 24.0);
  q = fma(q, z, -0.5);
  c = fma(q, z, 1.0);
}

// sin and cos of any finite x.
__device__ __forceinline__ void sincos_any(double x, double& s, double& c) {
  // x = k pi/2 + r; pi/2 in two parts, the first with all 53 bits. Past 2^51 the rounding of
  // x * 2/pi is off by whole quarter turns: the second pass takes off those that are left.
  const double k = rint(x * 0.63661977236758134308);
  double r = fma(k, -1.5707963267948965580, x);
  r = fma(k, -6.1232339957367658e-17, r);
  const double more = rint(r * 0.63661977236758134308);
  r = fma(more, -1.5707963267948965580, r);
  r = fma(more, -6.1232339957367658e-17, r);
  sincos_reduced(r, s, c);
  // k modulo 4 is exact for every finite k.
  const int quarter = int(k - 4.0 * floor(0.25 * k)) + int(more);
  if (quarter & 1) {
    const double swap = s;
    s = c;
    c = -swap;
  }
  if (quarter & 2) {
    s = -s;
    c = -c;
  }
}

}  // namespace tk_rotary_angles
