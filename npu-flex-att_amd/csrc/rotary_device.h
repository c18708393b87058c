// Positions of new tokens: the sine and cosine of a pair's angle, and a token's place, shared by the kernels that turn
// queries and keys (rotary.hip, norm_rotary.hip).
#pragma once
#include "flexatt_device.h"
#include "flexatt_kernels.h"

namespace flexatt {

// mag * cos and sgn * mag * sin of pos * freq radians.
__device__ __forceinline__ void turn_of(double pos, double freq, float mag, float sgn, float& c, float& s) {
  const double q = pos * (freq * 0.63661977236758134308);  // quarter turns: freq / (pi / 2)
  const double n = __builtin_rint(q);
  // |x| <= pi/4 (pi / 2 in 32 bits is off by 3e-8 of itself)
  const float x = (float)((q - n) * 1.57079632679489661923);
  // n mod 4 without leaving 64 bits, for any n a double holds
  const int k = (int)(n - 4.0 * __builtin_floor(n * 0.25));
  const float z = x * x;
  const float sp = x + x * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
  const float cp = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
  const float a = (k & 1) ? sp : cp, b = (k & 1) ? cp : sp;
  c = ((k == 1 || k == 2) ? -a : a) * mag;
  s = ((k & 2) ? -b : b) * (mag * sgn);
}

// Token n of the flattened (b, s): its sequence, index, cache slot and position.
__device__ __forceinline__ void token_of(const RotaryArgs& a, int64_t n, int& b, int& s, int64_t& slot, double& pos) {
  b = (int)(n / a.S);
  s = (int)(n % a.S);
  slot = a.lengths ? (int64_t)a.lengths[b] + s : s;
  if (a.pos_bytes == 8) pos = (double)((const int64_t*)a.positions)[b * a.pos_sb + s * a.pos_ss];
  else if (a.pos_bytes == 4) pos = (double)((const int32_t*)a.positions)[b * a.pos_sb + s * a.pos_ss];
  else pos = (double)slot;
}

}  // namespace flexatt
