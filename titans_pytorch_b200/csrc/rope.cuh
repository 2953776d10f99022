// The rotation of one (position, pair): shared by the rotary operator and the
// key/value cache write, which rotates on the way.
#pragma once

#include <stdint.h>

namespace tb {

// cos and sin of position * freq.  The product of an integer position and an
// fp32 frequency is exact in fp64 up to 2^53, so it is formed and reduced to
// [-pi, pi] there (2 pi as a sum of two doubles); an fp32 product would be off
// by 0.06 rad at a million tokens.  The reduced angle goes to sincosf.
__device__ __forceinline__ float2 rope_cos_sin(int64_t position, float freq, float amplitude) {
  const double a = (double)position * (double)freq;
  const double k = rint(a * 0.15915494309189535);           // a / (2 pi)
  double r = fma(-k, 6.283185307179586, a);                 // 2 pi, high part
  r = fma(-k, 2.4492935982947064e-16, r);                   // 2 pi, low part
  float s, c;
  sincosf((float)r, &s, &c);
  return make_float2(amplitude * c, amplitude * s);
}

}  // namespace tb
