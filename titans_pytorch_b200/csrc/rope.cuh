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

// n / d for n < 2^31 by a multiplication (Granlund & Montgomery, 1994): the
// hardware has no integer division, and three of them an item were two thirds
// of the rotation's instructions.
struct FastDiv {
  uint32_t d, m, s;
  FastDiv() : d(1), m(1), s(0) {}
  explicit FastDiv(uint32_t div) : d(div), s(0) {
    while ((1ull << s) < div) ++s;
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - div)) / div + 1);
  }
  __device__ __forceinline__ int operator()(int n, int& rest) const {
    const uint32_t q = (__umulhi((uint32_t)n, m) + (uint32_t)n) >> s;
    rest = n - (int)(q * d);
    return (int)q;
  }
};

// Tables of N consecutive pairs' cos and sin in shared memory, as two arrays:
// lanes read neighbouring 16-byte pieces (pairs side by side as float2 made the
// reads of a warp collide eight times).  N * 4 bytes aligned.
template <int N> __device__ __forceinline__ void table_load(const float* t, float (&v)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 a = *reinterpret_cast<const float4*>(t + i);
      v[i] = a.x; v[i + 1] = a.y; v[i + 2] = a.z; v[i + 3] = a.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 a = *reinterpret_cast<const float2*>(t + i);
      v[i] = a.x; v[i + 1] = a.y;
    }
  }
}

}  // namespace tb
