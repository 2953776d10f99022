// Layout and element types of the key/value cache, shared by its write, its
// read and the attention over it.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace tb {

// One of the two halves (keys or values) of a cache [B, H, S, d]: rows of d
// contiguous elements, any strides over B, H, S; scales [B, H, S] (fp32, one
// per row) for the 8-bit kinds.  Strides are in elements.
struct CacheView {
  void* data;
  float* scale;
  int64_t sb, sh, ss;     // data
  int64_t qb, qh, qs;     // scales
};

enum CacheKind : int { KV_F32 = 0, KV_BF16 = 1, KV_F16 = 2, KV_I8 = 3, KV_E4M3 = 4 };

struct e4m3 {
  uint8_t bits;
};

template <> __device__ __forceinline__ float to_f<int8_t>(int8_t v) { return (float)v; }
template <> __device__ __forceinline__ float to_f<e4m3>(e4m3 v) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(v.bits, __NV_E4M3)));
}

template <typename C> struct CacheTraits { static constexpr bool scaled = false; };
template <> struct CacheTraits<int8_t> {
  static constexpr bool scaled = true;
  static constexpr float top = 127.f;
  static __device__ __forceinline__ int8_t pack(float y) { return (int8_t)__float2int_rn(y); }
};
template <> struct CacheTraits<e4m3> {
  static constexpr bool scaled = true;
  static constexpr float top = 448.f;
  static __device__ __forceinline__ e4m3 pack(float y) {
    return e4m3{(uint8_t)__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3)};
  }
};

// 8 consecutive elements (8, 16 or 32 bytes, aligned to their size).
template <typename C> __device__ __forceinline__ void load8(const C* p, float (&v)[8]) {
  if constexpr (sizeof(C) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else if constexpr (sizeof(C) == 2) {
    load16<C>(p, v);
  } else {
    union { uint2 raw; C c[8]; } u;
    u.raw = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f<C>(u.c[i]);
  }
}
template <typename C> __device__ __forceinline__ void store8(C* p, const float (&v)[8]) {
  if constexpr (sizeof(C) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else if constexpr (sizeof(C) == 2) {
    store16<C>(p, v);
  } else {
    union { uint2 raw; C c[8]; } u;
#pragma unroll
    for (int i = 0; i < 8; ++i) u.c[i] = CacheTraits<C>::pack(v[i]);
    *reinterpret_cast<uint2*>(p) = u.raw;
  }
}

#define TB_DISPATCH_CACHE(kind, NAME, ...)                          \
  [&] {                                                             \
    switch (kind) {                                                 \
      case KV_F32: { using cache_t = float; return __VA_ARGS__(); }           \
      case KV_BF16: { using cache_t = __nv_bfloat16; return __VA_ARGS__(); }  \
      case KV_F16: { using cache_t = __half; return __VA_ARGS__(); }          \
      case KV_I8: { using cache_t = int8_t; return __VA_ARGS__(); }           \
      case KV_E4M3: { using cache_t = e4m3; return __VA_ARGS__(); }           \
    }                                                               \
    TORCH_CHECK(false, NAME, ": unsupported cache type");           \
  }()

inline int cache_kind(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kFloat: return KV_F32;
    case at::kBFloat16: return KV_BF16;
    case at::kHalf: return KV_F16;
    case at::kChar: return KV_I8;
    case at::kFloat8_e4m3fn: return KV_E4M3;
    default: TORCH_CHECK(false, what, ": a cache holds float32, bfloat16, float16, int8 or float8_e4m3fn, not ", t);
  }
  return -1;
}

// Checks one half of a cache and describes it.
inline CacheView cache_view(const at::Tensor& c, const c10::optional<at::Tensor>& scale, const char* what) {
  TORCH_CHECK(c.dim() == 4, what, ": the cache must be [B, H, slots, d]");
  const int kind = cache_kind(c.scalar_type(), what);
  const int64_t size = c.element_size(), d = c.size(3);
  TORCH_CHECK(d % 8 == 0 && d >= 8 && d <= 256, what, ": head_dim must be a multiple of 8 from 8 to 256, not ", d);
  TB_CHECK_CUDA(c);
  TORCH_CHECK(c.size(2) >= 1 && c.size(2) < (1ll << 30), what, ": a cache has 1 to 2^30 slots");
  const int64_t al = std::min<int64_t>(16, 8 * size);
  TORCH_CHECK(c.stride(3) == 1 && c.stride(2) * size % al == 0 && c.stride(1) * size % al == 0 &&
                  c.stride(0) * size % al == 0 && (uintptr_t)c.data_ptr() % al == 0,
              what, ": cache rows must be contiguous and aligned to ", al, " bytes");
  CacheView v{};
  v.data = c.data_ptr();
  v.sb = c.stride(0);
  v.sh = c.stride(1);
  v.ss = c.stride(2);
  const bool scaled = kind == KV_I8 || kind == KV_E4M3;
  const bool given = scale.has_value() && scale->defined();
  TORCH_CHECK(scaled == given, what, scaled ? ": an 8-bit cache needs its scales" : ": only 8-bit caches have scales");
  if (given) {
    TORCH_CHECK(scale->device() == c.device() && scale->scalar_type() == at::kFloat && scale->dim() == 3 &&
                    scale->size(0) == c.size(0) && scale->size(1) == c.size(1) && scale->size(2) == c.size(2),
                what, ": scales must be fp32 [B, H, slots] on the cache's device");
    v.scale = scale->data_ptr<float>();
    v.qb = scale->stride(0);
    v.qh = scale->stride(1);
    v.qs = scale->stride(2);
  }
  return v;
}

}  // namespace tb
