// Device helpers shared by the token-model kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "token_ops.h"

namespace token_ops {

using bf16 = __bf16;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Vec16;              // one 16-byte access
template <> struct Vec16<float> { static constexpr int n = 4; };
template <> struct Vec16<bf16> { static constexpr int n = 8; };

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f(float v) {
  return (T)v;                                    // to nearest, ties to even
}

// N elements from p into floats: 16-byte accesses where N allows, which needs
// p aligned to them; N == 1 has no alignment need beyond the element's.
template <int N>
__device__ __forceinline__ void load_n(const float* p, float (&v)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f32x4 t = *reinterpret_cast<const f32x4*>(p + i);
      v[i] = t.x; v[i + 1] = t.y; v[i + 2] = t.z; v[i + 3] = t.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = p[i];
  }
}
template <int N>
__device__ __forceinline__ void load_n(const bf16* p, float (&v)[N]) {
  if constexpr (N % 8 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 8) {
      const u32x4 t = *reinterpret_cast<const u32x4*>(p + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[i + 2 * j] = __uint_as_float(t[j] << 16);
        v[i + 2 * j + 1] = __uint_as_float(t[j] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)p[i];
  }
}
template <int N>
__device__ __forceinline__ void store_n(float* p, const float (&v)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<f32x4*>(p + i) =
          f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = v[i];
  }
}
template <int N>
__device__ __forceinline__ void store_n(bf16* p, const float (&v)[N]) {
  if constexpr (N % 8 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 8) {
      bf16x8 t;
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = (bf16)v[i + j];
      *reinterpret_cast<bf16x8*>(p + i) = t;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = (bf16)v[i];
  }
}

__device__ __forceinline__ float scale_of(const Scale& s, long long g) {
  if (!s.num) return 1.f;
  if (!s.den) return s.num[g];
  // nothing counted: nothing to scale
  return s.den[g] == 0.f ? 0.f : s.num[g] / s.den[g];
}

// v * s, and 0 where v is 0: what nothing counted towards stays without a
// gradient under a factor that is not finite.
__device__ __forceinline__ float scaled(float v, float s) {
  return v == 0.f ? 0.f : v * s;
}

// Sum over groups of W neighbouring lanes (W a power of two up to 64); every
// lane gets it, in an order that does not depend on timing.
template <int W> __device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

}  // namespace token_ops
