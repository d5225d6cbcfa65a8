// kvtypes.hpp -- the value types of the cache's kernels: fp16 and bf16, widened
// to fp32 and rounded from it (to nearest even), and OCP e4m3, rounded to.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace jasper_amd {

typedef _Float16 f16;
typedef __bf16 bf16;
struct e4m3 {
  uint8_t bits;
};

typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

// N consecutive values, loaded and stored whole.
template <typename T, int N>
struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void widen(const Pack<T, N>& p, float* out) {
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = (float)p.v[i];
}

// A stored e4m3 value saturates at +-448 (the type has no infinity); NaN stays.
__device__ __forceinline__ float clamp_e4m3(float x) {
  return x > 448.f ? 448.f : x < -448.f ? -448.f : x;
}

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> narrow(const float* x) {
  Pack<T, N> p;
  if constexpr (sizeof(T) == 1) {
    if constexpr (N == 1) {
      p.v[0].bits = (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(x[0]), 0.f, 0, false) & 0xFF);
    } else {
      uint32_t* w = reinterpret_cast<uint32_t*>(&p);
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        int b = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(x[4 * i]), clamp_e4m3(x[4 * i + 1]), 0, false);
        b = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(x[4 * i + 2]), clamp_e4m3(x[4 * i + 3]), b, true);
        w[i] = (uint32_t)b;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p.v[i] = (T)x[i];
  }
  return p;
}

}  // namespace jasper_amd
