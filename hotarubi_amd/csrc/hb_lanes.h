// Small pieces that the serving operators' kernels share: four elements of the
// tensors' types, the largest of three, a fence of one wave.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace hb {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <class T>
struct Four;
template <>
struct Four<float> {
  typedef f32x4 type;
};
template <>
struct Four<__bf16> {
  typedef bf16x4 type;
};
template <>
struct Four<_Float16> {
  typedef f16x4 type;
};

// Largest of three (a NaN loses).
__device__ __forceinline__ float Max3(float a, float b, float c) {
  float y;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(y) : "v"(a), "v"(b), "v"(c));
  return y;
}

// Ends what the wave's LDS accesses before may still do.
__device__ __forceinline__ void WaveFence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

}  // namespace hb
