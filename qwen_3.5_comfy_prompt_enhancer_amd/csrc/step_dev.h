// Device helpers of the kernels on vocabulary rows.
#pragma once

#include "qlin_dev.h"
#include "step_internal.h"

namespace qlin {

// Eight adjacent elements of a row at any element's address (rows of an odd number of tokens lie
// anywhere), as 32-bit numbers.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_any4 __attribute__((ext_vector_type(4), aligned(4)));

template <int DT>
struct Row8 {
  u32x4 r[DT == DT_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* row, long long i) {
    if constexpr (DT == DT_F32) {
      const auto p = (const __attribute__((address_space(1))) u32x4_any4*)((const float*)row + i);
      r[0] = p[0], r[1] = p[1];
    } else {
      r[0] = *(const __attribute__((address_space(1))) u32x4_any*)((const uint16_t*)row + i);
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (DT == DT_F32) return bitcast<float>(r[e / 4][e % 4]);
    const uint16_t h = (uint16_t)(r[0][e / 2] >> (16 * (e % 2)));
    if constexpr (DT == DT_BF16) return bf16_to_f32(h);
    return (float)bitcast<_Float16>(h);
  }
};

template <int DT>
__device__ __forceinline__ float load1(const void* row, long long i) {
  if constexpr (DT == DT_F32) return ((const float*)row)[i];
  const uint16_t h = ((const uint16_t*)row)[i];
  if constexpr (DT == DT_BF16) return bf16_to_f32(h);
  return (float)bitcast<_Float16>(h);
}

template <int DT>
__device__ __forceinline__ uint32_t round16(float v) {
  if constexpr (DT == DT_BF16) return f32_to_bf16(v);
  return bitcast<uint16_t>((_Float16)v);
}

template <int DT>
__device__ __forceinline__ void store1(void* row, long long i, float v) {
  if constexpr (DT == DT_F32) ((float*)row)[i] = v;
  else ((uint16_t*)row)[i] = (uint16_t)round16<DT>(v);
}

template <int DT>
__device__ __forceinline__ void store8(void* row, long long i, const float (&v)[8]) {
  if constexpr (DT == DT_F32) {
    const auto p = (__attribute__((address_space(1))) u32x4_any4*)((float*)row + i);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      p[h] = u32x4{bitcast<uint32_t>(v[4 * h]), bitcast<uint32_t>(v[4 * h + 1]), bitcast<uint32_t>(v[4 * h + 2]),
                   bitcast<uint32_t>(v[4 * h + 3])};
  } else {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = round16<DT>(v[2 * e]) | round16<DT>(v[2 * e + 1]) << 16;
    *(__attribute__((address_space(1))) u32x4_any*)((uint16_t*)row + i) = w;
  }
}

}  // namespace qlin
