// Device helpers of the attention kernels (gfx950): element types, MFMA products, and the
// place of a sequence's keys in memory.
#pragma once

#include <atomic>

#include "attn_internal.h"
#include "qlin_dev.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

namespace qlin {

constexpr float kNegInf = -__builtin_inff();

__device__ __forceinline__ uint32_t rfl32(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// Element types: fp32 pairs to a dword of two values (round to nearest even; EXACT: the values
// are whole numbers of at most 8 bits, which both types hold), and the MFMA products of 16-byte
// operands held as dwords.
struct Bf16 {
  static constexpr int DT = DT_BF16;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    return bitcast<uint32_t>(v2{(__bf16)a, (__bf16)b});
  }
  static __device__ __forceinline__ uint32_t pack_exact(float a, float b) {
    return perm(bitcast<uint32_t>(b), bitcast<uint32_t>(a), 0x07060302u);
  }
  static __device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bitcast<bf16x8>(a), bitcast<bf16x8>(b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(bitcast<bf16x8>(a), bitcast<bf16x8>(b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float get(uint16_t h) { return bf16_to_f32(h); }
};

struct F16 {
  static constexpr int DT = DT_F16;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return bitcast<uint32_t>(f16x2{(_Float16)a, (_Float16)b});
  }
  static __device__ __forceinline__ uint32_t pack_exact(float a, float b) {
    return bitcast<uint32_t>(__builtin_amdgcn_cvt_pkrtz(a, b));
  }
  static __device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(bitcast<f16x8>(a), bitcast<f16x8>(b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(bitcast<f16x8>(a), bitcast<f16x8>(b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float get(uint16_t h) { return (float)bitcast<_Float16>(h); }
};

// Keys of sequence b, clamped to what its row of the page table can hold.
__device__ __forceinline__ int kv_length(const KvSrc& kv, int b) {
  const long long most = (long long)kv.max_pages << kv.page_shift;
  const int n = kv.len[b];
  return n < 0 ? 0 : (long long)n > most ? (int)most : n;
}

// Inclusive prefix sum over a wave (rows of 16 by shifts, then across rows), without LDS.
template <typename N>
__device__ __forceinline__ N wave_scan(N v) {
  auto add = [&](auto ctrl, auto rows) {
    const int m = __builtin_amdgcn_update_dpp(0, bitcast<int>(v), decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
    v += bitcast<N>(m);
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});  // row_shr 1, 2, 4, 8
  add(integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
  add(integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
  add(integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
  add(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});  // row_bcast 15, 31
  add(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});
  return v;
}

// Inclusive prefix maximum of numbers that are not negative.
__device__ __forceinline__ int wave_scan_max(int v) {
  auto with = [&](auto ctrl, auto rows) {
    v = max(v, __builtin_amdgcn_update_dpp(0, v, decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
  };
  using std::integral_constant;
  with(integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});
  with(integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
  with(integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
  with(integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
  with(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});
  with(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});
  return v;
}

// Maximum over a wave, on every lane.
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, lane_xor<1>(v));
  v = fmaxf(v, lane_xor<2>(v));
  v = fmaxf(v, lane_xor<4>(v));
  v = fmaxf(v, lane_xor<8>(v));
  float x, y;
  lane_pair<16>(v, x, y);
  v = fmaxf(x, y);
  lane_pair<32>(v, x, y);
  return fmaxf(x, y);
}

// The value of one lane (a uniform number), the same on all.
template <typename N>
__device__ __forceinline__ N lane_value(N v, int at) {
  return bitcast<N>(__builtin_amdgcn_readlane(bitcast<int>(v), at));
}

// 2^x; of -inf (nothing seen yet, or scores of -inf alone) zero.
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// P = 2^(t - reference) of scores t, where P is an fp16 number for its product: 5 bits of exponent
// hold neither 2^16 nor, with all 11 bits of precision, less than 2^-14.  With the maximum so far as the
// reference, as 32-bit and bf16 numbers allow, many light keys beside a heavy one (25 octaves above
// them) would be rounded to multiples of 2^-24 or to zero, while the 32-bit sum of P has them.  So
// the reference follows the scores both ways: a block of keys whose largest score lies `lo` to `hi` above
// it (as powers of two) leaves it, any other moves it to `at` below that score.  A key as far as
// 14 + lo octaves below its block's largest keeps its precision, and what is lost of those further below
// is at most 2^-(25 + lo) of the block's largest P each.  The sums, of 32 bits, are rescaled with the
// reference; it stays where they are below 2^64, so that neither they nor the factors that join them
// leave 32 bits (keys 56 octaves lighter than the sum lose precision then).
__device__ __forceinline__ bool off_window(float d, float lo, float hi) {
  return fabsf(d - 0.5f * (lo + hi)) > 0.5f * (hi - lo);  // (no number: nothing seen yet on either side)
}
// The reference after a block of largest score `top`; l: the sum of P so far.
__device__ __forceinline__ float fp16_reference(float m, float top, float l, float lo, float at, float hi) {
  const float mn = off_window(top - m, lo, hi) && top != kNegInf ? top - at : m;
  return fmaxf(mn, m + __builtin_amdgcn_logf(l) - 64.0f);
}

// Lets a kernel take `bytes` of dynamic LDS on the current device; `done` holds a bit for each
// device where it may.
inline hipError_t allow_lds(const void* kernel, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return hipSuccess;
  e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

}  // namespace qlin
