// Queries, keys and values between the projections and attention: RMSNorm of every
// query and key head, rotary positions, keys and values into the paged cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * (w + 1 or w)                 per head of hd values
//   (y[i], y[i + r/2]) turned by pos[axis(i)] * freqs[i],  i < r/2; the rest unturned
//
// One workgroup per token: its threads first compute the token's r/2 cosines and sines
// into LDS (each is shared by every head), then teams of hd / 8 lanes take one head
// each, 8 values (16 bytes) per lane.  A pair's two values lie r/16 lanes apart.
// The angle is a 64-bit product reduced by whole turns before it becomes a float: in 32
// bits a position of 200000 would leave an error of 0.01 radians.  All else is 32 bits,
// rounded once, on the store; int8 codes are made of the unrounded values.
//
// Bound: bytes for long prompts (each value read and written once), a launch and two
// dependent memory round trips for a decode step.
#include "attn_internal.h"
#include "qlin_dev.h"

namespace qlin {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kMaxRot = 256;

__device__ __forceinline__ float ld16(const uint32_t w[4], int e, bool bf) {
  const uint16_t h = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
  return bf ? bf16_to_f32(h) : (float)bitcast<_Float16>(h);
}

__device__ __forceinline__ long long ld_index(const void* p, long long i, int is64) {
  return is64 ? ((const long long*)p)[i] : (long long)((const int*)p)[i];
}

// HD: head size, a team of HD / 8 lanes per head.
template <int HD>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(const RopeArgs a) {
  constexpr int TEAM = HD / 8;
  constexpr int TEAMS = kRopeThreads / TEAM;
  __shared__ float cs[kMaxRot / 2], sn[kMaxRot / 2];
  const int t = (int)blockIdx.x;
  const int tid = (int)threadIdx.x;
  const int half = a.rot / 2;
  const int l = tid % TEAM, team = tid / TEAM;
  const bool bf = a.dt == DT_BF16;

  for (int i = tid; i < half; i += kRopeThreads) {
    int ax;
    if (a.interleaved) {
      const int m = i % a.axes;
      ax = i < a.axes * a.sec[m] ? m : 0;
    } else {
      ax = (a.axes > 1 && i >= a.sec[0]) + (a.axes > 2 && i >= a.sec[0] + a.sec[1]);
    }
    const double p = (double)ld_index(a.pos, ax * a.pos_a + t * a.pos_t, a.pos64);
    const double f = a.freqs64 ? ((const double*)a.freqs)[i] : (double)((const float*)a.freqs)[i];
    const double u = p * f;
    // whole turns off in 64 bits (2 pi to 53 bits: the rest of a turn is off by |u| 2^-53)
    const double r = u - 6.283185307179586476925 * rint(u * 0.15915494309189533577);
    float s, c;
    sincosf((float)r, &s, &c);
    cs[i] = c;
    sn[i] = s;
  }
  __syncthreads();

  long long slot = -1;
  if (a.kc.p) {
    slot = ld_index(a.slots, t, a.slots64);
    if (slot >= a.nslots) slot = -1;  // out of the cache: not stored, as a negative slot
  }
  const long long page = slot >> a.page_shift, off = slot & ((1LL << a.page_shift) - 1);
  const int heads = a.HQ + a.HKV + (a.v ? a.HKV : 0);
  for (int h0 = 0; h0 < heads; h0 += TEAMS) {
    const int h = h0 + team;
    const bool there = h < heads;  // (all lanes take part in the shuffles)
    const int kind = h < a.HQ ? 0 : h < a.HQ + a.HKV ? 1 : 2;
    const int hh = kind == 0 ? h : kind == 1 ? h - a.HQ : h - a.HQ - a.HKV;
    const uint16_t* src = (const uint16_t*)(kind == 0 ? a.q : kind == 1 ? a.k : a.v);
    const long long so = kind == 0 ? t * a.qt + hh * a.qh : kind == 1 ? t * a.kt + hh * a.kh : t * a.vt + hh * a.vh;
    u32x4 raw = {0, 0, 0, 0};
    if (there) raw = ld_global<u32x4>(src + so + l * 8);
    const uint32_t rw[4] = {raw.x, raw.y, raw.z, raw.w};
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = ld16(rw, e, bf);
    if (kind != 2) {
      const void* w = kind == 0 ? a.qw : a.kw;
      if (w) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(y[e], y[e], ss);
#pragma unroll
        for (int m = TEAM / 2; m >= 1; m >>= 1) ss += __shfl_xor(ss, m, TEAM);
        const float inv = 1.0f / sqrtf(ss / (float)HD + a.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float wv = load_scale(w, a.wdt, l * 8 + e);
          y[e] = y[e] * inv * (a.one_plus ? wv + 1.0f : wv);
        }
      }
      // lanes [0, half/8) hold a pair's first value, [half/8, rot/8) its second
      const int hl = half / 8;
      const bool lo = l < hl, hi = !lo && l < 2 * hl;
      const int partner = lo ? l + hl : hi ? l - hl : l;
      const int i0 = (lo ? l : hi ? l - hl : 0) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float o = __shfl(y[e], partner, TEAM);
        if (lo || hi) {
          const float c = cs[i0 + e], s = sn[i0 + e];
          y[e] = lo ? y[e] * c - o * s : y[e] * c + o * s;
        }
      }
    }
    u32x4 res = raw;  // values pass as they are
    if (kind != 2) {
      uint32_t o4[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        o4[e] = (uint32_t)to_out16(y[2 * e], a.dt) | ((uint32_t)to_out16(y[2 * e + 1], a.dt) << 16);
      res = u32x4{o4[0], o4[1], o4[2], o4[3]};
    }
    if (there && kind == 0) *(u32x4*)((uint16_t*)a.qo + t * a.qot + hh * a.qoh + l * 8) = res;
    if (there && kind == 1 && a.ko) *(u32x4*)((uint16_t*)a.ko + t * a.kot + hh * a.koh + l * 8) = res;
    if (kind == 0 || !a.kc.p) continue;  // (uniform over a team)
    const PagedTensor& c = kind == 1 ? a.kc : a.vc;
    const long long at = page * c.sp + off * c.st + hh * c.sh;
    if (!c.s) {
      if (there && slot >= 0) *(u32x4*)((uint16_t*)c.p + at + l * 8) = res;
    } else {
      // the maximum over bit patterns keeps a NaN: its row's scale is NaN, and so is what is read
      uint32_t am = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) am = max(am, bitcast<uint32_t>(y[e]) & 0x7FFFFFFFu);
#pragma unroll
      for (int m = TEAM / 2; m >= 1; m >>= 1) am = max(am, (uint32_t)__shfl_xor((int)am, m, TEAM));
      const float amf = bitcast<float>(am);
      const float s = amf == amf ? fmaxf(amf / 127.0f, 1e-8f) : amf;
      uint32_t w[2] = {0u, 0u};
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e >> 2] |= ((uint32_t)round_i8(y[e] / s) & 0xFFu) << (8 * (e & 3));
      if (there && slot >= 0) {
        *(u32x2*)((int8_t*)c.p + at + l * 8) = u32x2{w[0], w[1]};
        if (l == 0) c.s[page * c.ssp + off * c.sst + hh * c.ssh] = s;
      }
    }
  }
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, hipStream_t st) {
  if (a.T <= 0) return hipSuccess;
  const dim3 grid((unsigned)a.T), block(kRopeThreads);
  if (a.hd == 256) hipLaunchKernelGGL(rope_kernel<256>, grid, block, 0, st, a);
  else if (a.hd == 128) hipLaunchKernelGGL(rope_kernel<128>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(rope_kernel<64>, grid, block, 0, st, a);
  return hipGetLastError();
}

}  // namespace qlin
