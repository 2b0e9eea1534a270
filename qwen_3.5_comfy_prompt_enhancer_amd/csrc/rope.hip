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
// Bound: a launch and two dependent memory round trips for a decode step (4.8 us for one token of 8 + 2
// heads of 256 values); for long prompts the bytes (each value read and written once) and, about as
// much, the vector work of the angles and of int8 codes: 4097 tokens of 16 + 4 heads into an int8
// cache, 92 MB, in 25 us, 3.7 TB/s where a large copy reaches 5.1.
#include "attn_dev.h"

namespace qlin {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kMaxRot = 256;

template <typename T>
__device__ __forceinline__ float ld16(const uint32_t* w, int e) {
  return T::get((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
}

__device__ __forceinline__ long long ld_index(const void* p, long long i, int is64) {
  return is64 ? ((const long long*)p)[i] : (long long)((const int*)p)[i];
}

// One of three values (values: a choice between variables would put them in memory).
template <typename V>
__device__ __forceinline__ V pick(int kind, V a, V b, V c) {
  return kind == 0 ? a : kind == 1 ? b : c;
}

// Over an aligned team of TEAM lanes: the sum, the maximum of bit patterns, and the value of the
// lane `d` away on the other side of a pair (d a power of two: lanes l and l ^ d).
template <int TEAM>
__device__ __forceinline__ float team_sum(float v) {
  if constexpr (TEAM >= 32) {
    float a, b;
    lane_pair<16>(v, a, b);
    v = a + b;
  }
  if constexpr (TEAM >= 16) v += lane_xor<8>(v);
  v += lane_xor<4>(v);
  v += lane_xor<2>(v);
  return v + lane_xor<1>(v);
}

template <int TEAM>
__device__ __forceinline__ uint32_t team_max(uint32_t m) {
  auto with = [](uint32_t a, float b) { return max(a, bitcast<uint32_t>(b)); };
  if constexpr (TEAM >= 32) {
    float a, b;
    lane_pair<16>(bitcast<float>(m), a, b);
    m = with(bitcast<uint32_t>(a), b);
  }
  if constexpr (TEAM >= 16) m = with(m, lane_xor<8>(bitcast<float>(m)));
  m = with(m, lane_xor<4>(bitcast<float>(m)));
  m = with(m, lane_xor<2>(bitcast<float>(m)));
  return with(m, lane_xor<1>(bitcast<float>(m)));
}

// The other values of 8 pairs whose halves lie d lanes apart.
template <int TEAM>
__device__ __forceinline__ void swap_pairs(const float (&y)[8], float (&o)[8], int d, int partner) {
  auto all = [&](auto&& f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = f(y[e]);
  };
  if (d == 1) all([](float v) { return lane_xor<1>(v); });
  else if (d == 2) all([](float v) { return lane_xor<2>(v); });
  else if (d == 4) all([](float v) { return lane_xor<4>(v); });
  else if (d == 8) all([](float v) { return lane_xor<8>(v); });
  else all([&](float v) { return __shfl(v, partner, TEAM); });
}

// HD: head size, a team of HD / 8 lanes per head.  A thread's first kAheadItems heads are loaded
// before the angles are made, so that the two chains of memory round trips run side by side.
constexpr int kAheadItems = 3;

template <typename T, int HD, bool Q8>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(const RopeArgs a) {
  constexpr int TEAM = HD / 8;
  constexpr int TEAMS = kRopeThreads / TEAM;
  __shared__ __attribute__((aligned(16))) float cs[kMaxRot / 2], sn[kMaxRot / 2];
  const int t = (int)blockIdx.x;
  const int tid = (int)threadIdx.x;
  const int half = a.rot / 2;
  const int l = tid % TEAM, team = tid / TEAM;
  const int heads = a.HQ + a.HKV + (a.v ? a.HKV : 0);

  auto kind_of = [&](int h) { return h < a.HQ ? 0 : h < a.HQ + a.HKV ? 1 : 2; };
  // the token's rows (uniform), and a head's place in them: strides are below 2^32 bytes
  const uint8_t* qr = (const uint8_t*)a.q + (long long)t * a.qt * 2;
  const uint8_t* kr = (const uint8_t*)a.k + (long long)t * a.kt * 2;
  const uint8_t* vr = (const uint8_t*)a.v + (long long)t * a.vt * 2;
  const uint32_t qhs = (uint32_t)(a.qh * 2), khs = (uint32_t)(a.kh * 2), vhs = (uint32_t)(a.vh * 2);
  auto place = [&](const uint8_t* row, int head, uint32_t stride) {
    return (uint8_t*)row + (uint64_t)(uint32_t)head * stride + (uint32_t)l * 16u;
  };
  auto load = [&](int h) {
    const int kind = kind_of(h);
    const int hh = kind == 0 ? h : kind == 1 ? h - a.HQ : h - a.HQ - a.HKV;
    return ld_global<u32x4>(place(pick(kind, qr, kr, vr), hh, pick(kind, qhs, khs, vhs)));
  };
  u32x4 ahead[kAheadItems];
#pragma unroll
  for (int i = 0; i < kAheadItems; ++i) {
    ahead[i] = u32x4{0, 0, 0, 0};
    if (i * TEAMS + team < heads) ahead[i] = load(i * TEAMS + team);
  }
  long long slot = -1;
  if (a.kc.p) {
    const uint64_t v = (uint64_t)ld_index(a.slots, t, a.slots64);
    slot = (long long)((uint64_t)rfl32((uint32_t)(v >> 32)) << 32 | rfl32((uint32_t)v));  // (uniform)
    if (slot >= a.nslots) slot = -1;  // out of the cache: not stored, as a negative slot
  }

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

  // lanes [0, half/8) hold a pair's first value, [half/8, rot/8) its second
  const int hl = half / 8;
  const bool lo = l < hl, hi = !lo && l < 2 * hl;
  const int partner = lo ? l + hl : hi ? l - hl : l;
  const int i0 = (lo ? l : hi ? l - hl : 0) * 8;
  const long long page = slot >> a.page_shift, off = slot & ((1LL << a.page_shift) - 1);
  constexpr int ES = Q8 ? 1 : 2;
  uint8_t* kc = (uint8_t*)a.kc.p + (page * a.kc.sp + off * a.kc.st) * ES;
  uint8_t* vc = (uint8_t*)a.vc.p + (page * a.vc.sp + off * a.vc.st) * ES;
  float* kcs = Q8 ? a.kc.s + (page * a.kc.ssp + off * a.kc.sst) : nullptr;
  float* vcs = Q8 ? a.vc.s + (page * a.vc.ssp + off * a.vc.sst) : nullptr;
  uint8_t* qo = (uint8_t*)a.qo + (long long)t * a.qot * 2;
  uint8_t* ko = (uint8_t*)a.ko + (long long)t * a.kot * 2;
  const bool to_ko = a.ko != nullptr;
  const uint32_t qohs = (uint32_t)(a.qoh * 2), kohs = (uint32_t)(a.koh * 2);
  const uint32_t kchs = (uint32_t)(a.kc.sh * ES), vchs = (uint32_t)(a.vc.sh * ES);
  const uint32_t kcss = (uint32_t)a.kc.ssh, vcss = (uint32_t)a.vc.ssh;
  const void *qw = a.qw, *kw = a.kw;

  auto item = [&](int h, u32x4 raw) __attribute__((always_inline)) {
    if (h >= heads) return;  // (a team's lanes leave together, and exchange among themselves alone)
    const int kind = kind_of(h);
    const int hh = kind == 0 ? h : kind == 1 ? h - a.HQ : h - a.HQ - a.HKV;
    const uint32_t rw[4] = {raw.x, raw.y, raw.z, raw.w};
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = ld16<T>(rw, e);
    u32x4 res = raw;  // values pass as they are
    if (kind != 2) {
      const void* w = pick(kind, qw, kw, kw);
      if (w) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(y[e], y[e], ss);
        ss = team_sum<TEAM>(ss);
        const float inv = __builtin_amdgcn_rsqf(ss * (1.0f / HD) + a.eps);  // within 1 ulp
        float wv[8];
        if (a.wdt == DT_F32) {
          const f32x4 w0 = ld_global<f32x4>((const float*)w + l * 8), w1 = ld_global<f32x4>((const float*)w + l * 8 + 4);
#pragma unroll
          for (int e = 0; e < 8; ++e) wv[e] = e < 4 ? w0[e] : w1[e - 4];
        } else {
          const u32x4 w0 = ld_global<u32x4>((const uint16_t*)w + l * 8);
          const uint32_t wr[4] = {w0.x, w0.y, w0.z, w0.w};
          if (a.wdt == DT_BF16) {
#pragma unroll
            for (int e = 0; e < 8; ++e) wv[e] = ld16<Bf16>(wr, e);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) wv[e] = ld16<F16>(wr, e);
          }
        }
        const float one = a.one_plus ? 1.0f : 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = y[e] * inv * (wv[e] + one);
      }
      if (lo || hi) {
        float o[8];
        swap_pairs<TEAM>(y, o, hl, partner);
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const f32x4 c = *(const f32x4*)(cs + i0 + e), s = *(const f32x4*)(sn + i0 + e);
#pragma unroll
          for (int x = 0; x < 4; ++x) y[e + x] = fmaf(y[e + x], c[x], lo ? -o[e + x] * s[x] : o[e + x] * s[x]);
        }
      }
      res = u32x4{T::pack(y[0], y[1]), T::pack(y[2], y[3]), T::pack(y[4], y[5]), T::pack(y[6], y[7])};
      if (kind == 0) {
        *(u32x4*)place(qo, hh, qohs) = res;
        return;
      }
      if (to_ko) *(u32x4*)place(ko, hh, kohs) = res;
    }
    if (slot < 0) return;
    uint8_t* to = pick(kind, kc, kc, vc) + (uint64_t)(uint32_t)hh * pick(kind, kchs, kchs, vchs) +
                  (uint32_t)l * 8u * ES;
    if constexpr (!Q8) {
      *(u32x4*)to = res;
    } else {
      // the maximum over bit patterns keeps a NaN: its row's scale is NaN, and so is what is read
      uint32_t am = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) am = max(am, bitcast<uint32_t>(y[e]) & 0x7FFFFFFFu);
      const float amf = bitcast<float>(team_max<TEAM>(am));
      const float s = amf == amf ? fmaxf(amf / 127.0f, 1e-8f) : amf;
      const float inv = __builtin_amdgcn_rcpf(s);  // (quant_i8 divides where the product is near a tie)
      uint32_t q[2] = {0u, 0u};
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e >> 2] |= ((uint32_t)quant_i8(y[e], s, inv) & 0xFFu) << (8 * (e & 3));
      *(u32x2*)to = u32x2{q[0], q[1]};
      if (l == 0) pick(kind, kcs, kcs, vcs)[(uint64_t)(uint32_t)hh * pick(kind, kcss, kcss, vcss)] = s;
    }
  };
#pragma unroll
  for (int i = 0; i < kAheadItems; ++i)
    if (i * TEAMS < heads) item(i * TEAMS + team, ahead[i]);
  for (int h0 = kAheadItems * TEAMS; h0 < heads; h0 += TEAMS) {
    u32x4 raw = {0, 0, 0, 0};
    if (h0 + team < heads) raw = load(h0 + team);
    item(h0 + team, raw);
  }
}

template <typename T, int HD>
void go(const RopeArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.T), block(kRopeThreads);
  if (a.kc.s) hipLaunchKernelGGL((rope_kernel<T, HD, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((rope_kernel<T, HD, false>), grid, block, 0, st, a);
}

template <typename T>
void go_hd(const RopeArgs& a, hipStream_t st) {
  if (a.hd == 256) go<T, 256>(a, st);
  else if (a.hd == 128) go<T, 128>(a, st);
  else go<T, 64>(a, st);
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, hipStream_t st) {
  if (a.T <= 0) return hipSuccess;
  if (a.dt == DT_BF16) go_hd<Bf16>(a, st);
  else go_hd<F16>(a, st);
  return hipGetLastError();
}

}  // namespace qlin
