// Attention of one new token per sequence over a paged key-value cache.
//
//   o[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - max),  j < len[b]
//
// Bound by the bytes of the cache: each key and value is read once for all query heads of its
// key head (up to 16 a launch unit; more take further units).  The keys of all sequences are
// cut into units of about the same number of 32-key blocks, so that a ragged batch fills the
// chip evenly; every workgroup finds its unit from the sequences' lengths on the device.
// 64 sequences of up to 16384 keys (4 key heads of 128 16-bit values, 1.01 GB) take 182 us, 5.5 TB/s,
// 8 of up to 8192 (2 of 256, 136 MB) 29 us, 4.6 TB/s, where a copy of 1 GiB reaches 5.1; one of
// 131072 int8 keys (136 MB) 33 us, 4.1 TB/s, with widening and joins; one of 1000 keys 9 us, the
// latency of lengths, pages, keys and joins one after the other.
//
// A workgroup's four waves take blocks in turn.  A block runs without LDS:
//   * scores: S^T = K Q^T on 16x16x32 MFMAs, K rows straight from memory as the A operand
//     (16 keys; a lane loads 16 bytes of one key), all query heads as the columns of B;
//   * P^T leaves the score layout as the B operand of O^T = V^T P^T without crossing lanes: lane
//     group g holds keys 4g .. 4g+3 and 16 + 4g .. 16 + 4g+3 of the block, and V's rows are
//     loaded in that order;
//   * V: a lane loads 8 keys' next hd/16 values; byte permutes pair the keys of a column, so
//     that column c of all lanes is an A operand of 16 value columns;
//   * int8: codes become 16-bit whole numbers (exact); a key's scale multiplies its scores in 32
//     bits, a value's scale its probability.
// The running maximum (the reference that P is taken against) is a column's, hence a lane's own.  P is rounded to 16 bits for its
// product (half a step of 2^-8 or 2^-11 of each term; the sum of P is of the unrounded); in fp16 it is
// taken against a reference that keeps a block's largest P between 2^4 and 2^15, as light keys would
// else leave fp16's range (fp16_reference).  With int8 values P times scale goes as the sum of two bf16
// numbers, which neither a small scale nor one heavy key can take precision from.
//
// Waves join through LDS, units of a sequence through memory: the last of 16 units to arrive
// adds their parts in unit order, the last of those groups adds the groups', so that the result
// does not depend on the order of arrival.  A group has 16 parts, or as many as it takes to keep a
// sequence's groups within its counters, and the last join one sum of each of up to 31 groups.
#include "attn_dev.h"

namespace qlin {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;

// Unit -> (sequence, part): all units of a (key head, group) numbered by sequence.
struct Unit {
  int b, s;       // sequence, its part
  int len;        // keys of the sequence
  int chunk;      // blocks of a part
  int parts;
  int base;       // number of part 0
};

__device__ __forceinline__ int blocks_of(int len) { return (len + kDecodeBlock - 1) / kDecodeBlock; }

__device__ __forceinline__ bool find_unit(const DecodeArgs& a, int u, Unit& r) {
  const int lane = (int)threadIdx.x & 63;
  auto mine = [&](int b0) { return b0 + lane < a.B ? kv_length(a.kv, b0 + lane) : 0; };
  const int first = mine(0);
  int chunk = 1 << 28;
  if (a.target > 0) {
    float total = 0.0f;  // (rounded up below; the same for all workgroups)
    for (int b0 = 0; b0 < a.B; b0 += 64) total += (float)blocks_of(b0 ? mine(b0) : first);
    total = lane_value(wave_scan(total), 63);
    // one workgroup a CU as long as that makes units of at most kDecodeLong blocks; longer work
    // goes to more of them, which come out more even and keep more loads in flight (8 sequences
    // of up to 8192 keys, 256 / 512 / 1024 units: 29 / 35 / 33 us; 64 of up to 16384, 256 / 768 /
    // 1536: 250 / 188 / 181)
    const float few = ceilf(total / (float)a.few);
    const float most = ceilf(total / (float)a.target);
    chunk = max((int)fminf(few <= (float)kDecodeLong ? few : fmaxf((float)kDecodeLong, most), 1e8f), 1);
    chunk = (chunk + kDecodeChunk - 1) / kDecodeChunk * kDecodeChunk;
  }
  int base = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int len = b0 ? mine(b0) : first;
    // an empty sequence has one part, which writes its zeros
    const int parts = b0 + lane < a.B ? max(1, (blocks_of(len) + chunk - 1) / chunk) : 0;
    const int end = wave_scan(parts), sum = lane_value(end, 63);
    if (u < base + sum) {
      const int at = __builtin_ctzll(__ballot(base + end > u));
      r.b = b0 + at;
      r.len = lane_value(len, at);
      r.parts = lane_value(parts, at);
      r.base = base + lane_value(end, at) - r.parts;
      r.s = u - r.base;
      r.chunk = chunk;
      return true;
    }
    base += sum;
  }
  return false;
}

// Dwords of codes that the compiler must not take apart before they are used (it would carry
// single bytes, a register each, around the loop).
__device__ __forceinline__ void opaque(uint32_t& a, uint32_t& b) { asm volatile("" : "+v"(a), "+v"(b)); }

// n values of a part, four at a time (float4 f of `rows * HD / 4`), and a row's maximum and sum
// behind them: a part's layout in memory.
template <int HD>
__device__ __forceinline__ unsigned part_ml(int rows) {
  return (unsigned)(rows * HD * 4);
}

template <typename T, int HD, bool Q8>
__global__ __launch_bounds__(kThreads, HD == 256 ? 2 : HD == 128 ? 3 : 4) void decode_kernel(const DecodeArgs a) {
  constexpr int STEPS = HD / 32;                 // score MFMAs of 16 keys
  constexpr int VW = HD >= 128 && !Q8 ? 8 : HD / 16;  // adjacent value columns of a lane
  constexpr int VC = HD / 16 / VW;               // runs of them, 16 VW columns apart
  constexpr int KL = Q8 ? HD / 64 : HD / 32;     // 16-byte loads of a key
  using TV = std::conditional_t<Q8, Bf16, T>;    // type of P and V in their product
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ int s_last;

  const int hg = a.HKV * a.gb;
  const int hh = (int)blockIdx.x % hg, unit = (int)blockIdx.x / hg;
  Unit U;
  if (!find_unit(a, unit, U)) return;
  for (int* x : {&U.b, &U.s, &U.len, &U.chunk, &U.parts, &U.base}) *x = (int)rfl32((uint32_t)*x);
  const int hk = hh % a.HKV, gi = hh / a.HKV;
  const int rows = min(16, a.G - 16 * gi);
  const int head0 = hk * a.G + 16 * gi;
  const int tid = (int)threadIdx.x;
  const int wave = (int)rfl32((uint32_t)tid >> 6), lane = tid & 63;
  const int j = lane & 15, g = lane >> 4;
  const uint16_t* q = (const uint16_t*)a.q + U.b * a.qb + head0 * a.qh;
  uint16_t* out = (uint16_t*)a.o + U.b * a.ob + head0 * a.oh;

  if (U.len == 0) {
    for (int f = tid; f < rows * (HD / 8); f += kThreads)
      *(u32x4*)(out + (f / (HD / 8)) * a.oh + (f % (HD / 8)) * 8) = u32x4{0, 0, 0, 0};
    return;
  }

  // query operand: column j = head j, the same hd order as a key's loads
  u32x4 qv[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int d = Q8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
    qv[s] = u32x4{0, 0, 0, 0};
    if (j < rows) qv[s] = ld_global<u32x4>(q + j * a.qh + d);
  }

  f32x4 O[VC * VW];
#pragma unroll
  for (int c = 0; c < VC * VW; ++c) O[c] = f32x4{0, 0, 0, 0};
  float m = kNegInf, l = 0.0f;
  bool bad = false;

  const int len = U.len;
  const int nblk = blocks_of(len);
  const int blk1 = (int)min((long long)nblk, (U.s + 1LL) * U.chunk);
  // (constant address space: page numbers come by scalar loads)
  const auto table = (const __attribute__((address_space(4))) int*)(a.kv.table + U.b * a.kv.table_stride);
  const uint32_t pmask = (1u << a.kv.page_shift) - 1u;
  constexpr int ES = Q8 ? 1 : 2;
  const uint32_t kst = (uint32_t)a.kv.k.st * ES, vst = (uint32_t)a.kv.v.st * ES;

  // A block's halves of 16 keys lie in one page each; keys behind the last are the last again.
  constexpr int VB = VW * ES;  // bytes of a run
  typedef std::conditional_t<VB == 16, u32x4, std::conditional_t<VB == 8, u32x2, uint32_t>> VReg;
  u32x4 kr[2][KL];
  VReg vr[8][VC];
  float sc = 0.0f;
  auto half_of = [&](int blk, int h) { return min(blk * kDecodeBlock + 16 * h, (len - 1) & ~15); };
  auto pages = [&](int blk, int (&pid)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) pid[h] = table[half_of(min(blk, nblk - 1), h) >> a.kv.page_shift];
  };
  auto valid = [&](int pid) {
    if ((unsigned)pid < (unsigned)a.kv.num_pages) return pid;
    bad = true;
    return 0;
  };
  auto base = [&](const PagedTensor& x, int hs, int pid) {
    return (const uint8_t*)x.p + ((uint64_t)(uint32_t)pid * (uint64_t)x.sp + ((uint32_t)hs & pmask) * (uint64_t)x.st +
                                  (uint64_t)hk * x.sh) * ES;
  };
  auto load_k = [&](int blk, const int (&pid)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int hs = half_of(blk, h);
      const uint8_t* p = base(a.kv.k, hs, valid(pid[h]));
      const uint32_t off = (uint32_t)min(j, len - 1 - hs) * kst + (uint32_t)g * 16u;
#pragma unroll
      for (int i = 0; i < KL; ++i) kr[h][i] = ld_global_nt<u32x4>(p + off + i * 64);
    }
    if constexpr (Q8) {
      // one scale a lane: the 32 keys', then the 32 values'
      const int h = (lane >> 4) & 1, hs = half_of(blk, h);
      const int r = min(j, len - 1 - hs), pc = h ? valid(pid[1]) : valid(pid[0]);
      const PagedTensor& x = lane < 32 ? a.kv.k : a.kv.v;
      const float* p = x.s + ((uint64_t)(uint32_t)pc * x.ssp + (uint64_t)((uint32_t)(hs & pmask) + r) * x.sst + (uint64_t)hk * x.ssh);
      sc = ld_global<float>(p);
    }
  };
  // value rows: slot s of lane group g is key 4g + s (s < 4) or 16 + 4g + s - 4
  auto load_v = [&](int blk, const int (&pid)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int hs = half_of(blk, h);
      const uint8_t* p = base(a.kv.v, hs, valid(pid[h]));
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint32_t off = (uint32_t)min(4 * g + s, len - 1 - hs) * vst + (uint32_t)j * VB;
#pragma unroll
        for (int c = 0; c < VC; ++c) vr[4 * h + s][c] = ld_global_nt<VReg>(p + off + c * 16 * VB);
      }
    }
  };

  // The next block's keys are loaded as soon as this one's are used, its values likewise, so that
  // a wave's loads are in flight while it computes.
  int blk = U.s * U.chunk + wave;
  int pid[2], pin[2];
  if (blk < blk1) {
    pages(blk, pid);
    load_k(blk, pid);
    load_v(blk, pid);
    pages(blk + kWaves, pin);
  }
  float* lsc = lds + wave * 64;
  for (; blk < blk1; blk += kWaves) {
    const bool more = blk + kWaves < blk1;
    f32x4 S[2];
    f32x4 ks[2], vs[2];
    if constexpr (Q8) {
      // a scale that is not finite makes no number of its key's score (an infinite one of a negative score
      // would leave its key out)
      uint64_t odd = __ballot(!(fabsf(sc) < __builtin_inff()));
      if (odd) {
        odd |= odd >> 32 | odd << 32;
        if (odd >> lane & 1) sc = lane < 32 ? __builtin_nanf("") : 0.0f;
      }
      // (a wave's LDS instructions take effect in order)
      lsc[lane] = sc;
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ks[h] = *(const f32x4*)(lsc + 16 * h + 4 * g);
        vs[h] = *(const f32x4*)(lsc + 32 + 16 * h + 4 * g);
      }
      __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      S[h] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        u32x4 kop;
        if constexpr (Q8) {
          const u32x4 r = kr[h][s / 2];
          const uint32_t w0 = s % 2 ? r.z : r.x, w1 = s % 2 ? r.w : r.y;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t w = e < 2 ? w0 : w1;
            const int c = 2 * (e % 2);
            asm volatile("" : "+v"(w));
            kop[e] = T::pack_exact((float)(int8_t)(w >> (8 * c)), (float)(int8_t)(w >> (8 * c + 8)));
          }
        } else {
          kop = kr[h][s];
        }
        if constexpr (Q8) __builtin_amdgcn_sched_barrier(0);
        S[h] = T::mma16(kop, qv[s], S[h]);
      }
    }
    if (more) load_k(blk + kWaves, pin);
    float t[8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) t[4 * h + i] = (Q8 ? S[h][i] * ks[h][i] : S[h][i]) * a.c;
    if (blk * kDecodeBlock + kDecodeBlock > len) {
      // (places behind the last key hold it again: its value may be infinite, which times zero is
      // no number)
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (blk * kDecodeBlock + 16 * (s / 4) + 4 * g + s % 4 >= len) {
          t[s] = kNegInf;
          if constexpr (Q8) vs[s / 4][s % 4] = 0.0f;
#pragma unroll
          for (int c = 0; c < VC; ++c) vr[s][c] = VReg{};
        }
    }
    float mx = t[0];
#pragma unroll
    for (int s = 1; s < 8; ++s) mx = fmaxf(mx, t[s]);
    const float top = group_max(mx);
    float mn = fmaxf(m, top);
    if constexpr (TV::DT == DT_F16) {
      mn = m;
      if (__any(off_window(top - m, 4.0f, 15.0f))) mn = fp16_reference(m, top, group_sum(l), 4.0f, 14.0f, 15.0f);
    }
    const float ms = mn == kNegInf ? 0.0f : mn;
    const float al = exp2_(m - ms);
    m = mn;
    float p[8], ps = 0.0f;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      p[s] = exp2_(t[s] - ms);
      ps += p[s];
    }
    l = l * al + ps;
    u32x4 pop[Q8 ? 2 : 1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (Q8) {
        const float p0 = p[2 * e] * vs[e / 2][2 * (e % 2)], p1 = p[2 * e + 1] * vs[e / 2][2 * (e % 2) + 1];
        const uint32_t w = TV::pack(p0, p1);
        pop[0][e] = w;
        pop[1][e] = TV::pack(p0 - bitcast<float>(w << 16), p1 - bitcast<float>(w & 0xFFFF0000u));
      } else {
        pop[0][e] = TV::pack(p[2 * e], p[2 * e + 1]);
      }
    }
    // (the rescaling is skipped while no row's reference moves)
    if (__any(al != 1.0f)) {
#pragma unroll
      for (int c = 0; c < VC * VW; ++c) O[c] *= al;
    }
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
      for (int x = 0; x < VW; ++x) {
        u32x4 vop;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t w0, w1;
          constexpr int PER = 4 / ES;  // columns of a dword
          if constexpr (VB == 4) {
            w0 = vr[2 * e][c];
            w1 = vr[2 * e + 1][c];
          } else {
            w0 = vr[2 * e][c][x / PER];
            w1 = vr[2 * e + 1][c][x / PER];
          }
          if constexpr (Q8) opaque(w0, w1);
          vop[e] = Q8 ? codes2<TV>(w0, w1, x % PER) : perm(w1, w0, x % 2 ? 0x07060302u : 0x05040100u);
        }
        // (left to itself the compiler widens every column first, and spills)
        if constexpr (Q8) __builtin_amdgcn_sched_barrier(0);
        f32x4& o = O[c * VW + x];
#pragma unroll
        for (int n = 0; n < (Q8 ? 2 : 1); ++n) o = TV::mma16(vop, pop[n], o);
      }
    if (more) {
      load_v(blk + kWaves, pin);
      pages(blk + 2 * kWaves, pin);
    }
  }
  if (bad) l = __builtin_nanf("");  // a page outside the cache: its sequence's output is NaN
  l = group_sum(l);

  if constexpr (Q8) __syncthreads();  // (the scales' place is taken again)
  // waves join in LDS: wave w's sums at w * rows * HD, maxima and sums of P behind all of them
  float* mlw = lds + kWaves * rows * HD;
  if (j < rows) {
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float* dst = lds + (wave * rows + j) * HD + c * 16 * VW + VW * (4 * g + i);
#pragma unroll
        for (int x = 0; x < VW; x += 4)
          *(f32x4*)(dst + x) = f32x4{O[c * VW + x][i], O[c * VW + x + 1][i], O[c * VW + x + 2][i], O[c * VW + x + 3][i]};
      }
    if (g == 0) {
      mlw[(wave * 16 + j) * 2] = m;
      mlw[(wave * 16 + j) * 2 + 1] = l;
    }
  }
  __syncthreads();

  const int nf = rows * (HD / 4);
  const unsigned slot_bytes = (unsigned)decode_slot_floats(min(16, a.G), HD) * 4u;
  const long long upart = (long long)hh * a.units + U.base;  // number of the sequence's first part
  const __amdgpu_buffer_rsrc_t rs = part_rsrc((const char*)a.part + upart * slot_bytes, (unsigned)U.parts * slot_bytes);
  auto store_out = [&](int f, f32x4 o, float ls) {
    const float inv = 1.0f / ls;
    const uint32_t lo = T::pack(o[0] * inv, o[1] * inv), hi = T::pack(o[2] * inv, o[3] * inv);
    *(u32x2*)(out + (f / (HD / 4)) * a.oh + (f % (HD / 4)) * 4) = u32x2{lo, hi};
  };
  auto store_part = [&](int part, int f, f32x4 o, float M, float ls) {
    const unsigned at = (unsigned)part * slot_bytes;
    st_coherent(o, rs, at + (unsigned)f * 16u);
    if (f % (HD / 4) == 0)
      st_coherent(f32x4{M, ls, 0, 0}, rs, at + part_ml<HD>(rows) + (unsigned)(f / (HD / 4)) * 16u);
  };

  for (int f = tid; f < nf; f += kThreads) {
    const int r = f / (HD / 4);
    float M = kNegInf;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, mlw[(w * 16 + r) * 2]);
    const float Ms = M == kNegInf ? 0.0f : M;
    f32x4 o = {0, 0, 0, 0};
    float ls = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float e = exp2_(mlw[(w * 16 + r) * 2] - Ms);
      const f32x4 x = *(const f32x4*)(lds + w * rows * HD + f * 4);
      o += x * e;
      ls += mlw[(w * 16 + r) * 2 + 1] * e;
    }
    if (U.parts == 1) store_out(f, o, ls);
    else store_part(U.s, f, o, M, ls);
  }
  if (U.parts == 1) return;

  // adds parts first, first + step, ... (n of them) in order
  auto join = [&](int first, int step, int n, auto&& put) {
    for (int f = tid; f < nf; f += kThreads) {
      const unsigned ml = part_ml<HD>(rows) + (unsigned)(f / (HD / 4)) * 16u;
      f32x4 o = {0, 0, 0, 0};
      float M = kNegInf, ls = 0.0f;
      constexpr int N = 8;  // parts in flight
      for (int i0 = 0; i0 < n; i0 += N) {
        f32x4 x[N];
        u32x2 y[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const unsigned at = (unsigned)(first + min(i0 + i, n - 1) * step) * slot_bytes;
          x[i] = bitcast<f32x4>(__builtin_amdgcn_raw_buffer_load_b128(rs, (unsigned)f * 16u, at, kCpolSc1));
          y[i] = __builtin_amdgcn_raw_buffer_load_b64(rs, ml, at, kCpolSc1);
        }
        // (no branch: the compiler would move each load behind it, next to its use, and wait for
        // every part by itself: 1000 keys 10.3 us against 8.8, 32768 of 128 values 27 against 17)
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const bool more = i0 + i < n;
          const float pm = more ? bitcast<float>(y[i].x) : kNegInf, pl = more ? bitcast<float>(y[i].y) : 0.0f;
          const f32x4 px = more ? x[i] : f32x4{0, 0, 0, 0};
          const float mn = fmaxf(M, pm);
          const float ms = mn == kNegInf ? 0.0f : mn;
          const float e0 = exp2_(M - ms), e1 = exp2_(pm - ms);
          o = o * e0 + px * e1;
          ls = ls * e0 + pl * e1;
          M = mn;
        }
      }
      put(f, o, M, ls);
    }
  };
  // whether this workgroup is the last of n at counter c (its stores done), which it then clears
  auto last_of = [&](unsigned* c, int n) {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    if (tid == 0) {
      const unsigned prev = __hip_atomic_fetch_add(c, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const int last = prev == (unsigned)(n - 1);
      if (last) __hip_atomic_store(c, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s_last = last;
    }
    __syncthreads();
    const bool r = s_last != 0;
    __syncthreads();
    return r;
  };

  unsigned* cnt = a.cnt + ((long long)U.b * hg + hh) * kDecodeCounters;
  // groups of 16 parts, or more where there would be more of them than counters
  const int per = max(kDecodeGroup, (U.parts + kDecodeCounters - 2) / (kDecodeCounters - 1));
  const int groups = (U.parts + per - 1) / per;
  const int gq = U.s / per;
  const int first = gq * per, members = min(per, U.parts - first);
  if (!last_of(cnt + 1 + gq, members)) return;
  if (groups == 1) {
    join(0, 1, members, [&](int f, f32x4 o, float, float ls) { store_out(f, o, ls); });
    return;
  }
  // a group's sum takes the place of its first part (read before by the same thread alone: the
  // maximum and sum behind a row's values are read by all of its threads, hence the barrier)
  {
    constexpr int MAXF = 16 * (HD / 4) / kThreads < 1 ? 1 : 16 * (HD / 4) / kThreads;
    f32x4 keep[MAXF];
    float km[MAXF], kl[MAXF];
    int at = 0;
    join(first, 1, members, [&](int, f32x4 o, float M, float ls) {
#pragma unroll
      for (int x = 0; x < MAXF; ++x)
        if (x == at) keep[x] = o, km[x] = M, kl[x] = ls;
      ++at;
    });
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
#pragma unroll
    for (int x = 0; x < MAXF; ++x) {
      const int f = tid + x * kThreads;
      if (f < nf) store_part(first, f, keep[x], km[x], kl[x]);
    }
  }
  if (!last_of(cnt, groups)) return;
  join(0, per, groups, [&](int f, f32x4 o, float, float ls) { store_out(f, o, ls); });
}

template <typename T, int HD, bool Q8>
hipError_t launch_q(const DecodeArgs& a, hipStream_t st) {
  const int rows = a.G < 16 ? a.G : 16;
  const size_t lds = ((size_t)kWaves * rows * HD + kWaves * 32) * sizeof(float);
  auto kern = decode_kernel<T, HD, Q8>;
  static std::atomic<uint64_t> done{0};
  const hipError_t e = allow_lds((const void*)kern, ((size_t)kWaves * 16 * HD + kWaves * 32) * sizeof(float), done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3((unsigned)(a.units * a.HKV * a.gb)), dim3(kThreads), lds, st, a);
  return hipGetLastError();
}

template <typename T, int HD>
hipError_t launch(const DecodeArgs& a, hipStream_t st) {
  return a.kv.k.s ? launch_q<T, HD, true>(a, st) : launch_q<T, HD, false>(a, st);
}

template <typename T>
hipError_t launch_hd(const DecodeArgs& a, int hd, hipStream_t st) {
  if (hd == 256) return launch<T, 256>(a, st);
  if (hd == 128) return launch<T, 128>(a, st);
  return launch<T, 64>(a, st);
}

}  // namespace

hipError_t launch_decode(const DecodeArgs& a, int dt, int hd, hipStream_t st) {
  return dt == DT_BF16 ? launch_hd<Bf16>(a, hd, st) : launch_hd<F16>(a, hd, st);
}

}  // namespace qlin
