// Attention of one new token per sequence, of groups of sequences that share a prefix: the kernel
// template, included by attn_shared_bf16.hip and attn_shared_f16.hip.
//
//   o[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - max)
//   over the prefix's keys of the sequence's group and the sequence's own keys
//
// Bound by the bytes of the cache as long as a group's rows are few: a prefix's keys are read once
// for all rows (sequences x query heads) of a key head, up to 16 NT of them in a workgroup; groups of
// more rows take further workgroups over the same keys, and from a few hundred rows on the matrix
// units bound it.
//
// Work units are runs of 32-key blocks, of a prefix for a tile of whole sequences (NT columns of 16
// rows), or of one sequence's own keys; every workgroup finds its unit from the lengths on the device.
// The four waves of a workgroup take blocks in turn.  A block runs without LDS for its keys:
//   * scores: S^T = K Q^T on 16x16x32 MFMAs, K rows straight from memory as the A operand (16
//     keys; a lane loads 16 bytes of one key), rows as the columns of B, read from LDS;
//   * P^T leaves the score layout as the B operand of O^T = V^T P^T without crossing lanes: lane group
//     g holds keys 4g .. 4g+3 and 16 + 4g .. 16 + 4g+3 of the block, and V's rows are loaded in that order;
//   * V: a lane loads 8 keys' next hd/16 values; byte permutes pair the keys of a column, once for all
//     tiles of rows;
//   * int8: codes become 16-bit whole numbers (exact), once for all tiles; a key's scale multiplies its
//     scores in 32 bits, a value's its probability.
// The running maximum (the reference that P is taken against) is a column's, hence a lane's own.  P is
// rounded to 16 bits for its product (half a step of each term; the sum of P is of the unrounded), in fp16
// against a reference that follows the scores (fp16_reference); with int8 values P times scale goes as
// the sum of two bf16 numbers.  Sums, maxima and O are of 32 bits.
//
// Each unit leaves its rows' 32-bit sums; a second launch joins a row's parts in the order of its keys,
// the prefix's first, so that results do not depend on the order in which units end.
#pragma once

#include "attn_dev.h"

namespace qlin {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;

__device__ __forceinline__ int blocks_of(int len) { return (len + kSharedBlock - 1) / kSharedBlock; }

// Groups g0 + lane (none behind the last): first sequence, sequences, keys of the prefix.  Bounds are
// clamped to the sequences there are and taken as rising; `start`: the highest bound so far, for
// calls with rising g0.
struct Group {
  int b0, n, len;
};
__device__ __forceinline__ Group group_of(const SharedArgs& a, int g0, int& start) {
  const int g = g0 + ((int)threadIdx.x & 63);
  Group r = {0, 0, 0};
  int c0 = 0, c1 = 0;
  if (g < a.G) {
    c0 = min(max(a.cu[g], 0), a.B);
    c1 = min(max(a.cu[g + 1], 0), a.B);
    r.len = kv_length(a.pre, g);
  }
  r.b0 = max(wave_scan_max(c0), start);
  r.n = max(0, c1 - r.b0);
  start = lane_value(max(wave_scan_max(max(c0, c1)), start), 63);
  return r;
}

// What all workgroups make of the lengths: blocks of a unit, and the sequences of some group
// (lo .. hi - 1).
struct Plan {
  int chunk, lo, hi;
};
__device__ __forceinline__ int own_length(const SharedArgs& a, const Plan& p, int b) {
  return b >= p.lo && b < p.hi ? kv_length(a.own, b) : 0;
}
__device__ __forceinline__ int tiles_of(const SharedArgs& a, const Group& g) {
  return g.len > 0 ? (g.n + a.spt - 1) / a.spt : 0;
}
__device__ __forceinline__ int parts_of(const Plan& p, int len) { return (blocks_of(len) + p.chunk - 1) / p.chunk; }

__device__ __forceinline__ Plan make_plan(const SharedArgs& a) {
#pragma clang fp contract(off)  // (both launches have to make the same of them)
  const int lane = (int)threadIdx.x & 63;
  Plan p;
  p.lo = min(max(a.cu[0], 0), a.B);
  int start = 0;
  float total = 0.0f;  // (an estimate where it is large; the same for all workgroups)
  for (int g0 = 0; g0 < a.G; g0 += 64) {
    const Group g = group_of(a, g0, start);
    total += (float)tiles_of(a, g) * (float)blocks_of(g.len);
  }
  p.hi = max(start, p.lo);
  for (int b0 = p.lo; b0 < p.hi; b0 += 64) total += (float)blocks_of(own_length(a, p, b0 + lane));
  total = lane_value(wave_scan(total), 63);
  const float few = ceilf(total / (float)a.few), most = ceilf(total / (float)a.target);
  p.chunk = max((int)fminf(few <= (float)kSharedLong ? few : fmaxf((float)kSharedLong, most), 1e8f), 1);
  p.chunk = (p.chunk + kWaves - 1) / kWaves * kWaves;
  return p;
}

// A unit: rows of `n` sequences from b0 on, blocks blk0 .. blk1 - 1 of a prefix or of own keys.
struct Unit {
  int prefix;   // 1: of the prefix `src`, 0: of the own keys of sequence `src`
  int src, len;
  int b0, n;
  int blk0, blk1;
  int slot;     // number of its part among the prefix's, or the own ones
};

// Tiles of one part (t) lie 8 parts apart, so that they run on one XCD at about the same time: the
// first to load a key brings it to the others' L2.
__device__ __forceinline__ void part_tile(int i, int parts, int tiles, int& part, int& tile) {
  const int band = i / (8 * tiles), in = i - band * 8 * tiles;
  const int width = min(8, parts - 8 * band);
  tile = in / width;
  part = 8 * band + in % width;
}

__device__ __forceinline__ bool find_unit(const SharedArgs& a, const Plan& p, int u, Unit& r) {
  const int lane = (int)threadIdx.x & 63;
  int base = 0, start = 0;
  for (int g0 = 0; g0 < a.G; g0 += 64) {
    const Group g = group_of(a, g0, start);
    const int tiles = tiles_of(a, g), parts = parts_of(p, g.len);
    const int end = wave_scan(tiles * parts), sum = lane_value(end, 63);
    if (u < base + sum) {
      const int at = __builtin_ctzll(__ballot(base + end > u));
      const int nt = lane_value(tiles, at), np = lane_value(parts, at), first = base + lane_value(end, at) - nt * np;
      int part, tile;
      part_tile(u - first, np, nt, part, tile);
      r.prefix = 1;
      r.src = g0 + at;
      r.len = lane_value(g.len, at);
      r.b0 = lane_value(g.b0, at) + tile * a.spt;
      r.n = min(a.spt, lane_value(g.n, at) - tile * a.spt);
      r.blk0 = part * p.chunk;
      r.slot = first + tile * np + part;
      r.blk1 = min(blocks_of(r.len), r.blk0 + p.chunk);
      return true;
    }
    base += sum;
  }
  int own = 0;
  for (int b0 = p.lo; b0 < p.hi; b0 += 64) {
    const int len = own_length(a, p, b0 + lane);
    const int parts = parts_of(p, len);
    const int end = wave_scan(parts), sum = lane_value(end, 63);
    if (u < base + own + sum) {
      const int at = __builtin_ctzll(__ballot(base + own + end > u));
      r.prefix = 0;
      r.src = r.b0 = b0 + at;
      r.n = 1;
      r.len = lane_value(len, at);
      r.slot = u - base;
      r.blk0 = (u - base - own - lane_value(end, at) + lane_value(parts, at)) * p.chunk;
      r.blk1 = min(blocks_of(r.len), r.blk0 + p.chunk);
      return true;
    }
    own += sum;
  }
  return false;
}

__device__ __forceinline__ float group_max(float v) {  // over the four lanes of a column
  float x, y;
  lane_pair<16>(v, x, y);
  v = fmaxf(x, y);
  lane_pair<32>(v, x, y);
  return fmaxf(x, y);
}

__device__ __forceinline__ float group_sum(float v) {
  float x, y;
  lane_pair<16>(v, x, y);
  v = x + y;
  lane_pair<32>(v, x, y);
  return x + y;
}

// Dwords of codes that the compiler must not take apart before they are used (it would carry
// single bytes, a register each, around the loop).
__device__ __forceinline__ void opaque(uint32_t& a, uint32_t& b) { asm volatile("" : "+v"(a), "+v"(b)); }

// Codes of byte column c (0-3 of dword w) of two keys as a pair of 16-bit numbers.
template <typename T>
__device__ __forceinline__ uint32_t codes2(uint32_t w0, uint32_t w1, int c) {
  return T::pack_exact((float)(int8_t)(w0 >> (8 * c)), (float)(int8_t)(w1 >> (8 * c)));
}

// Dynamic LDS: the queries of NT tiles as operands; behind the loop the waves' sums of a tile.
template <int HD>
constexpr int shared_lds(int nt) {
  const int q = nt * (HD / 32) * 1024 + kWaves * 256, join = kWaves * 16 * HD * 4 + kWaves * 128;
  return q > join ? q : join;
}

// One unit: NT tiles of 16 rows.
template <typename T, int HD, bool Q8, int NT>
__device__ __forceinline__ void run_unit(const SharedArgs& a, const Unit& U, int hk, float* lds) {
  constexpr int STEPS = HD / 32;                 // score MFMAs of 16 keys
  constexpr int VW = HD >= 128 && !Q8 ? 8 : HD / 16;  // adjacent value columns of a lane
  constexpr int VC = HD / 16 / VW;               // runs of them, 16 VW columns apart
  constexpr int KL = Q8 ? HD / 64 : HD / 32;     // 16-byte loads of a key
  using TV = std::conditional_t<Q8, Bf16, T>;    // type of P and V in their product
  const int tid = (int)threadIdx.x;
  const int wave = (int)rfl32((uint32_t)tid >> 6), lane = tid & 63;
  const int j = lane & 15, g = lane >> 4;
  const KvSrc& kv = U.prefix ? a.pre : a.own;
  const int rows = U.n * a.R;

  // queries to LDS, as operands: step s of tile t at ((t STEPS + s) 64 + lane) 16 bytes, column j = row
  // 16 t + j, the same hd order as a key's loads
  for (int x = tid; x < NT * STEPS * 64; x += kThreads) {
    const int l = x & 63, s = (x >> 6) % STEPS, row = (x >> 6) / STEPS * 16 + (l & 15);
    const int d = Q8 ? 64 * (s / 2) + 16 * (l >> 4) + 8 * (s % 2) : 32 * s + 8 * (l >> 4);
    const int seq = row / a.R;
    u32x4 v = {0, 0, 0, 0};
    if (row < rows)
      v = ld_global<u32x4>((const uint16_t*)a.q + (U.b0 + seq) * a.qb + (hk * a.R + (row - seq * a.R)) * a.qh + d);
    *(u32x4*)(lds + x * 4) = v;
  }
  const f32x4* lq = (const f32x4*)lds + lane;

  f32x4 O[NT][VC * VW];
  float m[NT], l[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t] = kNegInf, l[t] = 0.0f;
#pragma unroll
    for (int c = 0; c < VC * VW; ++c) O[t][c] = f32x4{0, 0, 0, 0};
  }
  bool bad = false;

  const int len = U.len, nblk = blocks_of(len), blk1 = U.blk1;
  // (constant address space: page numbers come by scalar loads)
  const auto table = (const __attribute__((address_space(4))) int*)(kv.table + U.src * kv.table_stride);
  const uint32_t pmask = (1u << kv.page_shift) - 1u;
  constexpr int ES = Q8 ? 1 : 2;
  const uint32_t kst = (uint32_t)kv.k.st * ES, vst = (uint32_t)kv.v.st * ES;

  // A block's halves of 16 keys lie in one page each; keys behind the last are the last again.
  constexpr int VB = VW * ES;  // bytes of a run
  typedef std::conditional_t<VB == 16, u32x4, std::conditional_t<VB == 8, u32x2, uint32_t>> VReg;
  u32x4 kr[2][KL];
  VReg vr[8][VC];
  float sc = 0.0f;
  auto half_of = [&](int blk, int h) { return min(blk * kSharedBlock + 16 * h, (len - 1) & ~15); };
  auto pages = [&](int blk, int (&pid)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) pid[h] = table[half_of(min(blk, nblk - 1), h) >> kv.page_shift];
  };
  auto valid = [&](int pid) {
    if ((unsigned)pid < (unsigned)kv.num_pages) return pid;
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
      const uint8_t* p = base(kv.k, hs, valid(pid[h]));
      const uint32_t off = (uint32_t)min(j, len - 1 - hs) * kst + (uint32_t)g * 16u;
#pragma unroll
      for (int i = 0; i < KL; ++i) kr[h][i] = ld_global<u32x4>(p + off + i * 64);
    }
    if constexpr (Q8) {
      // one scale a lane: the 32 keys', then the 32 values'
      const int h = (lane >> 4) & 1, hs = half_of(blk, h);
      const int r = min(j, len - 1 - hs), pc = h ? valid(pid[1]) : valid(pid[0]);
      const PagedTensor& x = lane < 32 ? kv.k : kv.v;
      const float* p = x.s + ((uint64_t)(uint32_t)pc * x.ssp + (uint64_t)((uint32_t)(hs & pmask) + r) * x.sst + (uint64_t)hk * x.ssh);
      sc = ld_global<float>(p);
    }
  };
  // value rows: slot s of lane group g is key 4g + s (s < 4) or 16 + 4g + s - 4
  auto load_v = [&](int blk, const int (&pid)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int hs = half_of(blk, h);
      const uint8_t* p = base(kv.v, hs, valid(pid[h]));
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint32_t off = (uint32_t)min(4 * g + s, len - 1 - hs) * vst + (uint32_t)j * VB;
#pragma unroll
        for (int c = 0; c < VC; ++c) vr[4 * h + s][c] = ld_global<VReg>(p + off + c * 16 * VB);
      }
    }
  };

  // The next block's keys are loaded as soon as this one's are used, its values likewise, so that
  // a wave's loads are in flight while it computes.
  int blk = U.blk0 + wave;
  int pid[2], pin[2];
  if (blk < blk1) {
    pages(blk, pid);
    load_k(blk, pid);
    load_v(blk, pid);
    pages(blk + kWaves, pin);
  }
  __syncthreads();  // (the queries)
  float* lsc = lds + NT * STEPS * 256 + wave * 64;
  for (; blk < blk1; blk += kWaves) {
    const bool more = blk + kWaves < blk1;
    f32x4 S[NT][2];
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
    for (int t = 0; t < NT; ++t) S[t][0] = S[t][1] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      u32x4 qv[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) qv[t] = bitcast<u32x4>(lq[(t * STEPS + s) * 64]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
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
#pragma unroll
        for (int t = 0; t < NT; ++t) S[t][h] = T::mma16(kop, qv[t], S[t][h]);
      }
    }
    if (more) load_k(blk + kWaves, pin);
    const bool last = blk * kSharedBlock + kSharedBlock > len;
    if (last) {
      // (places behind the last key hold it again: its value may be infinite, which times zero is
      // no number)
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (blk * kSharedBlock + 16 * (s / 4) + 4 * g + s % 4 >= len) {
          if constexpr (Q8) vs[s / 4][s % 4] = 0.0f;
#pragma unroll
          for (int c = 0; c < VC; ++c) vr[s][c] = VReg{};
        }
    }
    u32x4 pop[NT][Q8 ? 2 : 1];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float x[8];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[4 * h + i] = (Q8 ? S[t][h][i] * ks[h][i] : S[t][h][i]) * a.c;
      if (last) {
#pragma unroll
        for (int s = 0; s < 8; ++s)
          if (blk * kSharedBlock + 16 * (s / 4) + 4 * g + s % 4 >= len) x[s] = kNegInf;
      }
      float mx = x[0];
#pragma unroll
      for (int s = 1; s < 8; ++s) mx = fmaxf(mx, x[s]);
      const float top = group_max(mx);
      float mn = fmaxf(m[t], top);
      if constexpr (TV::DT == DT_F16) {
        mn = m[t];
        if (__any(off_window(top - m[t], 4.0f, 15.0f)))
          mn = fp16_reference(m[t], top, group_sum(l[t]), 4.0f, 14.0f, 15.0f);
      }
      const float ms = mn == kNegInf ? 0.0f : mn;
      const float al = exp2_(m[t] - ms);
      m[t] = mn;
      float p[8], ps = 0.0f;
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        p[s] = exp2_(x[s] - ms);
        ps += p[s];
      }
      l[t] = l[t] * al + ps;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (Q8) {
          const float p0 = p[2 * e] * vs[e / 2][2 * (e % 2)], p1 = p[2 * e + 1] * vs[e / 2][2 * (e % 2) + 1];
          const uint32_t w = TV::pack(p0, p1);
          pop[t][0][e] = w;
          pop[t][1][e] = TV::pack(p0 - bitcast<float>(w << 16), p1 - bitcast<float>(w & 0xFFFF0000u));
        } else {
          pop[t][0][e] = TV::pack(p[2 * e], p[2 * e + 1]);
        }
      }
      // (the rescaling is skipped while no row's reference moves)
      if (__any(al != 1.0f)) {
#pragma unroll
        for (int c = 0; c < VC * VW; ++c) O[t][c] *= al;
      }
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
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int n = 0; n < (Q8 ? 2 : 1); ++n) O[t][c * VW + x] = TV::mma16(vop, pop[t][n], O[t][c * VW + x]);
      }
    if (more) {
      load_v(blk + kWaves, pin);
      pages(blk + 2 * kWaves, pin);
    }
  }
  if (bad) {  // a page outside the cache: outputs that see it are NaN
#pragma unroll
    for (int t = 0; t < NT; ++t) l[t] = __builtin_nanf("");
  }

  // waves join in LDS, tile by tile: wave w's sums at w 16 HD, references and sums of P behind all
  float* mlw = lds + kWaves * 16 * HD;
  const long long row0 = (long long)hk * a.rows + (U.prefix ? (long long)U.slot * (a.spt * a.R)
                                                            : a.own_rows + (long long)U.slot * a.R);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = min(16, rows - 16 * t);
    if (n <= 0) break;
    __syncthreads();
    const float ls = group_sum(l[t]);
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float* dst = lds + (wave * 16 + j) * HD + c * 16 * VW + VW * (4 * g + i);
#pragma unroll
        for (int x = 0; x < VW; x += 4)
          *(f32x4*)(dst + x) = f32x4{O[t][c * VW + x][i], O[t][c * VW + x + 1][i], O[t][c * VW + x + 2][i], O[t][c * VW + x + 3][i]};
      }
    if (g == 0) {
      mlw[(wave * 16 + j) * 2] = m[t];
      mlw[(wave * 16 + j) * 2 + 1] = ls;
    }
    __syncthreads();
    for (int f = tid; f < n * (HD / 4); f += kThreads) {
      const int r = f / (HD / 4);
      float M = kNegInf;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) M = fmaxf(M, mlw[(w * 16 + r) * 2]);
      const float Ms = M == kNegInf ? 0.0f : M;
      f32x4 o = {0, 0, 0, 0};
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float e = exp2_(mlw[(w * 16 + r) * 2] - Ms);
        const f32x4 x = *(const f32x4*)(lds + w * 16 * HD + f * 4);
        o += x * e;
        sum += mlw[(w * 16 + r) * 2 + 1] * e;
      }
      const long long row = row0 + 16 * t + r;
      *(f32x4*)(a.part + row * HD + (f % (HD / 4)) * 4) = o;
      if (f % (HD / 4) == 0) {
        a.ml[row * 2] = M;
        a.ml[row * 2 + 1] = sum;
      }
    }
  }
}

// Workgroups that a CU holds by registers.
constexpr int shared_occupancy(int hd, int nt) {
  return hd == 256 ? (nt == 1 ? 2 : 1) : hd == 128 ? (nt == 1 ? 3 : nt == 2 ? 2 : 1) : (nt <= 2 ? 3 : 2);
}

// NT: tiles of a prefix's unit, NO: of an own one.
template <typename T, int HD, bool Q8, int NT, int NO>
__global__ __launch_bounds__(kThreads, shared_occupancy(HD, NT)) void shared_kernel(const SharedArgs a) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int hk = (int)blockIdx.x % a.HKV, unit = (int)blockIdx.x / a.HKV;
  const Plan p = make_plan(a);
  Unit U;
  if (!find_unit(a, p, unit, U)) return;
  for (int* x : {&U.prefix, &U.src, &U.len, &U.b0, &U.n, &U.blk0, &U.blk1, &U.slot}) *x = (int)rfl32((uint32_t)*x);
  if (U.prefix) run_unit<T, HD, Q8, NT>(a, U, hk, lds);
  else run_unit<T, HD, Q8, NO>(a, U, hk, lds);
}

// A row (sequence, query head) a workgroup: its parts, the prefix's first, in turn over 1024 / HD
// slices of HD / 4 threads, whose sums meet in LDS.
template <typename T, int HD>
__global__ __launch_bounds__(kThreads) void shared_join_kernel(const SharedArgs a) {
  constexpr int LPR = HD / 4, SL = kThreads / LPR, N = 8;
  __shared__ __attribute__((aligned(16))) float so[SL * HD];
  __shared__ float sm[SL * 2];
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int hq = (int)blockIdx.x % (a.HKV * a.R), b = (int)blockIdx.x / (a.HKV * a.R);
  const int hk = hq / a.R, head = hq - hk * a.R;
  const Plan p = make_plan(a);
  if (b < p.lo || b >= p.hi) return;  // a row of no group
  // parts of the prefix: slots pslot, pslot + 1, ..., row prow of each
  int base = 0, start = 0, pslot = 0, np = 0, prow = 0;
  for (int g0 = 0; g0 < a.G; g0 += 64) {
    const Group g = group_of(a, g0, start);
    const int tiles = tiles_of(a, g), parts = parts_of(p, g.len);
    const int end = wave_scan(tiles * parts);
    const uint64_t mine = __ballot(b >= g.b0 && b < g.b0 + g.n);
    if (mine) {
      const int at = __builtin_ctzll(mine);
      const int nt = lane_value(tiles, at), in = b - lane_value(g.b0, at);
      np = nt ? lane_value(parts, at) : 0;
      pslot = base + lane_value(end, at) - nt * np + in / a.spt * np;
      prow = in % a.spt * a.R + head;
      break;
    }
    base += lane_value(end, 63);
  }
  int oslot = 0, no = 0;
  for (int b0 = p.lo; b0 < p.hi; b0 += 64) {
    const int parts = parts_of(p, own_length(a, p, b0 + lane));
    const int end = wave_scan(parts);
    if (b < b0 + 64) {
      no = lane_value(parts, b - b0);
      oslot += lane_value(end, b - b0) - no;
      break;
    }
    oslot += lane_value(end, 63);
  }
  const long long first = (long long)hk * a.rows;
  const long long pre0 = first + (long long)pslot * (a.spt * a.R) + prow;
  const long long own0 = first + a.own_rows + (long long)oslot * a.R + head;
  const int n = np + no;
  auto row_of = [&](int i) { return i < np ? pre0 + (long long)i * (a.spt * a.R) : own0 + (long long)(i - np) * a.R; };
  const int s = tid / LPR, f = tid % LPR;
  f32x4 o = {0, 0, 0, 0};
  float M = kNegInf, ls = 0.0f;
  for (int i0 = s; i0 < n; i0 += SL * N) {
    f32x4 x[N];
    float pm[N], pl[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const long long r = row_of(min(i0 + i * SL, n - 1));
      x[i] = ld_global<f32x4>(a.part + r * HD + f * 4);
      pm[i] = ld_global<float>(a.ml + r * 2);
      pl[i] = ld_global<float>(a.ml + r * 2 + 1);
    }
    // (no branch: the compiler would move each load behind it and wait for every part by itself)
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool more = i0 + i * SL < n;
      const float qm = more ? pm[i] : kNegInf, ql = more ? pl[i] : 0.0f;
      const f32x4 qx = more ? x[i] : f32x4{0, 0, 0, 0};
      const float mn = fmaxf(M, qm), ms = mn == kNegInf ? 0.0f : mn;
      const float e0 = exp2_(M - ms), e1 = exp2_(qm - ms);
      o = o * e0 + qx * e1;
      ls = ls * e0 + ql * e1;
      M = mn;
    }
  }
  *(f32x4*)(so + s * HD + f * 4) = o;
  if (f == 0) sm[s * 2] = M, sm[s * 2 + 1] = ls;
  __syncthreads();
  if (tid >= LPR) return;
  f32x4 r = {0, 0, 0, 0};
  float top = kNegInf, sum = 0.0f;
#pragma unroll
  for (int i = 0; i < SL; ++i) top = fmaxf(top, sm[i * 2]);
  const float ts = top == kNegInf ? 0.0f : top;
#pragma unroll
  for (int i = 0; i < SL; ++i) {
    const float e = exp2_(sm[i * 2] - ts);
    r += *(const f32x4*)(so + i * HD + tid * 4) * e;
    sum += sm[i * 2 + 1] * e;
  }
  const float inv = n == 0 ? 0.0f : 1.0f / sum;  // a sequence without keys: zeros
  *(u32x2*)((uint16_t*)a.o + b * a.ob + hq * a.oh + tid * 4) =
      u32x2{T::pack(r[0] * inv, r[1] * inv), T::pack(r[2] * inv, r[3] * inv)};
}

template <typename T, int HD, bool Q8, int NT, int NO>
hipError_t launch_nt(const SharedArgs& a, hipStream_t st) {
  auto kern = shared_kernel<T, HD, Q8, NT, NO>;
  constexpr size_t lds = shared_lds<HD>(NT > NO ? NT : NO);
  static std::atomic<uint64_t> done{0};
  hipError_t e = allow_lds((const void*)kern, lds, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3((unsigned)(a.units * a.HKV)), dim3(kThreads), lds, st, a);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  hipLaunchKernelGGL((shared_join_kernel<T, HD>), dim3((unsigned)(a.B * a.HKV * a.R)), dim3(kThreads), 0, st, a);
  return hipGetLastError();
}

template <typename T, int HD, bool Q8>
hipError_t launch_q(const SharedArgs& a, hipStream_t st) {
  if (a.R > 16) return launch_nt<T, HD, Q8, 4, 4>(a, st);
  if (a.tiles == 1) return launch_nt<T, HD, Q8, 1, 1>(a, st);
  if (a.tiles == 2) return launch_nt<T, HD, Q8, 2, 1>(a, st);
  return launch_nt<T, HD, Q8, 4, 1>(a, st);
}

template <typename T, int HD>
hipError_t launch_hd(const SharedArgs& a, hipStream_t st) {
  return a.own.k.s ? launch_q<T, HD, true>(a, st) : launch_q<T, HD, false>(a, st);
}

}  // namespace

template <typename T>
hipError_t launch_shared_t(const SharedArgs& a, int hd, hipStream_t st) {
  if (hd == 256) return launch_hd<T, 256>(a, st);
  if (hd == 128) return launch_hd<T, 128>(a, st);
  return launch_hd<T, 64>(a, st);
}

}  // namespace qlin
