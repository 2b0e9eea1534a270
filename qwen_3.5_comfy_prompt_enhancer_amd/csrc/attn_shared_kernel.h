// Attention of one new token per sequence, of groups of sequences that share a prefix: the kernel
// templates, included by attn_shared_{bf16,f16}.hip and, for many rows, attn_shared_wide_{bf16,f16}.hip.
//
//   o[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - max)
//   over the prefix's keys of the sequence's group and the sequence's own keys
//
// Bound by the bytes of the cache where prefixes are long and a group's rows (sequences x query heads of a key
// head) few: a prefix's keys are read once for all rows of a tile, further tiles over the same keys meet them in
// the L2.  8 sequences behind 100003 tokens of two key heads of 256 values: 45 us (4.5 TB/s), int8 42 us, bound by
// the vector instructions that widen values.  Where little is read, latency bounds it: 4 candidates of a prompt of
// 180 tokens 12.1 us, of which 2 go to finding a workgroup's unit, 3.6 to its first loads, 5 to the second launch.
//
// Work units are runs of 32-key blocks, of a prefix for a tile of whole sequences, or of one sequence's own keys;
// lengths are on the device alone, so every workgroup makes the same plan from them and finds its unit in it.
// Units come in two forms:
//   * thin (run_unit): one or two tiles of 16 rows.  The four waves of a workgroup take blocks in turn, whose keys
//     never pass through LDS:
//     - scores: S^T = K Q^T on 16x16x32 MFMAs, K rows straight from memory as the A operand (16 keys; a lane loads
//       16 bytes of one key), rows as the columns of B, read from LDS;
//     - P^T leaves the score layout as the B operand of O^T = V^T P^T without crossing lanes: lane group g holds
//       keys 4g .. 4g+3 and 16 + 4g .. 16 + 4g+3 of the block, and V's rows are loaded in that order;
//     - V: a lane loads 8 keys' next hd/16 values; byte permutes pair the keys of a column, once for all tiles;
//     - int8 keys stay whole numbers and meet the queries' digits where those hold them (see DIGITS); values become
//       16-bit whole numbers (exact), a key's scale multiplies its scores in 32 bits, a value's its probability.
//   * wide (wide_unit): 128 rows, 32 of each wave, over keys that land in LDS for all four.  64 sequences of 30 keys of their own
//     behind 16384 tokens, 32 query heads of 128 values to 4 key heads: 42 us, in tiles of 32 rows 54; of 1000 50 and 66.  int8
//     keys are written to LDS again as 16-bit numbers (a second barrier a block): 58 and 66 us, of 8 + 2 heads of 256 51 and 48,
//     where 16-bit ones take 33 and 52.
// The running maximum (the reference that P is taken against) is a column's, hence a lane's own.  P is
// rounded to 16 bits for its product (half a step of each term; the sum of P is of the unrounded), in fp16
// against a reference that follows the scores (fp16_reference); with int8 values P times scale goes as
// the sum of two bf16 numbers.  Sums, maxima and O are of 32 bits.
//
// Each unit leaves its rows' 32-bit sums; a second launch joins a row's parts in the order of its keys,
// the prefix's first, so that results do not depend on the order in which units end.  (The last unit of a sequence
// joining its parts took 12.9 us for the call of 12.0 above, and 21 instead of 12.2 behind 2000 tokens: one workgroup
// reads for a whole tile what the second launch reads with one for each row.)
#pragma once

#include "attn_prompt_kernel.h"

namespace qlin {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;

__device__ __forceinline__ int blocks_of(int len) { return (len + kSharedBlock - 1) / kSharedBlock; }

// Bounds and prefix length of group g0 + lane (none behind the last), and keys of sequence b0 + lane, as they are.
struct Lens {
  int c0, c1, len;
};
__device__ __forceinline__ Lens load_group(const SharedArgs& a, int g0) {
  const int g = g0 + ((int)threadIdx.x & 63);
  Lens r = {0, 0, 0};
  if (g < a.G) {
    r.c0 = a.cu[g];
    r.c1 = a.cu[g + 1];
    r.len = kv_length(a.pre, g);
  }
  return r;
}
__device__ __forceinline__ int load_own(const SharedArgs& a, int b0) {
  const int b = b0 + ((int)threadIdx.x & 63);
  return b < a.B ? kv_length(a.own, b) : 0;
}

// Groups g0 + lane: first sequence, sequences, keys of the prefix.  Bounds are clamped to the sequences there
// are and taken as rising; `start`: the highest bound so far, for calls with rising g0.
struct Group {
  int b0, n, len;
};
__device__ __forceinline__ Group group_of(const SharedArgs& a, const Lens& l, int& start) {
  const int c0 = min(max(l.c0, 0), a.B), c1 = min(max(l.c1, 0), a.B);
  Group r;
  r.b0 = max(wave_scan_max(c0), start);
  r.n = max(0, c1 - r.b0);
  r.len = l.len;
  start = lane_value(max(wave_scan_max(max(c0, c1)), start), 63);
  return r;
}

// What all workgroups make of the lengths: blocks of a unit, and the sequences of some group
// (lo .. hi - 1).  The first 64 groups' and sequences' lengths are read once, together.
struct Plan {
  int chunk, lo, hi;
  Lens groups;
  int own;
};
__device__ __forceinline__ Lens groups_at(const SharedArgs& a, const Plan& p, int g0) { return g0 ? load_group(a, g0) : p.groups; }
__device__ __forceinline__ int own_at(const SharedArgs& a, const Plan& p, int b0) {
  const int n = b0 ? load_own(a, b0) : p.own, b = b0 + ((int)threadIdx.x & 63);
  return b >= p.lo && b < p.hi ? n : 0;
}
__device__ __forceinline__ int tiles_of(const SharedArgs& a, const Group& g) {
  return g.len > 0 ? (g.n + a.spt - 1) / a.spt : 0;
}
__device__ __forceinline__ int parts_of(const Plan& p, int len) { return (blocks_of(len) + p.chunk - 1) / p.chunk; }

__device__ __forceinline__ Plan make_plan(const SharedArgs& a) {
#pragma clang fp contract(off)  // (both launches have to make the same of them)
  Plan p;
  p.groups = load_group(a, 0);
  p.own = load_own(a, 0);
  p.lo = min(max(lane_value(p.groups.c0, 0), 0), a.B);
  int start = 0;
  float total = 0.0f;  // (an estimate where it is large; the same for all workgroups)
  for (int g0 = 0; g0 < a.G; g0 += 64) {
    const Group g = group_of(a, groups_at(a, p, g0), start);
    total += (float)tiles_of(a, g) * (float)blocks_of(g.len);
  }
  p.hi = max(start, p.lo);
  for (int b0 = 0; b0 < p.hi; b0 += 64) total += (float)blocks_of(own_at(a, p, b0));
  total = lane_value(wave_scan(total), 63);
  const float few = ceilf(total / (float)a.few), most = ceilf(total / (float)a.target);
  p.chunk = max((int)fminf(few <= (float)a.brief ? few : fmaxf((float)a.brief, most), 1e8f), 1);
  p.chunk = (p.chunk + kWaves - 1) / kWaves * kWaves;
  return p;
}

// A unit: rows of `n` sequences from b0 on, blocks blk0 .. blk1 - 1 of a prefix or of own keys.
struct Unit {
  int prefix;   // 1: of the prefix `src`, 0: of the own keys of sequence `src`
  int src, len;
  int b0, n;
  int blk0, blk1;
  int row;      // of its key head's: the first one of its sums
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
  int base = 0, start = 0, rows = 0;
  for (int g0 = 0; g0 < a.G; g0 += 64) {
    const Group g = group_of(a, groups_at(a, p, g0), start);
    const int tiles = tiles_of(a, g), parts = parts_of(p, g.len);
    const int end = wave_scan(tiles * parts), sum = lane_value(end, 63);
    const int sums = wave_scan(parts * g.n);
    if (u < base + sum) {
      const int at = __builtin_ctzll(__ballot(base + end > u));
      const int n = lane_value(g.n, at), nt = lane_value(tiles, at), np = lane_value(parts, at);
      const int first = base + lane_value(end, at) - nt * np;
      int part, tile;
      part_tile(u - first, np, nt, part, tile);
      r.prefix = 1;
      r.src = g0 + at;
      r.len = lane_value(g.len, at);
      r.b0 = lane_value(g.b0, at) + tile * a.spt;
      r.n = min(a.spt, n - tile * a.spt);
      r.blk0 = part * p.chunk;
      r.row = (rows + lane_value(sums, at) + (part - np) * n + tile * a.spt) * a.R;
      r.blk1 = min(blocks_of(r.len), r.blk0 + p.chunk);
      return true;
    }
    base += sum;
    rows += lane_value(sums, 63);
  }
  int own = 0;
  for (int b0 = 0; b0 < p.hi; b0 += 64) {
    const int len = own_at(a, p, b0);
    const int parts = parts_of(p, len);
    const int end = wave_scan(parts), sum = lane_value(end, 63);
    if (u < base + own + sum) {
      const int at = __builtin_ctzll(__ballot(base + own + end > u));
      r.prefix = 0;
      r.src = r.b0 = b0 + at;
      r.n = 1;
      r.len = lane_value(len, at);
      r.row = (int)a.own_rows + (u - base) * a.R;
      r.blk0 = (u - base - own - lane_value(end, at) + lane_value(parts, at)) * p.chunk;
      r.blk1 = min(blocks_of(r.len), r.blk0 + p.chunk);
      return true;
    }
    own += sum;
  }
  return false;
}

// Dwords of codes that the compiler must not take apart before they are used (it would carry
// single bytes, a register each, around the loop).
__device__ __forceinline__ void opaque(uint32_t& a) { asm volatile("" : "+v"(a)); }
__device__ __forceinline__ void opaque(u32x2& a) { asm volatile("" : "+v"(a)); }
__device__ __forceinline__ void opaque(u32x4& a) { asm volatile("" : "+v"(a)); }

// int8 keys: a query is the sum of three int8 digits, q = 2^(E - 5) (d0 + d1 / 2^8 + d2 / 2^16) where the row's largest
// value lies from 2^E to 2^(E + 1).  The products with codes are then whole numbers of the matrix units, added up
// exactly, and no code is widened (8 sequences behind 100003 keys of 256 values: 41.4 us, as 16-bit numbers 44.8).
// That holds a bf16 value exactly down to 2^(E - 14), an fp16 one to 2^(E - 11), where most rows have nothing or little
// below; of smaller values it leaves out up to half of 2^(E - 21).  What a row's digits leave out, summed over its
// values, times the largest code and a key's scale, bounds how far off a score is.  A block where a key's score could be
// off by more than 2^-16 (in powers of two: as much as P loses as two bf16 numbers) takes its codes as 16-bit numbers and
// the queries as they are: rows of very different values, whose large ones may meet codes of zero.
constexpr int DIGITS = 3;
constexpr float kLeftOut = 0x1p-16f;

// Dynamic LDS: the queries of NT tiles as operands (int8 keys: digits, and as they are); behind the loop the waves' sums of
// a tile.
template <int HD>
constexpr int shared_lds(int nt, bool q8) {
  const int q = nt * ((q8 ? DIGITS * (HD / 64) : 0) + HD / 32) * 1024 + nt * 128 + kWaves * 256, join = kWaves * 16 * (HD + 4) * 4 + kWaves * 128;
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

  // queries, column j = row 16 t + j: loaded in front of the first block, written to LDS as operands behind its loads
  constexpr int QL = (NT * STEPS + kWaves - 1) / kWaves;
  u32x4 qr[QL];
  auto q_at = [&](int i, int& row, int& s, int& l) {
    const int x = i * kThreads + tid;
    l = x & 63, s = (x >> 6) % STEPS, row = (x >> 6) / STEPS * 16 + (l & 15);
    return x < NT * STEPS * 64;
  };
#pragma unroll
  for (int i = 0; i < QL; ++i) {
    int row, s, l;
    const bool some = q_at(i, row, s, l);
    const int d = Q8 ? 64 * (s / 2) + 16 * (l >> 4) + 8 * (s % 2) : 32 * s + 8 * (l >> 4);
    const int seq = row / a.R;
    qr[i] = u32x4{0, 0, 0, 0};
    if (some && row < rows)
      qr[i] = ld_global<u32x4>((const uint16_t*)a.q + (U.b0 + seq) * a.qb + (hk * a.R + (row - seq * a.R)) * a.qh + d);
  }
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
  __builtin_amdgcn_sched_barrier(0);
  constexpr int DF = Q8 ? NT * DIGITS * KL * 256 : 0;  // floats of the digits,
  constexpr int QF = DF + NT * STEPS * 256;            // and of the operands
  float qscale[NT], left_out = 0.0f;
  // step s of tile t at ((t STEPS + s) 64 + lane) 16 bytes behind the digits
#pragma unroll
  for (int i = 0; i < QL; ++i)
    if (i * kThreads + tid < NT * STEPS * 64) *(u32x4*)(lds + DF + (i * kThreads + tid) * 4) = qr[i];
  if constexpr (Q8) {
    // digit n of 64 values i of tile t at (((t DIGITS + n) KL + i) 64 + lane) 16 bytes
    constexpr uint32_t LEAST = 21;  // (exponent of 2^-106: 2^21 over it is a number)
    uint32_t* most = (uint32_t*)(lds + QF);  // the rows' largest, as bits
    uint32_t* lost = most + NT * 16;         // what their digits leave out, in 2^-8 of the last one's unit
    if (tid < NT * 32) most[tid] = 0u;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < QL; ++i) {
      int row, s, l;
      if (!q_at(i, row, s, l)) continue;
      uint32_t top = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, bitcast<uint32_t>(T::get((uint16_t)(qr[i][e / 2] >> (16 * (e % 2))))) & 0x7FFFFFFFu);
      atomicMax(most + row, top);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < QL; ++i) {
      int row, s, l;
      if (!q_at(i, row, s, l)) continue;
      // to whole numbers of at most 2^22
      const float to = bitcast<float>((275u - max(most[row] >> 23, LEAST)) << 23);
      uint32_t w[DIGITS][2] = {};
      float rest = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = fminf(fmaxf(T::get((uint16_t)(qr[i][e / 2] >> (16 * (e % 2)))) * to, -0x1p22f), 0x1p22f);
        const float whole = rintf(x);
        rest += fabsf(x - whole);
        // bytes of the number with 128 added to the lower two, and taken off again
        const uint32_t d = ((uint32_t)(int)whole + 0x8080u) ^ 0x8080u;
#pragma unroll
        for (int n = 0; n < DIGITS; ++n) w[n][e / 4] |= (d >> (8 * (DIGITS - 1 - n)) & 0xFFu) << (8 * (e % 4));
      }
      if (rest > 0.0f) atomicAdd(lost + row, (uint32_t)ceilf(rest * 256.0f));
      const int t = row / 16;
#pragma unroll
      for (int n = 0; n < DIGITS; ++n)
        *(u32x2*)((uint32_t*)lds + (((t * DIGITS + n) * KL + s / 2) * 64 + l) * 4 + 2 * (s % 2)) = u32x2{w[n][0], w[n][1]};
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint32_t exponent = most[16 * t + j] >> 23;
      // (a query that is not finite makes numbers of no score)
      const float unit = bitcast<float>((max(exponent, LEAST) - 5u) << 23) * a.c;
      qscale[t] = exponent < 255u ? unit : __builtin_nanf("");
      if (exponent < 255u) left_out = fmaxf(left_out, (float)lost[16 * t + j] * (128.0f * 0x1p-24f) * unit);
    }
    left_out = wave_max(left_out);
  }
  __syncthreads();
  const f32x4* lq = (const f32x4*)(lds + DF) + lane;
  float* lsc = lds + QF + NT * 32 + wave * 64;
  for (; blk < blk1; blk += kWaves) {
    const bool more = blk + kWaves < blk1;
    f32x4 S[NT][2];
    f32x4 ks[2], vs[2];
    bool exact = false;
    if constexpr (Q8) {
      // a scale that is not finite makes no number of its key's score (an infinite one of a negative score
      // would leave its key out)
      uint64_t odd = __ballot(!(fabsf(sc) < __builtin_inff()));
      if (odd) {
        odd |= odd >> 32 | odd << 32;
        if (odd >> lane & 1) sc = lane < 32 ? __builtin_nanf("") : 0.0f;
      }
      exact = __any(lane < 32 && fabsf(sc) * left_out > kLeftOut);
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
    if (Q8 && !exact) {
      // the codes as they are, times each digit of the queries: whole numbers
      const u32x4* lw = (const u32x4*)lds + lane;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          i32x4 D[DIGITS];
#pragma unroll
          for (int n = 0; n < DIGITS; ++n) {
            D[n] = i32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < KL; ++i)
              D[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bitcast<i32x4>(kr[h][i]), bitcast<i32x4>(lw[((t * DIGITS + n) * KL + i) * 64]), D[n], 0, 0, 0);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
            S[t][h][e] = fmaf(fmaf((float)D[2][e], 0x1p-8f, (float)D[1][e]), 0x1p-8f, (float)D[0][e]) * ks[h][e];
        }
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t) S[t][0] = S[t][1] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        u32x4 qv[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) qv[t] = bitcast<u32x4>(lq[(t * STEPS + s) * 64]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u32x4 k;
          if constexpr (Q8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t w = kr[h][s / 2][2 * (s % 2) + e / 2] >> (16 * (e % 2));
              k[e] = T::pack_exact((float)(int8_t)w, (float)(int8_t)(w >> 8));
            }
          } else {
            k = kr[h][s];
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) S[t][h] = T::mma16(k, qv[t], S[t][h]);
        }
      }
      if constexpr (Q8) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) S[t][h] *= ks[h];
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
      float cs = a.c;
      if constexpr (Q8) cs = exact && qscale[t] == qscale[t] ? a.c : qscale[t];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[4 * h + i] = S[t][h][i] * cs;
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
    if constexpr (Q8) {
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int c = 0; c < VC; ++c) opaque(vr[r][c]);
    }
    // value column y of the lane's VC VW: its 8 keys
    auto v_op = [&](int y) {
      const int c = y / VW, x = y % VW;
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
        vop[e] = Q8 ? codes2<TV>(w0, w1, x % PER) : perm(w1, w0, x % 2 ? 0x07060302u : 0x05040100u);
      }
      return vop;
    };
    u32x4 vop;
    if constexpr (Q8) vop = v_op(0);
#pragma unroll
    for (int y = 0; y < VC * VW; ++y) {
      const u32x4 now = Q8 ? vop : v_op(y);
      if constexpr (Q8) {
        if (y + 1 < VC * VW) vop = v_op(y + 1);
        __builtin_amdgcn_sched_barrier(0);  // (left to itself the compiler widens every column first, and spills)
      }
#pragma unroll
      for (int n = 0; n < (Q8 ? 2 : 1); ++n)
#pragma unroll
        for (int t = 0; t < NT; ++t) O[t][y] = TV::mma16(now, pop[t][n], O[t][y]);
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
  // (rows HD + 4 apart: the 16 of a tile start in different banks; HD apart the stores took 3 us more)
  constexpr int ST = HD + 4;
  float* mlw = lds + kWaves * 16 * ST;
  const long long row0 = (long long)hk * a.rows + U.row;
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
        float* dst = lds + (wave * 16 + j) * ST + c * 16 * VW + VW * (4 * g + i);
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
        const f32x4 x = *(const f32x4*)(lds + (w * 16 + r) * ST + (f % (HD / 4)) * 4);
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

// One unit of many rows: a tile of 128, 32 to a wave, over keys that land in LDS for all four waves (as
// prompt_kernel's: a ring of two blocks by 16-byte LDS DMA, 32x32x16 MFMAs with Q and O in registers, a lane
// half a row).
template <typename T, int HD, bool Q8>
__device__ __forceinline__ void wide_unit(const SharedArgs& a, const Unit& U, int hk, uint32_t lds0) {
  using G = PGeo<HD>;
  using TV = std::conditional_t<Q8, Bf16, T>;  // type of P and V in their product
  constexpr int PN = Q8 ? 2 : 1;               // P x scale as two bf16 numbers
  constexpr int ES = Q8 ? 1 : 2;
  const int tid = (int)threadIdx.x;
  const int wave = (int)rfl32((uint32_t)tid >> 6), lane = tid & 63;
  const int col = lane & 31, h = lane >> 5;
  const KvSrc& kv = U.prefix ? a.pre : a.own;
  const int rows = U.n * a.R, R0 = wave * 32, row = R0 + col;
  const int kb0 = U.blk0, kb1 = U.blk1, nk = U.len;
  u32x4 Q[G::NS];
  {
    const int seq = row / a.R;
    const uint16_t* q = (const uint16_t*)a.q + (U.b0 + min(seq, U.n - 1)) * a.qb + (hk * a.R + (row - seq * a.R)) * a.qh + 8 * h;
#pragma unroll
    for (int s = 0; s < G::NS; ++s) Q[s] = ld_global<u32x4>(q + 16 * s);
  }
  f32x16 O[G::ND];
  float m = kNegInf, l = 0.0f;
#pragma unroll
  for (int d = 0; d < G::ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) O[d][i] = 0.0f;

  const int* table = kv.table + U.src * kv.table_stride;
  // whether a page of the unit's keys lies outside the cache: looked at by every wave (each fetches a quarter
  // of the keys that all of them use)
  bool any_bad = false;
  {
    const int e1 = (min(kb1 * G::KB, nk) - 1) >> kv.page_shift;
    for (int e = (kb0 * G::KB) >> kv.page_shift; e <= e1; e += 64)
      any_bad |= (unsigned)table[min(e + lane, e1)] >= (unsigned)kv.num_pages;
    any_bad = __any(any_bad);
  }
  // this wave's 8 keys of a block: the first one's place (keys behind the last are the last)
  auto key8_of = [&](int kb) { return min(min(kb, kb1 - 1) * G::KB + 8 * wave, (nk - 1) & ~7); };
  // (a scalar load: a vector one's wait would also wait for the copies in flight)
  auto page_of = [&](int kb) {
    return ((const __attribute__((address_space(4))) int*)table)[key8_of(kb) >> kv.page_shift];
  };
  struct Place {
    const uint8_t* p;
    uint32_t sp, st;
  };
  const Place kpl = {(const uint8_t*)kv.k.p + hk * kv.k.sh * ES, (uint32_t)kv.k.sp * ES, (uint32_t)kv.k.st * ES};
  const Place vpl = {(const uint8_t*)kv.v.p + hk * kv.v.sh * ES, (uint32_t)kv.v.sp * ES, (uint32_t)kv.v.st * ES};
  const Place kspl = {(const uint8_t*)(kv.k.s + hk * kv.k.ssh), (uint32_t)kv.k.ssp * 4u, (uint32_t)kv.k.sst * 4u};
  const Place vspl = {(const uint8_t*)(kv.v.s + hk * kv.v.ssh), (uint32_t)kv.v.ssp * 4u, (uint32_t)kv.v.sst * 4u};
  const uint32_t pmask = (1u << kv.page_shift) - 1u;
  auto base_of = [&](const Place& x, int key, int pid) {
    return x.p + ((uint64_t)(uint32_t)pid * x.sp + (uint64_t)((uint32_t)key & pmask) * x.st);
  };
  // copies of this wave's 8 keys of block kb; 16-bit: to their swizzled places in a stage
  auto issue = [&](uint32_t stage, int kb, int pid) __attribute__((always_inline)) {
    // (from a value that the compiler takes for a new one each time: kept through the loop, the copies'
    // offsets would push operands out of the registers)
    int lane = (int)threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int r_in = lane / G::LPR, p16 = lane % G::LPR;
    const int key8 = key8_of(kb);
    pid = (unsigned)pid >= (unsigned)kv.num_pages ? 0 : pid;
    const int rmax = nk - 1 - key8;
    const uint8_t* kp = rfl_p(base_of(kpl, key8, pid));
    const uint8_t* vp = rfl_p(base_of(vpl, key8, pid));
    if constexpr (!Q8) {
      const uint32_t at = stage + (uint32_t)(8 * wave * G::ROWB);
#pragma unroll
      for (int i = 0; i < G::NI; ++i) {
        const int r = G::RPI * i + r_in, krow = 8 * wave + r;
        const int ck = p16 ^ G::swk(krow);
        const int cv = (((p16 >> 2) ^ G::swv(krow)) << 2) | (p16 & 3);
        const uint32_t rc = (uint32_t)min(r, rmax);
        dma16(kp, rc * kpl.st + (uint32_t)ck * 16u, at + (uint32_t)(G::RPI * i * G::ROWB));
        dma16(vp, rc * vpl.st + (uint32_t)cv * 16u, at + (uint32_t)(G::HALF + G::RPI * i * G::ROWB));
      }
    } else {
      // codes of row r at 8 wave HD + r HD (keys, then values), scales of keys and values behind
      constexpr int L8 = HD / 16, R8 = 64 / L8;  // lanes of a row, rows of a copy
      const uint32_t at = stage + (uint32_t)(8 * wave * HD);
      if (R8 <= 8 || lane < 8 * L8) {
#pragma unroll
        for (int i = 0; i < (R8 < 8 ? 8 / R8 : 1); ++i) {
          const uint32_t rc = (uint32_t)min(R8 * i + lane / L8, rmax);
          const uint32_t c = (uint32_t)(lane % L8) * 16u;
          dma16(kp, rc * kpl.st + c, at + (uint32_t)(R8 * i * HD));
          dma16(vp, rc * vpl.st + c, at + (uint32_t)(G::KB * HD + R8 * i * HD));
        }
      }
      if (lane < 8) {
        const uint32_t r = (uint32_t)min(lane, rmax);
        const uint32_t sc = stage + (uint32_t)(G::STAGE / 2 + 64 * wave);
        dma4(rfl_p(base_of(kspl, key8, pid)), r * kspl.st, sc);
        dma4(rfl_p(base_of(vspl, key8, pid)), r * vspl.st, sc + 32u);
      }
    }
  };
  // int8: this wave's codes of a block as 16-bit whole numbers, to their places in the tile
  auto widen = [&](uint32_t codes) __attribute__((always_inline)) {
    constexpr int CH = HD / 16;  // 16-byte chunks of a row of codes
    int lane = (int)threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    // this wave's scales: keys', then values'
    const uint32_t scales = codes + (uint32_t)(G::STAGE / 2 + 64 * wave + 4 * (lane & 15));
    const uint64_t odd = __ballot(!(fabsf(lds_ld<float>(scales)) < __builtin_inff()));
#pragma unroll
    for (int i = 0; i < 8 * CH / 64 || i == 0; ++i) {
      const int x = i * 64 + lane, r = x / CH, c16 = x % CH, krow = 8 * wave + r;
      if (8 * CH < 64 && x >= 8 * CH) break;
      const uint32_t from = codes + (uint32_t)(krow * HD + c16 * 16);
      const u32x4 kc = lds_ld<u32x4>(from), vc = lds_ld<u32x4>(from + G::KB * HD);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        u32x4 ko, vo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t wk = kc[2 * y + e / 2], wv = vc[2 * y + e / 2];
          const int b = 16 * (e % 2);
          ko[e] = T::pack_exact((float)(int8_t)(wk >> b), (float)(int8_t)(wk >> (b + 8)));
          vo[e] = TV::pack_exact((float)(int8_t)(wv >> b), (float)(int8_t)(wv >> (b + 8)));
        }
        const int c = 2 * c16 + y;
        const uint32_t to = lds0 + (uint32_t)(krow * G::ROWB);
        lds_st(to + (uint32_t)((c ^ G::swk(krow)) << 4), ko);
        lds_st(to + (uint32_t)(G::HALF + (((((c >> 2) ^ G::swv(krow)) << 2) | (c & 3)) << 4)), vo);
      }
    }
    // a scale that is not finite makes no number of its key's score; as a value's it is taken out
    if (odd && ((odd | odd >> 8) >> (lane & 7) & 1)) lds_st(scales, lane & 8 ? 0.0f : __builtin_nanf(""));
  };
  // 16-bit keys: values behind the last key, which hold it again and may be infinite, as zeros (this wave's 8)
  auto clear = [&](uint32_t stage, int kb) __attribute__((always_inline)) {
    int lane = (int)threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
#pragma unroll
    for (int i = 0; i < G::NI; ++i) {
      const int r = 8 * wave + G::RPI * i + lane / G::LPR;
      if (kb * G::KB + r >= nk) lds_st(stage + (uint32_t)(G::HALF + r * G::ROWB + (lane % G::LPR) * 16), u32x4{0, 0, 0, 0});
    }
  };

  // LDS places of this lane's operands: step s of K at ka ^ 32 s (the swizzle reaches 256 bytes), 32-wide block d of
  // V at va ^ 64 (d % 4), two transposing reads of 4 keys each
  const int s16 = lane & 15;
  const uint32_t ka = lds0 + (uint32_t)(col * G::ROWB + ((h ^ G::swk(col)) << 4));
  const uint32_t va = lds0 + (uint32_t)(G::HALF + (4 * h + (s16 >> 2)) * G::ROWB + (G::swv(s16 >> 2) << 6) +
                                        ((lane >> 4) & 1) * 32 + (s16 & 3) * 8);
  auto step = [&](auto stage_c, int kb, uint32_t scales) __attribute__((always_inline)) {
    constexpr uint32_t stage = decltype(stage_c)::value;
    if (R0 >= rows) return;
    // operands are read kAhead products ahead
    auto k_at = [&](int s) {
      return lds_ld<u32x4>((ka ^ (uint32_t)((s & 7) << 5)) + stage + (s >= 8 ? 256u : 0u));
    };
    f32x16 S = {};
    {
      u32x4 k[kAhead];
#pragma unroll
      for (int s = 0; s < kAhead; ++s) k[s] = k_at(s);
#pragma unroll
      for (int s = 0; s < G::NS; ++s) {
        __builtin_amdgcn_sched_barrier(0);
        S = T::mma32(k[s % kAhead], Q[s], S);
        if (s + kAhead < G::NS) k[s % kAhead] = k_at(s + kAhead);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (Q8) {
      // scales of keys 8 i + 4 h ..: this lane's four runs of scores
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 ks = lds_ld<f32x4>(scales + (uint32_t)(64 * i + 16 * h));
#pragma unroll
        for (int e = 0; e < 4; ++e) S[4 * i + e] *= ks[e];
      }
    }
    if (kb * G::KB + G::KB > nk) {
      int lane = (int)threadIdx.x & 63;
      asm volatile("" : "+v"(lane));
      const int rel = nk - kb * G::KB - 4 * (lane >> 5);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (8 * (i / 4) + i % 4 >= rel) S[i] = kNegInf;
    }
    float mx = fmaxf(fmaxf(S[0], S[1]), S[2]);
#pragma unroll
    for (int i = 3; i < 15; i += 2) mx = fmaxf(fmaxf(mx, S[i]), S[i + 1]);
    mx = fmaxf(mx, S[15]);
    float x, y;
    lane_pair<32>(mx, x, y);
    mx = fmaxf(x, y) * a.c;
    // (sums are rescaled only when a row's maximum has grown by more than 2^8, in fp16 when a block's largest P would
    // leave 2^4 .. 2^15 on either side: as for few rows, keys down to 18 octaves below it keep their weight.  From the window's
    // middle, as one of a wave's 32 rows that leaves it costs them all: 64 sequences behind 16384 tokens of 128 values 46.6 us,
    // from 2^14 48; a window from 2^-8, which holds 6 octaves, 44.8)
    constexpr bool NARROW = TV::DT == DT_F16;
    if (NARROW ? __any(off_window(mx - m, 4.0f, 15.0f)) : __any(mx > m + 8.0f)) {
      float mn = fmaxf(m, mx);
      if constexpr (NARROW) {
        lane_pair<32>(l, x, y);
        mn = fp16_reference(m, mx, x + y, 4.0f, 9.0f, 15.0f);
      }
      const float al = exp2_(m - (mn == kNegInf ? 0.0f : mn));
      m = mn;
      l *= al;
#pragma unroll
      for (int d = 0; d < G::ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) O[d][i] *= al;
    }
    const float ms = m == kNegInf ? 0.0f : m;
    u32x4 P[PN][2];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = exp2_(fmaf(S[8 * k + e], a.c, -ms));
        sum += p[e];
      }
      f32x4 vs[2];
      if constexpr (Q8) {
#pragma unroll
        for (int i = 0; i < 2; ++i) vs[i] = lds_ld<f32x4>(scales + (uint32_t)(64 * (2 * k + i) + 32 + 16 * h));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float p0 = p[2 * e], p1 = p[2 * e + 1];
        if constexpr (Q8) {
          p0 *= vs[e / 2][2 * (e % 2)];
          p1 *= vs[e / 2][2 * (e % 2) + 1];
        }
        const uint32_t w = TV::pack(p0, p1);
        P[0][k][e] = w;
        if constexpr (PN == 2) P[1][k][e] = TV::pack(p0 - bitcast<float>(w << 16), p1 - bitcast<float>(w & 0xFFFF0000u));
      }
    }
    l += sum;
    auto v_at = [&](int x) {  // operand of block x / 2, keys 16 (x % 2) ..
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      u32x2 v[2];
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const int d = x / 2, k = x % 2;
        const uint32_t at = (va ^ (uint32_t)((d & 3) << 6)) + stage +
                            (uint32_t)((d >> 2) * 256 + (16 * k + 8 * z) * G::ROWB);
        v[z] = bitcast<u32x2>(__builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)at));
      }
      return u32x4{v[0].x, v[0].y, v[1].x, v[1].y};
    };
    u32x4 v[kAhead];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < kAhead; ++x) v[x] = v_at(x);
#pragma unroll
    for (int x = 0; x < 2 * G::ND; ++x) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < PN; ++n) O[x / 2] = TV::mma32(v[x % kAhead], P[n][x % 2], O[x / 2]);
      if (x + kAhead < 2 * G::ND) v[x % kAhead] = v_at(x + kAhead);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // this wave's copies have landed and its LDS accesses are done, and so for all waves
  auto meet = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(wait_vm(0));
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  auto lds_done = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  int pid = page_of(kb0);
  if constexpr (!Q8) {
    constexpr std::integral_constant<uint32_t, 0> s0;
    constexpr std::integral_constant<uint32_t, (uint32_t)G::STAGE> s1;
    issue(lds0, kb0, pid);
    pid = page_of(kb0 + 1);
    auto turn = [&](auto stage_c, int kb) __attribute__((always_inline)) {
      constexpr uint32_t stage = decltype(stage_c)::value;
      meet();
      if (kb * G::KB + G::KB > nk) {
        clear(lds0 + stage, kb);
        lds_done();
      }
      issue(lds0 + (stage ? 0u : (uint32_t)G::STAGE), kb + 1, pid);
      pid = page_of(kb + 2);
      step(stage_c, kb, 0);
    };
    for (int kb = kb0;;) {
      turn(s0, kb);
      if (++kb >= kb1) break;
      turn(s1, kb);
      if (++kb >= kb1) break;
    }
  } else {
    // codes of block kb + 1 land while block kb is widened and used
    const uint32_t c0 = lds0 + G::STAGE;
    constexpr uint32_t CODES = G::STAGE / 2 + G::SCALES;
    constexpr std::integral_constant<uint32_t, 0> s0;
    uint32_t codes = c0;
    issue(codes, kb0, pid);
    pid = page_of(kb0 + 1);
    for (int kb = kb0; kb < kb1; ++kb) {
      meet();  // the tile has been read, this block's codes and scales are there
      const uint32_t next = codes == c0 ? c0 + CODES : c0;
      issue(next, kb + 1, pid);
      pid = page_of(kb + 2);
      widen(codes);
      lds_done();  // the tile is written
      step(s0, kb, codes + G::STAGE / 2);
      codes = next;
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(wait_vm(0));  // no copy may outlive the workgroup
  __builtin_amdgcn_sched_barrier(0);

  // (the lane's row anew, instead of in a register through the loop)
  int last = (int)threadIdx.x;
  asm volatile("" : "+v"(last));
  const int mine = R0 + (last & 31), half = (last >> 5) & 1;
  if (mine >= rows) return;
  float x, y;
  lane_pair<32>(l, x, y);
  l = any_bad ? __builtin_nanf("") : x + y;
  const long long at = (long long)hk * a.rows + U.row + mine;
  float* o = a.part + at * HD + 4 * half;
#pragma unroll
  for (int d = 0; d < G::ND; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *(f32x4*)(o + 32 * d + 8 * i) = f32x4{O[d][4 * i], O[d][4 * i + 1], O[d][4 * i + 2], O[d][4 * i + 3]};
  if (half == 0) {
    a.ml[at * 2] = m;
    a.ml[at * 2 + 1] = l;
  }
}

// Workgroups that a CU holds by registers.
constexpr int shared_occupancy(int hd, int nt) {
  return hd == 256 ? (nt == 2 ? 1 : 2) : hd == 128 ? (nt == 2 ? 2 : 3) : 3;
}

// NT: tiles of a prefix's unit (0: the wide form, for own keys too where a key head has more than 16 query heads).
template <typename T, int HD, bool Q8, int NT>
__global__ __launch_bounds__(kThreads, shared_occupancy(HD, NT)) void shared_kernel(const SharedArgs a) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int hk = (int)blockIdx.x % a.HKV, unit = (int)blockIdx.x / a.HKV;
  const Plan p = make_plan(a);
  Unit U;
  if (!find_unit(a, p, unit, U)) return;
  for (int* x : {&U.prefix, &U.src, &U.len, &U.b0, &U.n, &U.blk0, &U.blk1, &U.row}) *x = (int)rfl32((uint32_t)*x);
  if constexpr (NT == 0) {
    if (U.prefix || a.R > 16) {
      wide_unit<T, HD, Q8>(a, U, hk, (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds);
      return;
    }
  } else if (U.prefix) {
    run_unit<T, HD, Q8, NT>(a, U, hk, (float*)lds);
    return;
  }
  run_unit<T, HD, Q8, 1>(a, U, hk, (float*)lds);
}

// Joins the parts of a sequence's rows of one key head: a workgroup takes ROWS of them, in 1024 / (HD ROWS) slices of
// ROWS HD / 4 threads, which take parts in turn, the prefix's first; slices meet in LDS.  Few rows take one of them a
// workgroup, many rows as many as there are threads for (each workgroup finds its parts from the lengths again).
template <typename T, int HD, int ROWS, int THREADS>
__global__ __launch_bounds__(THREADS) void shared_join_kernel(const SharedArgs a) {
  constexpr int LPR = HD / 4, SL = THREADS / (LPR * ROWS), N = 8;
  __shared__ __attribute__((aligned(16))) float so[SL > 1 ? SL * ROWS * HD : 4];
  __shared__ float sm[SL * ROWS * 2];
  const int tid = (int)threadIdx.x;
  const int runs = (a.R + ROWS - 1) / ROWS;
  const int u = (int)blockIdx.x / runs, b = u / a.HKV, hk = u - b * a.HKV;
  const int s = tid / (LPR * ROWS), rr = tid / LPR % ROWS, f = tid % LPR;
  const int head = ((int)blockIdx.x - u * runs) * ROWS + rr;
  const Plan p = make_plan(a);
  if (b < p.lo || b >= p.hi) return;  // a row of no group
  // parts of the prefix: row prow of the first, pn rows to the next
  int start = 0, prow = 0, pn = 0, np = 0;
  for (int g0 = 0; g0 < a.G; g0 += 64) {
    const Group g = group_of(a, groups_at(a, p, g0), start);
    const int parts = parts_of(p, g.len), sums = wave_scan(parts * g.n);
    const uint64_t mine = __ballot(b >= g.b0 && b < g.b0 + g.n);
    if (mine) {
      const int at = __builtin_ctzll(mine);
      np = lane_value(parts, at);
      pn = lane_value(g.n, at);
      prow += lane_value(sums, at) - np * pn + b - lane_value(g.b0, at);
      break;
    }
    prow += lane_value(sums, 63);
  }
  int oslot = 0, no = 0;
  for (int b0 = 0; b0 < p.hi; b0 += 64) {
    const int parts = parts_of(p, own_at(a, p, b0));
    const int end = wave_scan(parts);
    if (b < b0 + 64) {
      no = lane_value(parts, b - b0);
      oslot += lane_value(end, b - b0) - no;
      break;
    }
    oslot += lane_value(end, 63);
  }
  const int hrow = min(head, a.R - 1);  // (rows behind the last are the last again, and not stored)
  const long long first = (long long)hk * a.rows;
  const long long pre0 = first + (long long)prow * a.R + hrow;
  const long long own0 = first + a.own_rows + (long long)oslot * a.R + hrow;
  const int n = np + no;
  auto row_of = [&](int i) { return i < np ? pre0 + (long long)i * (pn * a.R) : own0 + (long long)(i - np) * a.R; };
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
  if constexpr (SL > 1) {
    *(f32x4*)(so + tid * 4) = o;
    if (f == 0) sm[tid / LPR * 2] = M, sm[tid / LPR * 2 + 1] = ls;
    __syncthreads();
    if (s > 0) return;
    float top = kNegInf, sum = 0.0f;
    o = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < SL; ++i) top = fmaxf(top, sm[(i * ROWS + rr) * 2]);
    const float ts = top == kNegInf ? 0.0f : top;
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      const float e = exp2_(sm[(i * ROWS + rr) * 2] - ts);
      o += *(const f32x4*)(so + (i * ROWS * LPR + tid) * 4) * e;
      sum += sm[(i * ROWS + rr) * 2 + 1] * e;
    }
    ls = sum;
  }
  if (head >= a.R) return;
  const float inv = n == 0 ? 0.0f : 1.0f / ls;  // a sequence without keys: zeros
  *(u32x2*)((uint16_t*)a.o + b * a.ob + (hk * a.R + head) * a.oh + f * 4) =
      u32x2{T::pack(o[0] * inv, o[1] * inv), T::pack(o[2] * inv, o[3] * inv)};
}

template <typename T, int HD, bool Q8, int NT>
hipError_t launch_nt(const SharedArgs& a, hipStream_t st) {
  auto kern = shared_kernel<T, HD, Q8, NT>;
  constexpr int wide = NT == 0 ? prompt_lds<HD, Q8, 1>() : 0, thin = shared_lds<HD>(NT == 0 ? 1 : NT, Q8);
  constexpr size_t lds = wide > thin ? wide : thin;
  static std::atomic<uint64_t> done{0};
  hipError_t e = allow_lds((const void*)kern, lds, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3((unsigned)(a.units * a.HKV)), dim3(kThreads), lds, st, a);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  // (64 rows of 65 parts with 256 / 512 / 1024 threads: 6.1 / 5.3 / 6.6 us, of few parts 4.3 / 5.1 / 5.9; 576 rows of 45
  // 6.7 / 7.6 / 12.6; 2048 rows of 17 one by one 13.6, eight to a workgroup 8.5)
  constexpr int MANY = 1024 / HD;
  const long long rows = (long long)a.B * a.HKV * a.R;
  if (rows >= kSharedManyRows && a.R >= MANY)
    hipLaunchKernelGGL((shared_join_kernel<T, HD, MANY, 256>), dim3((unsigned)(a.B * a.HKV * ((a.R + MANY - 1) / MANY))),
                       dim3(256), 0, st, a);
  else if (HD < 256 || rows > kSharedFewRows || a.pre.max_pages <= (kSharedManyKeys >> a.pre.page_shift))
    hipLaunchKernelGGL((shared_join_kernel<T, HD, 1, 256>), dim3((unsigned)rows), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((shared_join_kernel<T, HD, 1, 512>), dim3((unsigned)rows), dim3(512), 0, st, a);
  return hipGetLastError();
}

}  // namespace

// WIDE: the form of many rows (in files of their own, as it is compiled with other flags)
template <typename T, int HD, bool WIDE>
hipError_t launch_shared_hd(const SharedArgs& a, hipStream_t st) {
  const bool q8 = a.own.k.s != nullptr;
  if constexpr (WIDE) {
    return q8 ? launch_nt<T, HD, true, 0>(a, st) : launch_nt<T, HD, false, 0>(a, st);
  } else {
    if (a.tiles == 2 && !q8) return launch_nt<T, HD, false, 2>(a, st);
    return q8 ? launch_nt<T, HD, true, 1>(a, st) : launch_nt<T, HD, false, 1>(a, st);
  }
}

template <typename T, bool WIDE>
hipError_t launch_shared_t(const SharedArgs& a, int hd, hipStream_t st) {
  if (hd == 256) return launch_shared_hd<T, 256, WIDE>(a, st);
  if (hd == 128) return launch_shared_hd<T, 128, WIDE>(a, st);
  return launch_shared_hd<T, 64, WIDE>(a, st);
}

}  // namespace qlin
