// Attention of packed prompts (causal or not) over packed keys or a paged cache: the kernel
// template, included by attn_prompt_bf16.hip and attn_prompt_f16.hip.
//
//   o[i, h] = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - max_i)
//   over the keys j <= i + Lk - Lq of the row's sequence (all keys where not causal)
//
// One pass over the keys with a running maximum and sum.  A workgroup holds a tile of 128 rows: the
// tokens' rows of all G query heads of one key head next to each other (row = token G + head), so
// that a key block serves G heads and a causal tile spans few tokens.  Each of its four waves owns 32
// rows; keys come in blocks of 32 through an LDS ring of two stages.
//   * S^T = K Q^T and O^T = V^T P^T on 32x32x16 MFMAs with Q (as the B operand) and O in
//     registers: a lane holds one row (column of S^T), so its maximum and sum are its own but
//     for one exchange between the wave's halves, and P^T becomes the B operand of the second
//     product in place: lane half h holds keys 8i + 4h .. 8i + 4h + 3, the order in which V's
//     operand is read.
//   * K rows are read from LDS as 16-byte operands, V columns by the transposing 8-byte reads.
//     Both land by 16-byte LDS DMA whose lanes fetch swizzled chunks, so that a read's lanes
//     meet different banks (16-bit keys: no bank conflict is counted).
//   * int8 caches: codes land in a ring of their own and each wave widens its 8 keys to 16-bit whole
//     numbers (exact) in LDS; a key's scale multiplies its scores, a value's its probability, both
//     in 32 bits.  P x scale is rounded once for its product (to bf16; for fp16 queries it goes as
//     the sum of two bf16 numbers, as fp16 may not hold it).
//   * The sums are rescaled only when a row's maximum has grown by more than 2^8 (P stays below 2^8,
//     which bf16 holds with full relative precision), in fp16 when a block's largest P would leave
//     2^-8 .. 2^15 on either side (fp16_reference).  P is rounded to the queries' type for its product;
//     its sum, the maximum and O are 32-bit.
//
// What bounds it: the MFMAs (of 256 values, 32 products of 32 cycles a block and wave), then the softmax's
// vector work and LDS.  32 rows a wave, operands read three products ahead and two workgroups a CU (256
// values; three or four of smaller heads) took 310 us for an 8192-token prompt of 8 heads of 256 values
// where 64 rows a wave, each operand feeding two MFMAs, took 696: two waves a SIMD hide each other's
// softmax and waits, and a wave of 64 rows has no registers left to read ahead.  With the cuts and the
// order below 253 us now: 275 Gflop at 1.09 Pflop/s, where an 8192^3 library product reaches 1.20.
// Even batches that fill the chip reach 1.06 - 1.1 Pflop/s at 256 values, 0.95 at 128, 0.78 at 64
// (the softmax's work is the same for fewer products), over int8 caches 0.75 - 0.8 and 0.63 (widening
// takes as many vector instructions as the softmax).
//
//   * Where there are fewer or less even tiles than the chip holds, keys of all tiles are cut into
//     units of about equal length; units leave 32-bit partial sums, which are joined in key order by
//     the last unit of a tile to arrive, or by a second launch where tiles are few.  512 tokens over
//     6000 int8 keys: 52 us and 13 for the join of 60 MB of parts.
//   * Few tiles of 16-bit keys are halved (KG = 2): two waves hold 64 rows, the other two the same rows
//     over every second block, and their sums are added in LDS.
//
// A row's masked keys have no part in it whatever they hold.  Scores are replaced before the maximum.  An
// int8 value's scale that is not finite is taken out, and makes its key's score no number instead.  A 16-bit
// value that is no number is none times a P of zero either: a unit whose sums come out non-finite after
// masked blocks is computed again, finite values apart from the others (split): prompts of 512 / 2048 tokens
// whose first value is NaN take 66 / 170 us, of numbers 22 / 48.
#pragma once

#include "attn_dev.h"

namespace qlin {

namespace {

constexpr int kPromptThreads = 256;

// s_waitcnt vmcnt(n) lgkmcnt(0)
constexpr int wait_vm(int n) { return (n & 15) | (((n >> 4) & 3) << 14) | 0x70; }

// 16-byte LDS DMA: lane i copies 16 bytes from sbase + voff to LDS m0 + 16 i.  The compiler
// separates instructions that must not follow each other closely, but does not look into inline
// assembly: a base that a vector instruction (v_readfirstlane) wrote needs five wait states
// before a memory instruction reads it, m0 one.
__device__ __forceinline__ void dma16(const void* sbase, uint32_t voff, uint32_t m0) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(sbase), "{m0}"(m0) : "memory");
}

// 4-byte LDS DMA: lane i copies 4 bytes from sbase + voff to LDS m0 + 4 i.
__device__ __forceinline__ void dma4(const void* sbase, uint32_t voff, uint32_t m0) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dword %0, %1" ::"v"(voff), "s"(sbase), "{m0}"(m0) : "memory");
}

// LDS operands that are read ahead of their products.
constexpr int kAhead = 3;

template <typename P>
__device__ __forceinline__ P* rfl_p(P* p) {
  const uint64_t v = (uint64_t)p;
  return (P*)(((uint64_t)rfl32((uint32_t)(v >> 32)) << 32) | rfl32((uint32_t)v));
}

// A sequence: its rows of q, its keys.
struct Seq {
  int q0, nq;   // first row, rows
  int k0, nk;   // first packed row of its keys, keys
};

// Sequences b0 + lane (none behind the last).  Bounds are clamped to the rows there are and taken as
// rising: a sequence starts no earlier than any bound before it, so that sequences share no rows
// and never have more row tiles than the grid was made for, whatever `cu` holds.  `start`: the
// highest bound so far, for calls with rising b0.
__device__ __forceinline__ Seq seq_of(const PromptArgs& a, int b0, int& start) {
  const int b = b0 + ((int)threadIdx.x & 63);
  Seq s = {0, 0, 0, 0};
  int c0 = 0, c1 = 0;
  if (b < a.B) {
    c0 = min(max(a.cu[b], 0), a.T);
    c1 = min(max(a.cu[b + 1], 0), a.T);
    if (a.kv.table) {
      s.nk = kv_length(a.kv, b);
    } else {
      s.k0 = min(max(a.kv.cu[b], 0), a.kv.rows);
      s.nk = max(0, min(max(a.kv.cu[b + 1], 0), a.kv.rows) - s.k0);
    }
  }
  s.q0 = max(wave_scan_max(c0), start);
  s.nq = max(0, c1 - s.q0);
  start = lane_value(s.q0, 63);
  return s;
}

// Keys that row token i of a sequence sees.
__device__ __forceinline__ int seen(const PromptArgs& a, const Seq& s, int i) {
  return a.causal ? min(max(i + s.nk - s.nq + 1, 0), s.nk) : s.nk;
}

struct Tile {
  int b, tile;        // sequence, row tile
  Seq s;
  int nblk;           // key blocks that the tile sees
  int chunk;          // blocks of a unit
  int parts, part;    // units of the tile, this one
  int slot, step;     // partial of the tile's first unit, and the distance to the next
  int index;          // number of the tile among those of its key head
  // the same for all lanes, which the compiler cannot see
  __device__ __forceinline__ void uniform() {
    for (int* x : {&b, &tile, &s.q0, &s.nq, &s.k0, &s.nk, &nblk, &chunk, &parts, &part, &slot, &step, &index})
      *x = (int)rfl32((uint32_t)*x);
  }
};

// Work unit u (UNITS), or the first unit of row tile u, of a key head.
//
// Tiles of a sequence are ranked from its last, which sees most keys.  A unit is `chunk` blocks of
// a tile's keys, the tile's last unit what is left; units are numbered part by part, by rank
// within a part.  With chunk the average over the workgroups that run at once, long causal
// prompts then come out even: whole chunks start first, and the workgroup that gets the
// shortest rest of one part goes on with the longest of the next.
//
// Uncut tiles of up to 64 sequences start by rank over all of them, longest first (sequence by
// sequence: nine ragged prompts of up to 1500 tokens 66.8 us, by rank 61.8).
template <int ROWS, bool UNITS>
__device__ __forceinline__ bool find_tile(const PromptArgs& a, int u, Tile& r) {
  auto tiles_of = [&](const Seq& s) { return (int)(((long long)s.nq * a.G + ROWS - 1) / ROWS); };
  auto blocks_of = [&](const Seq& s) { return (s.nk + kPromptBlock - 1) / kPromptBlock; };
  int start = 0;
  const Seq first = seq_of(a, 0, start);
  const int start1 = start;
  constexpr int kUncut = 1 << 30;
  int chunk = kUncut;
  if (a.target > 0) {
    float w = 0.0f, longest = 0.0f;  // (an estimate; the same for all workgroups)
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const Seq s = b0 ? seq_of(a, b0, start) : first;
      const float t = (float)tiles_of(s), n = (float)blocks_of(s);
      // causal rows see half of their own keys on average (never less than half of all)
      w += a.causal ? fmaxf(t * (n - (float)(s.nq / (2 * kPromptBlock))), t * n * 0.5f) : t * n;
      if (t > 0.0f) longest = fmaxf(longest, n);
    }
    w = lane_value(wave_scan(w), 63);
    longest = wave_max(longest);
    // a cut that takes less than a third off the longest tile, or too few blocks, costs more than
    // it gives
    const float c = fmaxf(ceilf(w * (float)a.HKV / (float)a.target), (float)a.shortest);
    if (longest >= fmaxf(1.5f * c, c + (float)a.gain)) chunk = (int)fminf(c, 1e9f);
    else if (!UNITS) return false;  // (nothing to join)
  }
  auto take = [&](const Seq& s, int b0, int at, int nt, int rank, int part) {
    r.b = b0 + at;
    r.s.q0 = lane_value(s.q0, at);
    r.s.nq = lane_value(s.nq, at);
    r.s.k0 = lane_value(s.k0, at);
    r.s.nk = lane_value(s.nk, at);
    r.part = part;
    r.tile = nt - 1 - rank;
    r.step = nt;
    r.chunk = chunk;
    const int last = min((int)(((long long)(r.tile + 1) * ROWS - 1) / a.G), r.s.nq - 1);
    r.nblk = (seen(a, r.s, last) + kPromptBlock - 1) / kPromptBlock;
    r.parts = max(1, (r.nblk + chunk - 1) / chunk);
    return r.part < r.parts;
  };
  if (UNITS && chunk == kUncut && a.B > 1 && a.B <= 64) {
    const int tiles = tiles_of(first);
    auto before = [&](int rank) { return lane_value(wave_scan(min(tiles, rank)), 63); };
    int lo = 0, hi = lane_value(wave_scan_max(tiles), 63);  // before(lo) <= u < before(hi)
    if (u >= before(hi)) return false;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before(mid) <= u) lo = mid;
      else hi = mid;
    }
    const uint64_t have = __ballot(tiles > lo);
    const int mine = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(have >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)have, 0u));
    const int at = __builtin_ctzll(have & __ballot(mine == u - before(lo)));
    r.slot = r.index = 0;  // (of parts, which there are none of)
    return take(first, 0, at, lane_value(tiles, at), lo, 0);
  }
  int ubase = 0, tbase = 0;
  start = start1;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const Seq s = b0 ? seq_of(a, b0, start) : first;
    const int tiles = tiles_of(s);
    const int most = max(1, (blocks_of(s) + chunk - 1) / chunk);
    const int ue = wave_scan(tiles * most), te = wave_scan(tiles);
    const int usum = lane_value(ue, 63), tsum = lane_value(te, 63);
    if (u < (UNITS ? ubase + usum : tbase + tsum)) {
      const int at = __builtin_ctzll(__ballot((UNITS ? ubase + ue : tbase + te) > u));
      const int nt = lane_value(tiles, at), mp = lane_value(most, at);
      const int u0 = ubase + lane_value(ue, at) - nt * mp;
      const int t0 = tbase + lane_value(te, at) - nt;
      const int rank = UNITS ? (u - u0) % nt : u - t0;
      r.index = t0 + rank;
      r.slot = u0 + rank;
      return take(s, b0, at, nt, rank, UNITS ? (u - u0) / nt : 0);
    }
    ubase += usum;
    tbase += tsum;
  }
  return false;
}

// blockIdx.x -> (key head, index): workgroups go to the 8 XCDs in turn, and those of one key
// head stay on as few as there are for it, whose L2 then holds its keys.
__device__ __forceinline__ void split_grid(int hkv, int n, int& head, int& idx) {
  const int u = (int)blockIdx.x, x = u & 7, k = u >> 3;
  if (8 % hkv == 0) {
    const int per = 8 / hkv;
    head = x / per;
    idx = k * per + x % per;
  } else if (hkv % 8 == 0) {
    head = x + 8 * (k / n);
    idx = k % n;
  } else {
    head = u % hkv;
    idx = u / hkv;
  }
}
inline unsigned grid_of(int hkv, int n) {
  if (8 % hkv == 0) {
    const int per = 8 / hkv;
    return (unsigned)((n + per - 1) / per) * 8u;
  }
  return (unsigned)hkv * (unsigned)n;
}

template <int HD>
struct PGeo {
  static constexpr int KB = kPromptBlock;
  static constexpr int NS = HD / 16;       // MFMA steps of a score
  static constexpr int ND = HD / 32;       // 32-wide blocks of a value
  static constexpr int ROWB = HD * 2;      // bytes of a row in LDS
  static constexpr int LPR = HD / 8;       // lanes (16 bytes) of a row
  static constexpr int RPI = 64 / LPR;     // rows of a copy
  static constexpr int NI = 8 / RPI;       // copies of a wave's 8 rows
  static constexpr int HALF = KB * ROWB;   // bytes of a K or V tile
  static constexpr int STAGE = 2 * HALF;
  static constexpr int SCALES = 4 * 64;    // bytes of a block's scales: a wave's 8 of K and 8 of V
  static __device__ __forceinline__ int swk(int r) { return HD >= 128 ? r & 15 : (r >> 1) & 7; }
  static __device__ __forceinline__ int swv(int r) { return HD >= 128 ? r & 3 : (r >> 1) & 1; }
};

// LDS of a workgroup.  16-bit keys: a ring of two stages of KG blocks.  int8: one 16-bit tile, made from a
// ring of two tiles of codes and their scales.
template <int HD, bool Q8, int KG>
constexpr int prompt_lds() {
  return Q8 ? PGeo<HD>::STAGE + 2 * (PGeo<HD>::STAGE / 2 + PGeo<HD>::SCALES) : 2 * KG * PGeo<HD>::STAGE;
}

template <typename V>
__device__ __forceinline__ V lds_ld(uint32_t at) {
  return *(const __attribute__((address_space(3))) V*)(uintptr_t)at;
}
template <typename V>
__device__ __forceinline__ void lds_st(uint32_t at, V v) {
  *(__attribute__((address_space(3))) V*)(uintptr_t)at = v;
}

// Values that are no numbers, in the pass that looks out for them.  A pair of 16-bit values is split into
// its finite ones (zero in the others' place) and marks of the others; the product of marks and weights
// (1 for a key that a row sees, kOddNan where its P is zero, 0 for masked ones) adds up, exactly, to what
// a row's sum becomes: of at most 32 keys each, infinities of either sign stay below kOddNan.
constexpr float kOddPlus = 1.0f, kOddMinus = 64.0f, kOddNan = 4096.0f;

template <typename T>
__device__ __forceinline__ u32x2 split(uint32_t w) {
  constexpr uint32_t EXP = T::DT == DT_BF16 ? 0x7F80u : 0x7C00u, MANT = 0x7FFFu & ~EXP;
  constexpr uint32_t ONE = T::DT == DT_BF16 ? 0x3F80u : 0x3C00u, STEP = ONE == 0x3F80u ? 6u << 7 : 6u << 10;  // 2^6
  uint32_t finite = 0u, odd = 0u;
#pragma unroll
  for (int z = 0; z < 32; z += 16) {  // (without branches: the sums would be copied around them)
    const uint32_t x = (w >> z) & 0xFFFFu;
    const uint32_t mark = ONE + ((x & MANT) != 0u ? 2u * STEP : (x >> 15) * STEP);
    const bool number = (x & EXP) != EXP;
    finite |= (number ? x : 0u) << z;
    odd |= (number ? 0u : mark) << z;
  }
  return u32x2{finite, odd};
}

// What marks add up to: 0, an infinity, or no number.
__device__ __forceinline__ float odd_sum(float n) {
  const float minus = n < kOddNan && floorf(n / kOddMinus) * kOddMinus == n ? kNegInf : __builtin_nanf("");
  return n == 0.0f ? 0.0f : n < kOddMinus ? __builtin_inff() : minus;
}

// Q8: int8 cache.  KG = 2: two waves hold the rows of a tile of 64, the other two the same rows
// over every second block, and their sums are added through LDS at the end: for few tiles, each of
// which then takes half as long.
template <typename T, int HD, bool Q8, bool PAGED, int KG>
__global__ __launch_bounds__(kPromptThreads, KG == 2 ? 1 : HD == 64 ? 4 : HD == 128 ? 3 : 2)
void prompt_kernel(const PromptArgs a) {
  static_assert(KG == 1 || !Q8, "int8 keys: one group");
  using G = PGeo<HD>;
  using TV = std::conditional_t<Q8, Bf16, T>;  // type of P and V in their product
  // fp16 queries over int8 values: P x scale as two bf16 numbers, so that neither range nor
  // precision is lost
  constexpr int PN = Q8 && T::DT == DT_F16 ? 2 : 1;
  constexpr int ROWS = kPromptRows / KG;
  constexpr int ES = Q8 ? 1 : 2;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds;

  int hk, unit;
  split_grid(a.HKV, a.units, hk, unit);
  Tile t;
  if (hk >= a.HKV || unit >= a.units || !find_tile<ROWS, true>(a, unit, t)) return;
  t.uniform();
  const int tid = (int)threadIdx.x;
  const int wave = (int)rfl32((uint32_t)tid >> 6), lane = tid & 63;
  const int col = lane & 31, h = lane >> 5;
  const int kb0 = t.part * t.chunk, kb1 = min(t.nblk - kb0, t.chunk) + kb0;

  // this lane's row is R0 + col; its wave takes blocks kb0 + kg, kb0 + kg + KG, ...
  const int rg = wave % (4 / KG), kg = wave / (4 / KG);
  const int R0 = t.tile * ROWS + rg * 32;
  u32x4 Q[G::NS];
  auto load_q = [&](const PromptArgs& a, int col, int h) __attribute__((always_inline)) {
    const int i = (R0 + col) / a.G, ic = min(i, t.s.nq - 1);
    const uint16_t* q = (const uint16_t*)a.q + (t.s.q0 + ic) * a.qt + (hk * a.G + (R0 + col - i * a.G)) * a.qh + 8 * h;
#pragma unroll
    for (int s = 0; s < G::NS; ++s) Q[s] = ld_global<u32x4>(q + 16 * s);
    return seen(a, t.s, ic);
  };
  const int lim = load_q(a, col, h);
  // what every row of the wave sees, and what some row sees
  const int wmin = seen(a, t.s, min(R0 / a.G, t.s.nq - 1));
  const int wmax = R0 / a.G >= t.s.nq ? 0 : seen(a, t.s, min((R0 + 31) / a.G, t.s.nq - 1));

  f32x16 O[G::ND];
  float m = kNegInf, l = 0.0f;
#pragma unroll
  for (int d = 0; d < G::ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) O[d][i] = 0.0f;

  const int* table = PAGED ? a.kv.table + t.b * a.kv.table_stride : nullptr;
  const int nk = t.s.nk;
  // whether a page of the unit's keys lies outside the cache: looked at once, by every wave (each
  // fetches a quarter of the keys that all of them use)
  bool any_bad = false;
  if constexpr (PAGED) {
    const int e1 = (min(kb1 * G::KB, nk) - 1) >> a.kv.page_shift;
    for (int e = (kb0 * G::KB) >> a.kv.page_shift; e <= e1; e += 64)
      any_bad |= (unsigned)table[min(e + lane, e1)] >= (unsigned)a.kv.num_pages;
    any_bad = __any(any_bad);
  }
  // this wave's 8 keys of a block: the first one's place (keys behind the last are the last)
  auto key8_of = [&](int kb) { return min(min(kb, kb1 - 1) * G::KB + 8 * wave, (nk - 1) & ~7); };
  // (a scalar load: a vector one's wait would also wait for the copies in flight)
  auto page_of = [&](int kb) {
    return PAGED ? ((const __attribute__((address_space(4))) int*)table)[key8_of(kb) >> a.kv.page_shift] : 0;
  };
  // places of this head's keys: strides below 2^32 bytes, products of 64 bits
  struct Place {
    const uint8_t* p;
    uint32_t sp, st;
  };
  auto place = [&](const PagedTensor& x) {
    return Place{(const uint8_t*)x.p + ((PAGED ? 0LL : (long long)t.s.k0 * x.st) + hk * x.sh) * ES,
                 (uint32_t)x.sp * ES, (uint32_t)x.st * ES};
  };
  auto scale_place = [&](const PagedTensor& x) {
    return Place{(const uint8_t*)(x.s + hk * x.ssh), (uint32_t)x.ssp * 4u, (uint32_t)x.sst * 4u};
  };
  const Place kpl = place(a.kv.k), vpl = place(a.kv.v);
  const Place kspl = scale_place(a.kv.k), vspl = scale_place(a.kv.v);
  const uint32_t pmask = PAGED ? (1u << a.kv.page_shift) - 1u : 0u;
  auto base_of = [&](const Place& x, int key, int pid) {
    return PAGED ? x.p + ((uint64_t)(uint32_t)pid * x.sp + (uint64_t)((uint32_t)key & pmask) * x.st)
                 : x.p + (uint64_t)(uint32_t)key * x.st;
  };
  auto checked = [&](int pid) { return PAGED && (unsigned)pid >= (unsigned)a.kv.num_pages ? 0 : pid; };

  // Copies of this wave's 8 keys of block kb.  16-bit: to their swizzled places in a stage.
  auto issue = [&](uint32_t stage, int kb, int pid) __attribute__((always_inline)) {
    // (from a value that the compiler takes for a new one each time: kept through the loop, the
    // copies' offsets would push operands out of the registers)
    int lane = (int)threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int r_in = lane / G::LPR, p16 = lane % G::LPR;
    const int key8 = key8_of(kb);
    pid = checked(pid);
    const int rmax = nk - 1 - key8;
    const uint8_t* kp = rfl_p(base_of(kpl, key8, pid));
    const uint8_t* vp = rfl_p(base_of(vpl, key8, pid));
    if constexpr (!Q8) {
      const uint32_t at = stage + (uint32_t)(8 * wave * G::ROWB);
#pragma unroll
      for (int i = 0; i < G::NI; ++i) {
        const int r = G::RPI * i + r_in, row = 8 * wave + r;
        const int ck = p16 ^ G::swk(row);
        const int cv = (((p16 >> 2) ^ G::swv(row)) << 2) | (p16 & 3);
        const uint32_t rc = (uint32_t)min(r, rmax);
        dma16(kp, rc * kpl.st + (uint32_t)ck * 16u, at + (uint32_t)(G::RPI * i * G::ROWB));
        dma16(vp, rc * vpl.st + (uint32_t)cv * 16u,
              at + (uint32_t)(G::HALF + G::RPI * i * G::ROWB));
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
      const int x = i * 64 + lane, r = x / CH, c16 = x % CH, row = 8 * wave + r;
      if (8 * CH < 64 && x >= 8 * CH) break;
      const uint32_t from = codes + (uint32_t)(row * HD + c16 * 16);
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
        const uint32_t to = lds0 + (uint32_t)(row * G::ROWB);
        lds_st(to + (uint32_t)((c ^ G::swk(row)) << 4), ko);
        lds_st(to + (uint32_t)(G::HALF + (((((c >> 2) ^ G::swv(row)) << 2) | (c & 3)) << 4)), vo);
      }
    }
    // a scale that is not finite makes no number of its key's score, hence of every row that sees it; as a
    // value's it would make none of the rows that do not, either
    if (odd && ((odd | odd >> 8) >> (lane & 7) & 1)) lds_st(scales, lane & 8 ? 0.0f : __builtin_nanf(""));
  };

  // LDS places of this lane's operands: step s of K at ka ^ 32 s (the swizzle reaches 256 bytes),
  // 32-wide block d of V at va ^ 64 (d % 4), two transposing reads of 4 keys each
  const int s16 = lane & 15;
  const uint32_t mine = lds0 + (uint32_t)(kg * G::STAGE);
  const uint32_t ka = mine + (uint32_t)(col * G::ROWB + ((h ^ G::swk(col)) << 4));
  const uint32_t va = mine + (uint32_t)(G::HALF + (4 * h + (s16 >> 2)) * G::ROWB + (G::swv(s16 >> 2) << 6) +
                                        ((lane >> 4) & 1) * 32 + (s16 & 3) * 8);

  auto step = [&](auto stage_c, int kb, uint32_t scales, auto careful_c) __attribute__((always_inline)) {
    constexpr uint32_t stage = decltype(stage_c)::value;
    constexpr bool CAREFUL = decltype(careful_c)::value;
    if (kb * G::KB >= wmax || (KG > 1 && kb >= kb1)) return;
    // operands are read kAhead products ahead (the order is fixed: left to itself the compiler
    // reads each just before its product, and the wave waits for LDS every time)
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
    if (kb * G::KB + G::KB > wmin) {
      const int rel = lim - kb * G::KB - 4 * h;
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
    // (fp16: a block's largest P stays between 2^-8 and 2^15, see fp16_reference; every score of a deviation
    // below 3 then rescales about as seldom as the line of 2^8)
    constexpr bool NARROW = TV::DT == DT_F16;
    if (NARROW ? __any(off_window(mx - m, -8.0f, 15.0f)) : __any(mx > m + 8.0f)) {
      float mn = fmaxf(m, mx);
      if constexpr (NARROW) {
        lane_pair<32>(l, x, y);
        mn = fp16_reference(m, mx, x + y, -8.0f, 8.0f, 15.0f);
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
    u32x4 P[PN][2], W[2];
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
        P[0][k][e] = TV::pack(p0, p1);
        if constexpr (CAREFUL) {
          const int i = 8 * k + 2 * e, key = 8 * (i / 4) + i % 4, rel = lim - kb * G::KB - 4 * h;
          W[k][e] = TV::pack(key < rel ? p0 == 0.0f ? kOddNan : kOddPlus : 0.0f,
                             key + 1 < rel ? p1 == 0.0f ? kOddNan : kOddPlus : 0.0f);
        }
        if constexpr (PN == 2) {
          const uint32_t w = P[0][k][e];
          P[1][k][e] = TV::pack(p0 - bitcast<float>(w << 16), p1 - bitcast<float>(w & 0xFFFF0000u));
        }
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
    if constexpr (CAREFUL) {
      // finite values as ever; of the others, a second product counts what each row sees (see split)
#pragma unroll
      for (int d = 0; d < G::ND; ++d) {
        f32x16 seen_odd = {};
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const u32x4 v = v_at(2 * d + k);
          u32x4 finite, odd;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const u32x2 s = split<TV>(v[e]);
            finite[e] = s.x, odd[e] = s.y;
          }
          O[d] = TV::mma32(finite, P[0][k], O[d]);
          seen_odd = TV::mma32(odd, W[k], seen_odd);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) O[d][i] += odd_sum(seen_odd[i]);
        asm volatile("" : "+v"(O[d]));  // (now, not behind all others)
      }
      return;
    }
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
  // this wave's copies have landed and its LDS reads returned, and so for all waves
  auto meet = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(wait_vm(0));
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  // 16-bit keys: KG blocks of a stage
  constexpr uint32_t RING = KG * G::STAGE;
  constexpr std::integral_constant<uint32_t, 0> s0;
  constexpr std::integral_constant<uint32_t, RING> s1;
  int pid[KG];
  auto pages = [&](int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < KG; ++x) pid[x] = page_of(kb + x);
  };
  auto fetch = [&](uint32_t stage, int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < KG; ++x) issue(stage + (uint32_t)(x * G::STAGE), kb + x, pid[x]);
  };
  if (kb0 < kb1) {
    if constexpr (!Q8) {
      pages(kb0);
      fetch(lds0, kb0);
      pages(kb0 + KG);
      for (int kb = kb0;;) {
        meet();
        fetch(lds0 + RING, kb + KG);
        pages(kb + 2 * KG);
        step(s0, kb + kg, 0, std::false_type{});
        if ((kb += KG) >= kb1) break;
        meet();
        fetch(lds0, kb + KG);
        pages(kb + 2 * KG);
        step(s1, kb + kg, 0, std::false_type{});
        if ((kb += KG) >= kb1) break;
      }
    } else {
      pages(kb0);
      // codes of block kb + 1 land while block kb is widened and used
      const uint32_t c0 = lds0 + G::STAGE;
      constexpr uint32_t CODES = G::STAGE / 2 + G::SCALES;
      uint32_t codes = c0;
      issue(codes, kb0, pid[0]);
      pages(kb0 + 1);
      for (int kb = kb0; kb < kb1; ++kb) {
        meet();  // the tile has been read, this block's codes and scales are there
        const uint32_t next = codes == c0 ? c0 + CODES : c0;
        issue(next, kb + 1, pid[0]);
        pages(kb + 2);
        widen(codes);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the tile is written
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        step(s0, kb, codes + G::STAGE / 2, std::false_type{});
        codes = next;
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(wait_vm(0));  // no copy may outlive the workgroup
    __builtin_amdgcn_sched_barrier(0);
  }
  // (the row again, from a thread index that the compiler takes for another, and the arguments read
  // again, so that nothing of what follows is kept in registers through the loop)
  int tid2 = (int)threadIdx.x;
  asm volatile("" : "+v"(tid2));
  auto kernarg = (const __attribute__((address_space(4))) PromptArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(kernarg));
  const PromptArgs& ea = *(const PromptArgs*)kernarg;

  // Sums that are no numbers, after blocks that are masked for the wave: the unit again, a stage at a time,
  // finite values apart from the others.  (A row that sees such a value gets there too; its second
  // computation changes nothing.)
  const bool masked = kb1 * G::KB > seen(ea, t.s, min(t.tile * ROWS / ea.G, t.s.nq - 1));  // for some row of the tile
  if (!Q8 && masked) {
    __shared__ int s_spoiled[4];
    float z[4] = {};  // (four chains of additions)
    if (kb1 * G::KB > wmin) {
#pragma unroll
      for (int d = 0; d < G::ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i % 4] = fmaf(O[d][i], 0.0f, z[i % 4]);
    }
    const bool spoiled = __any(!((z[0] + z[1]) + (z[2] + z[3]) == 0.0f));
    if (lane == 0) s_spoiled[wave] = spoiled;
    __syncthreads();
    int any = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) any |= s_spoiled[w];
    if (rfl32((uint32_t)any)) {
      m = kNegInf, l = 0.0f;
#pragma unroll
      for (int d = 0; d < G::ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) O[d][i] = 0.0f;
      for (int kb = kb0; kb < kb1; kb += KG) {
        pages(kb);
        __syncthreads();  // the stage has been read
        fetch(lds0, kb);
        load_q(ea, tid2 & 31, (tid2 >> 5) & 1);
        meet();
        step(s0, kb + kg, 0, std::true_type{});
      }
    }
  }
  if constexpr (KG == 2) {
    // the second group's sums, then its maxima and sums of P, to LDS (every wave has read its last
    // stage); the first group adds them
    const uint32_t at = lds0 + (uint32_t)(rg * (32 * HD * 4 + 512) + lane * 16);
    const uint32_t aml = lds0 + (uint32_t)(rg * (32 * HD * 4 + 512) + 32 * HD * 4 + lane * 8);
    __syncthreads();
    if (kg == 1) {
#pragma unroll
      for (int d = 0; d < G::ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          lds_st(at + (uint32_t)((d * 4 + i) * 1024),
                 f32x4{O[d][4 * i], O[d][4 * i + 1], O[d][4 * i + 2], O[d][4 * i + 3]});
      lds_st(aml, u32x2{bitcast<uint32_t>(m), bitcast<uint32_t>(l)});
    }
    __syncthreads();
    if (kg == 0) {
      const u32x2 o1 = lds_ld<u32x2>(aml);
      const float m1 = bitcast<float>(o1.x), mn = fmaxf(m, m1), ms = mn == kNegInf ? 0.0f : mn;
      const float e0 = exp2_(m - ms), e1 = exp2_(m1 - ms);
      l = l * e0 + bitcast<float>(o1.y) * e1;
      m = mn;
#pragma unroll
      for (int d = 0; d < G::ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 x = lds_ld<f32x4>(at + (uint32_t)((d * 4 + i) * 1024));
#pragma unroll
          for (int e = 0; e < 4; ++e) O[d][4 * i + e] = O[d][4 * i + e] * e0 + x[e] * e1;
        }
    }
  }

  const int row = R0 + (tid2 & 31), tok = row / ea.G;
  const int head = hk * ea.G + (row - tok * ea.G);
  const int h2 = (tid2 >> 5) & 1;

  float x, y;
  lane_pair<32>(l, x, y);
  l = x + y;
  // partials: unit p of the tile at (slot + p step) of the key head's; 32-bit sums by row set,
  // 32-wide block, run of 8 values and lane, so that a wave moves 1 KiB at a time; then (maximum, sum
  // of P) of each row
  constexpr unsigned SLOT = (unsigned)prompt_slot_floats(HD, ROWS) * 4u;
  const __amdgpu_buffer_rsrc_t rs =
      part_rsrc((const char*)ea.part + (long long)hk * ea.units * SLOT + (long long)t.slot * SLOT, 0x7FFFFFF0u);
  const unsigned stride = (unsigned)t.step * SLOT;
  constexpr unsigned ML = ROWS * HD * 4;
  auto st_ml = [&](unsigned part, int r, float M, float ls) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    __builtin_amdgcn_raw_buffer_store_b64(bitcast<u32x2>(f32x2{M, ls}), rs, part * stride + ML + (unsigned)r * 8u, 0,
                                          kCpolSc1);
  };
  auto ld_ml = [&](unsigned part, int r) {
    return __builtin_amdgcn_raw_buffer_load_b64(rs, part * stride + ML + (unsigned)r * 8u, 0, kCpolSc1);
  };

  if (kg == 0) {
    if (any_bad) l = __builtin_nanf("");
    if (t.parts > 1) {
      if (R0 / ea.G < t.s.nq) {
        const unsigned at = (unsigned)t.part * stride + (unsigned)(rg * 32 * HD * 4) + (unsigned)(tid2 & 63) * 16u;
#pragma unroll
        for (int d = 0; d < G::ND; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            st_coherent(f32x4{O[d][4 * i], O[d][4 * i + 1], O[d][4 * i + 2], O[d][4 * i + 3]}, rs,
                        at + (unsigned)(d * 4 + i) * 1024u);
        if (h2 == 0) st_ml((unsigned)t.part, rg * 32 + (tid2 & 31), m, l);
      }
    } else {
      // a row that sees no key is zero
      const float f = seen(ea, t.s, min(tok, t.s.nq - 1)) > 0 ? 1.0f / l : 0.0f;
      uint16_t* o = (uint16_t*)ea.o + (long long)(t.s.q0 + tok) * ea.ot + head * ea.oh;
#pragma unroll
      for (int d = 0; d < G::ND; ++d)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // halves hold 4 values each of two runs of 8: exchanged, each stores one run
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int z = 0; z < 2; ++z)
              w[2 * e + z] = T::pack(O[d][8 * i + 4 * e + 2 * z] * f, O[d][8 * i + 4 * e + 2 * z + 1] * f);
          const auto r0 = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
          const auto r1 = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
          if (tok < t.s.nq)
            *(u32x4*)(o + 32 * d + 16 * i + 8 * h2) =
                u32x4{(uint32_t)r0[0], (uint32_t)r1[0], (uint32_t)r0[1], (uint32_t)r1[1]};
        }
    }
  }
  if (t.parts == 1 || ea.join_apart) return;

  // The last unit of a group of parts to arrive adds them in key order, the last of the groups adds
  // the groups' sums: the result does not depend on who was last, and no workgroup adds more than
  // the square root of the parts (or 4).  Waves share the 32-wide blocks of the row sets there are.
  __shared__ int s_last;
  auto last_of = [&](unsigned* c, int n) {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);  // this wave's stores have been made
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
  const int sets = min(ROWS / 32, (int)(((long long)(t.s.nq - 1) * ea.G + ea.G - (long long)t.tile * ROWS + 31) / 32));
  // parts first, first + by, ... (n): to the output, or in place of the first
  auto join = [&](int first, int by, int n, bool final) {
    for (int w = wave; w < sets * G::ND; w += 4) {
      const int set = w / G::ND, d = w % G::ND;
      const int R2 = t.tile * ROWS + set * 32 + col, i = R2 / ea.G;
      f32x4 o[4] = {};
      float M = kNegInf, ls = 0.0f;
      const unsigned off = (unsigned)((set * G::ND + d) * 4096 + lane * 16);
      constexpr int N = 2;  // parts in flight (four: an 8192-token prompt 258 -> 264 us, parts are few)
      for (int s0 = 0; s0 < n; s0 += N) {
        f32x4 x[N][4];
        u32x2 y[N];
#pragma unroll
        for (int s = 0; s < N; ++s) {
          const unsigned p = (unsigned)(first + min(s0 + s, n - 1) * by);
          y[s] = ld_ml(p, set * 32 + col);
#pragma unroll
          for (int f = 0; f < 4; ++f) x[s][f] = ld_coherent(rs, p * stride + off + (unsigned)f * 1024u);
        }
        // (no branch: the compiler would move each load behind it, next to its use, and wait for
        // every part by itself)
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < N; ++s) {
          const bool more = s0 + s < n;
          const float pm = more ? bitcast<float>(y[s].x) : kNegInf, pl = more ? bitcast<float>(y[s].y) : 0.0f;
          const float mn = fmaxf(M, pm), ms = mn == kNegInf ? 0.0f : mn;
          const float e0 = exp2_(M - ms), e1 = exp2_(pm - ms);
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const f32x4 px = more ? x[s][f] : f32x4{0, 0, 0, 0};
            o[f] = o[f] * e0 + px * e1;
          }
          ls = ls * e0 + pl * e1;
          M = mn;
        }
      }
      if (final) {
        if (i < t.s.nq) {
          const float inv = seen(ea, t.s, i) > 0 ? 1.0f / ls : 0.0f;
          uint16_t* out = (uint16_t*)ea.o + (long long)(t.s.q0 + i) * ea.ot + (hk * ea.G + (R2 - i * ea.G)) * ea.oh;
#pragma unroll
          for (int f = 0; f < 4; ++f)
            *(u32x2*)(out + d * 32 + f * 8 + 4 * h) =
                u32x2{T::pack(o[f][0] * inv, o[f][1] * inv), T::pack(o[f][2] * inv, o[f][3] * inv)};
        }
      } else {
        // (these values were read by this lane alone; maxima and sums by every wave, so they wait)
#pragma unroll
        for (int f = 0; f < 4; ++f) st_coherent(o[f], rs, (unsigned)first * stride + off + (unsigned)f * 1024u);
      }
    }
    if (final) return;
    float M = kNegInf, ls = 0.0f;
    for (int s = 0; s < n && wave < sets; ++s) {
      const u32x2 y = ld_ml((unsigned)(first + s * by), wave * 32 + col);
      const float pm = bitcast<float>(y.x), mn = fmaxf(M, pm), ms = mn == kNegInf ? 0.0f : mn;
      ls = ls * exp2_(M - ms) + bitcast<float>(y.y) * exp2_(pm - ms);
      M = mn;
    }
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    if (wave < sets && h == 0) st_ml((unsigned)first, wave * 32 + col, M, ls);
  };
  unsigned* cnt = ea.cnt + ((long long)hk * ea.tiles + t.index) * kPromptCounters;
  int by = 4;
  while (by * by < t.parts || by * (kPromptCounters - 1) < t.parts) ++by;
  const int groups = (t.parts + by - 1) / by, gq = t.part / by;
  if (!last_of(cnt + 1 + gq, min(by, t.parts - gq * by))) return;
  if (groups > 1) {
    join(gq * by, 1, min(by, t.parts - gq * by), false);
    if (!last_of(cnt, groups)) return;
    join(0, by, groups, true);
  } else {
    join(0, 1, t.parts, true);
  }
}

// The join as a launch of its own, for few tiles cut many times: a workgroup takes 32 values of 32
// rows, a thread four, so that the whole chip reads the parts.  (In the kernel above one workgroup
// would read a tile's: 512 tokens over 6000 int8 keys 80 us against 61 so, three prompts of 1000 tokens
// 44 against 40; above 256 tiles of two or three parts it gives nothing, 148 against 150 for 534.)
// Eight parts are in flight, sixteen made few parts dearer (four chunks of 700 over 3000 keys 67 -> 69).
template <typename T, int HD, int ROWS>
__global__ __launch_bounds__(kPromptThreads) void prompt_join_kernel(const PromptArgs a, int per) {
  constexpr int SETS = ROWS / 32, ND = HD / 32;
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int runs = ND / per;  // workgroups of a row set, `per` 32-wide blocks each
  const int d0 = (int)blockIdx.x % runs * per, set = (int)blockIdx.x / runs % SETS, u = (int)blockIdx.x / (runs * SETS);
  const int hk = u % a.HKV;
  Tile t;
  if (!find_tile<ROWS, false>(a, u / a.HKV, t)) return;
  t.uniform();
  const int R = t.tile * ROWS + set * 32 + (lane & 31), i = R / a.G;
  if (t.parts == 1 || i >= t.s.nq) return;
  // a part's place in scalars, this thread's in it: all of a key head's parts lie below 2^31 bytes
  constexpr unsigned SLOT = (unsigned)prompt_slot_floats(HD, ROWS) * 4u;
  const __amdgpu_buffer_rsrc_t rs =
      part_rsrc((const char*)a.part + ((long long)hk * a.units + t.slot) * SLOT, 0x7FFFFFF0u);
  const unsigned stride = (unsigned)t.step * SLOT;
  const unsigned ml = (unsigned)(ROWS * HD + (set * 32 + (lane & 31)) * 2) * 4u;
  uint16_t* out = (uint16_t*)a.o + (long long)(t.s.q0 + i) * a.ot + (hk * a.G + (R - i * a.G)) * a.oh;
  const bool some = seen(a, t.s, i) > 0;
  for (int d = d0; d < d0 + per; ++d) {
    const unsigned px = (unsigned)(set * 32 * HD + d * 1024 + tid * 4) * 4u;
    f32x4 o = {0, 0, 0, 0};
    float M = kNegInf, l = 0.0f;
    auto add = [&](auto in_flight) __attribute__((always_inline)) {
      constexpr int N = decltype(in_flight)::value;
      for (int s0 = 0; s0 < t.parts; s0 += N) {
        f32x4 x[N];
        u32x2 y[N];
#pragma unroll
        for (int s = 0; s < N; ++s) {
          const unsigned at = (unsigned)min(s0 + s, t.parts - 1) * stride;
          x[s] = bitcast<f32x4>(__builtin_amdgcn_raw_buffer_load_b128(rs, px, at, 0));
          y[s] = __builtin_amdgcn_raw_buffer_load_b64(rs, ml, at, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        // (no branch: the compiler would move each load behind it, next to its use, and wait for
        // every part: a 16-token chunk over 30000 keys, 94 parts, 57 us against 32)
#pragma unroll
        for (int s = 0; s < N; ++s) {
          const bool more = s0 + s < t.parts;
          const float pm = more ? bitcast<float>(y[s].x) : kNegInf, pl = more ? bitcast<float>(y[s].y) : 0.0f;
          const f32x4 po = more ? x[s] : f32x4{0, 0, 0, 0};
          const float mn = fmaxf(M, pm), ms = mn == kNegInf ? 0.0f : mn;
          const float e0 = exp2_(M - ms), e1 = exp2_(pm - ms);
          o = o * e0 + po * e1;
          l = l * e0 + pl * e1;
          M = mn;
        }
      }
    };
    if (t.parts == 2) add(std::integral_constant<int, 2>{});
    else if (t.parts <= 4) add(std::integral_constant<int, 4>{});
    else add(std::integral_constant<int, 8>{});
    const float inv = some ? 1.0f / l : 0.0f;
    *(u32x2*)(out + d * 32 + (tid >> 6) * 8 + 4 * (lane >> 5)) =
        u32x2{T::pack(o[0] * inv, o[1] * inv), T::pack(o[2] * inv, o[3] * inv)};
  }
}

template <typename T, int HD, bool Q8, bool PAGED, int KG>
hipError_t prompt_go(const PromptArgs& a, hipStream_t st) {
  constexpr int ROWS = kPromptRows / KG;
  const size_t lds = (size_t)prompt_lds<HD, Q8, KG>();
  auto kern = prompt_kernel<T, HD, Q8, PAGED, KG>;
  static std::atomic<uint64_t> done{0};
  const hipError_t e = allow_lds((const void*)kern, lds, done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3(grid_of(a.HKV, a.units)), dim3(kPromptThreads), lds, st, a);
  if (a.target > 0 && a.join_apart) {
    const int sets = a.tiles * a.HKV * (ROWS / 32);
    int per = 1;  // at most about as many workgroups as run at once
    while (per < HD / 32 && sets * (HD / 32 / per) > 2048) per *= 2;
    hipLaunchKernelGGL((prompt_join_kernel<T, HD, ROWS>), dim3((unsigned)(sets * (HD / 32 / per))),
                       dim3(kPromptThreads), 0, st, a, per);
  }
  return hipGetLastError();
}

template <typename T, int HD>
hipError_t prompt_src(const PromptArgs& a, hipStream_t st) {
  if (a.kv.table && a.kv.k.s) return prompt_go<T, HD, true, true, 1>(a, st);
  if (a.kv.table) return a.rows == kPromptRows ? prompt_go<T, HD, false, true, 1>(a, st)
                                               : prompt_go<T, HD, false, true, 2>(a, st);
  return a.rows == kPromptRows ? prompt_go<T, HD, false, false, 1>(a, st) : prompt_go<T, HD, false, false, 2>(a, st);
}

template <typename T>
hipError_t prompt_dispatch(const PromptArgs& a, int hd, hipStream_t st) {
  if (hd == 256) return prompt_src<T, 256>(a, st);
  if (hd == 128) return prompt_src<T, 128>(a, st);
  return prompt_src<T, 64>(a, st);
}

}  // namespace

}  // namespace qlin
