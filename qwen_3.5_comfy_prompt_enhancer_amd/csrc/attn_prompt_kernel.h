// Attention of packed prompts (causal or not) over packed keys or a paged cache: the kernel
// template, included by attn_prompt_bf16.hip and attn_prompt_f16.hip.
//
//   o[i, h] = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - max_i)
//   over the keys j <= i + Lk - Lq of the row's sequence (all keys where not causal)
//
// One pass over the keys with a running maximum and sum.  A workgroup's four waves hold a tile
// of rows: the tokens' rows of all G query heads of one key head next to each other (row = token
// G + head), so that a key tile serves G heads and a causal tile spans few tokens.  A wave owns
// 32 or 64 rows; keys come in blocks of 32 through an LDS ring.
//   * S^T = K Q^T and O^T = V^T P^T on 32x32x16 MFMAs with Q (as the B operand) and O in
//     registers: a lane holds one row (column of S^T), so its maximum and sum are its own but
//     for one exchange between the wave's halves, and P^T becomes the B operand of the second
//     product in place: lane half h holds keys 8i + 4h .. 8i + 4h + 3, the order in which V's
//     operand is read.
//   * K rows are read from LDS as 16-byte operands, V columns by the transposing 8-byte reads.
//     Both land by 16-byte LDS DMA whose lanes fetch swizzled chunks, so that a read's lanes
//     meet different banks.  int8 caches pass through registers: code x scale, rounded once to
//     the queries' type, as a 16-bit cache would have held it.
//   * With 64 rows a wave, each K and V operand feeds two MFMAs: LDS (128 bytes a clock and CU)
//     then needs half the time of the MFMAs; with 32 rows as long as they do.
//   * The sums are rescaled only when a row's maximum has grown by more than 2^8: P stays below
//     2^8, which both 16-bit types hold with full relative precision.  P is rounded to the
//     queries' type for its product; its sum, the maximum and O are 32-bit.
//   * Keys of all tiles are cut into about equal units where there are fewer tiles than the chip
//     holds; units leave 32-bit partial sums, which a second launch joins in key order.
//
// A row's masked keys have no part in it whatever they hold: scores are replaced before the
// maximum, and as zero times a value that is no number is none, a tile whose sums come out
// non-finite after masked blocks is computed again row by row over its visible keys alone.
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

__device__ __forceinline__ Seq seq_of(const PromptArgs& a, int b) {
  Seq s;
  const int c0 = min(max(a.cu[b], 0), a.T), c1 = min(max(a.cu[b + 1], 0), a.T);
  s.q0 = c0;
  s.nq = max(0, c1 - c0);
  if (a.kv.table) {
    s.k0 = 0;
    s.nk = kv_length(a.kv, b);
  } else {
    const int e0 = min(max(a.kv.cu[b], 0), a.kv.rows), e1 = min(max(a.kv.cu[b + 1], 0), a.kv.rows);
    s.k0 = e0;
    s.nk = max(0, e1 - e0);
  }
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
  int parts, part;    // units of the tile, this one
  int slot;           // partial of the tile's first unit
  // the same for all lanes, which the compiler cannot see
  __device__ __forceinline__ void uniform() {
    for (int* x : {&b, &tile, &s.q0, &s.nq, &s.k0, &s.nk, &nblk, &parts, &part, &slot}) *x = (int)rfl32((uint32_t)*x);
  }
};

// Work unit u (UNITS) or row tile u of a key head.  Tiles of a sequence are numbered from the
// last, which sees most keys, so that long units start first.
template <int ROWS, bool UNITS>
__device__ __forceinline__ bool find_tile(const PromptArgs& a, int u, Tile& r) {
  const int lane = (int)threadIdx.x & 63;
  int chunk = 1 << 30;
  if (a.target > 0) {
    long long w = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      if (b0 + lane < a.B) {
        const Seq s = seq_of(a, b0 + lane);
        const long long t = ((long long)s.nq * a.G + ROWS - 1) / ROWS;
        const long long n = (s.nk + kPromptBlock - 1) / kPromptBlock;
        // causal rows see half of their own keys on average (never less than half of all)
        w += a.causal ? max(t * n - t * (s.nq / (2 * kPromptBlock)), (t * n + 1) / 2) : t * n;
      }
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) w += __shfl_xor(w, m);
    chunk = (int)min((w * a.HKV + a.target - 1) / a.target, (long long)1 << 30);
    chunk = max(chunk, kPromptMinBlocks);
  }
  int ubase = 0, tbase = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    Seq s = {0, 0, 0, 0};
    if (b0 + lane < a.B) s = seq_of(a, b0 + lane);
    const int tiles = (int)(((long long)s.nq * a.G + ROWS - 1) / ROWS);
    const int n = (s.nk + kPromptBlock - 1) / kPromptBlock;
    const int most = max(1, (n + chunk - 1) / chunk);
    int ue = tiles * most, te = tiles;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int x = __shfl_up(ue, m), y = __shfl_up(te, m);
      if (lane >= m) ue += x, te += y;
    }
    const int usum = __shfl(ue, 63), tsum = __shfl(te, 63);
    if (u < (UNITS ? ubase + usum : tbase + tsum)) {
      const int at = __builtin_ctzll(__ballot((UNITS ? ubase + ue : tbase + te) > u));
      r.b = b0 + at;
      r.s.q0 = (int)rfl32((uint32_t)__shfl(s.q0, at));
      r.s.nq = (int)rfl32((uint32_t)__shfl(s.nq, at));
      r.s.k0 = (int)rfl32((uint32_t)__shfl(s.k0, at));
      r.s.nk = (int)rfl32((uint32_t)__shfl(s.nk, at));
      const int nt = (int)rfl32((uint32_t)__shfl(tiles, at)), mp = (int)rfl32((uint32_t)__shfl(most, at));
      const int u0 = ubase + (int)rfl32((uint32_t)__shfl(ue, at)) - nt * mp;
      const int t0 = tbase + (int)rfl32((uint32_t)__shfl(te, at)) - nt;
      const int rank = UNITS ? (u - u0) / mp : u - t0;
      r.part = UNITS ? (u - u0) % mp : 0;
      r.tile = nt - 1 - rank;
      r.slot = u0 + rank * mp;
      const int last = min((int)(((long long)(r.tile + 1) * ROWS - 1) / a.G), r.s.nq - 1);
      r.nblk = (seen(a, r.s, last) + kPromptBlock - 1) / kPromptBlock;
      r.parts = max(1, (r.nblk + chunk - 1) / chunk);
      return r.part < r.parts;
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
  static __device__ __forceinline__ int swk(int r) { return HD >= 128 ? r & 15 : (r >> 1) & 7; }
  static __device__ __forceinline__ int swv(int r) { return HD >= 128 ? r & 3 : (r >> 1) & 1; }
};

template <bool Q8>
constexpr int prompt_stages() { return Q8 ? 2 : 4; }

// RS: row sets of 32 a wave holds.  Q8: int8 cache.
template <typename T, int HD, int RS, bool Q8, bool PAGED>
__global__ __launch_bounds__(kPromptThreads, 1) void prompt_kernel(const PromptArgs a) {
  using G = PGeo<HD>;
  constexpr int ROWS = prompt_rows(RS);
  constexpr int NST = prompt_stages<Q8>();
  constexpr int ES = Q8 ? 1 : 2;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds;

  int hk, unit;
  split_grid(a.HKV, a.units, hk, unit);
  Tile t;
  if (hk >= a.HKV || unit >= a.units || !find_tile<ROWS, true>(a, unit, t)) return;
  t.uniform();
  const int tid = (int)threadIdx.x;
  const int wave = (int)rfl32((uint32_t)tid >> 6), lane = tid & 63;
  const int col = lane & 31, h = lane >> 5;
  const int per = (t.nblk + t.parts - 1) / t.parts;
  const int kb0 = t.part * per, kb1 = min(t.nblk, kb0 + per);

  // rows: this lane's column of set rs is row R0 + 32 rs + col
  const int R0 = t.tile * ROWS + wave * 32 * RS;
  int tok[RS], head[RS], lim[RS];
  u32x4 Q[RS][G::NS];
#pragma unroll
  for (int rs = 0; rs < RS; ++rs) {
    const int R = R0 + 32 * rs + col;
    const int i = R / a.G;
    head[rs] = hk * a.G + (R - i * a.G);
    tok[rs] = i < t.s.nq ? i : -1;
    const int ic = min(i, t.s.nq - 1);
    lim[rs] = seen(a, t.s, ic);
    const uint16_t* q = (const uint16_t*)a.q + (t.s.q0 + ic) * a.qt + head[rs] * a.qh + 8 * h;
#pragma unroll
    for (int s = 0; s < G::NS; ++s) Q[rs][s] = ld_global<u32x4>(q + 16 * s);
  }
  // what every row of the wave sees, and what some row sees
  const int wmin = seen(a, t.s, min(R0 / a.G, t.s.nq - 1));
  const int wmax = R0 / a.G >= t.s.nq ? 0 : seen(a, t.s, min((R0 + 32 * RS - 1) / a.G, t.s.nq - 1));

  f32x16 O[RS][G::ND];
  float m[RS], l[RS];
#pragma unroll
  for (int rs = 0; rs < RS; ++rs) {
    m[rs] = kNegInf;
    l[rs] = 0.0f;
#pragma unroll
    for (int d = 0; d < G::ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) O[rs][d][i] = 0.0f;
  }

  bool bad = false;
  const int* table = PAGED ? a.kv.table + t.b * a.kv.table_stride : nullptr;
  const int nk = t.s.nk;
  // this wave's 8 keys of a block: the first one's place (keys behind the last are the last)
  auto key8_of = [&](int kb) { return min(min(kb, kb1 - 1) * G::KB + 8 * wave, (nk - 1) & ~7); };
  // (a scalar load: a vector one's wait would also wait for the copies in flight)
  auto page_of = [&](int kb) {
    return PAGED ? ((const __attribute__((address_space(4))) int*)table)[key8_of(kb) >> a.kv.page_shift] : 0;
  };
  auto base_of = [&](const PagedTensor& x, int key8, int pid) {
    const long long at = PAGED ? pid * x.sp + (key8 & ((1 << a.kv.page_shift) - 1)) * x.st
                               : (long long)(t.s.k0 + key8) * x.st;
    return (const uint8_t*)x.p + (at + hk * x.sh) * ES;
  };
  auto checked = [&](int pid) {
    if (PAGED && (unsigned)pid >= (unsigned)a.kv.num_pages) {
      bad = true;
      return 0;
    }
    return pid;
  };

  // 16-bit: this lane's copies
  const int r_in = lane / G::LPR, p16 = lane % G::LPR;
  auto issue = [&](int slot, int kb, int pid) __attribute__((always_inline)) {
    const int key8 = key8_of(kb);
    pid = checked(pid);
    const int rmax = nk - 1 - key8;
    const uint8_t* kp = rfl_p(base_of(a.kv.k, key8, pid));
    const uint8_t* vp = rfl_p(base_of(a.kv.v, key8, pid));
    const uint32_t at = lds0 + (uint32_t)(slot * G::STAGE + 8 * wave * G::ROWB);
#pragma unroll
    for (int i = 0; i < G::NI; ++i) {
      const int r = G::RPI * i + r_in, row = 8 * wave + r;
      const int ck = p16 ^ G::swk(row);
      const int cv = (((p16 >> 2) ^ G::swv(row)) << 2) | (p16 & 3);
      const uint32_t rc = (uint32_t)min(r, rmax);
      dma16(kp, rc * (uint32_t)(a.kv.k.st * 2) + (uint32_t)ck * 16u, at + (uint32_t)(G::RPI * i * G::ROWB));
      dma16(vp, rc * (uint32_t)(a.kv.v.st * 2) + (uint32_t)cv * 16u,
            at + (uint32_t)(G::HALF + G::RPI * i * G::ROWB));
    }
  };
  // int8: 16 codes a lane; rows of HD bytes take HD/16 lanes
  constexpr int L8 = HD / 16, R8 = 64 / L8, N8 = R8 >= 8 ? 1 : 8 / R8;
  u32x4 ck8[N8], cv8[N8];
  float sk8[N8], sv8[N8];
  auto load8 = [&](int kb, int pid) __attribute__((always_inline)) {
    const int key8 = key8_of(kb);
    pid = checked(pid);
    const int rmax = nk - 1 - key8;
    const uint8_t* kp = base_of(a.kv.k, key8, pid);
    const uint8_t* vp = base_of(a.kv.v, key8, pid);
    const long long off = key8 & ((1 << a.kv.page_shift) - 1);
    const float* ks = a.kv.k.s + pid * a.kv.k.ssp + off * a.kv.k.sst + hk * a.kv.k.ssh;
    const float* vs = a.kv.v.s + pid * a.kv.v.ssp + off * a.kv.v.sst + hk * a.kv.v.ssh;
#pragma unroll
    for (int i = 0; i < N8; ++i) {
      const int r = min(min(R8 * i + lane / L8, 7), rmax);
      ck8[i] = ld_global<u32x4>(kp + r * a.kv.k.st + (lane % L8) * 16);
      cv8[i] = ld_global<u32x4>(vp + r * a.kv.v.st + (lane % L8) * 16);
      sk8[i] = ks[r * a.kv.k.sst];
      sv8[i] = vs[r * a.kv.v.sst];
    }
  };
  auto put8 = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < N8; ++i) {
      const int r = R8 * i + lane / L8;
      if (R8 > 8 && r >= 8) break;
      const int row = 8 * wave + r;
      auto wide = [&](u32x4 c, float s, int half) {
        u32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t w = c[2 * half + e / 2];
          const int b = 16 * (e % 2);
          o[e] = T::pack((float)(int8_t)(w >> b) * s, (float)(int8_t)(w >> (b + 8)) * s);
        }
        return o;
      };
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int c = 2 * (lane % L8) + x;
        uint8_t* at = lds + slot * G::STAGE + row * G::ROWB;
        *(u32x4*)(at + ((c ^ G::swk(row)) << 4)) = wide(ck8[i], sk8[i], x);
        *(u32x4*)(at + G::HALF + (((((c >> 2) ^ G::swv(row)) << 2) | (c & 3)) << 4)) = wide(cv8[i], sv8[i], x);
      }
    }
  };

  // this lane's places in a stage: K operand s at row col, V operand (d, k) by two transposing
  // reads of 4 keys each
  auto step = [&](int slot, int kb) __attribute__((always_inline)) {
    if (kb * G::KB >= wmax) return;
    const bool masked = kb * G::KB + G::KB > wmin;
    const uint8_t* st = lds + slot * G::STAGE;
    f32x16 S[RS];
#pragma unroll
    for (int rs = 0; rs < RS; ++rs)
#pragma unroll
      for (int i = 0; i < 16; ++i) S[rs][i] = 0.0f;
#pragma unroll
    for (int s = 0; s < G::NS; ++s) {
      const u32x4 k = *(const u32x4*)(st + col * G::ROWB + (((2 * s + h) ^ G::swk(col)) << 4));
#pragma unroll
      for (int rs = 0; rs < RS; ++rs) S[rs] = T::mma32(k, Q[rs][s], S[rs]);
    }
    u32x4 P[RS][2];
#pragma unroll
    for (int rs = 0; rs < RS; ++rs) {
      if (masked) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (kb * G::KB + 8 * (i / 4) + 4 * h + i % 4 >= lim[rs]) S[rs][i] = kNegInf;
      }
      float mx = S[rs][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, S[rs][i]);
      float x, y;
      lane_pair<32>(mx, x, y);
      mx = fmaxf(x, y) * a.c;
      if (__any(mx > m[rs] + 8.0f)) {
        const float mn = fmaxf(m[rs], mx);
        const float al = exp2_(m[rs] - (mn == kNegInf ? 0.0f : mn));
        m[rs] = mn;
        l[rs] *= al;
#pragma unroll
        for (int d = 0; d < G::ND; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) O[rs][d][i] *= al;
      }
      const float ms = m[rs] == kNegInf ? 0.0f : m[rs];
      float p[16], sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[i] = exp2_(fmaf(S[rs][i], a.c, -ms));
        sum += p[i];
      }
      l[rs] += sum;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) P[rs][k][e] = T::pack(p[8 * k + 2 * e], p[8 * k + 2 * e + 1]);
    }
    const int s16 = lane & 15, dsub = (lane >> 4) & 1;
#pragma unroll
    for (int d = 0; d < G::ND; ++d)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        u32x2 v[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int row = 16 * k + 8 * x + 4 * h + (s16 >> 2);
          typedef short s16x4 __attribute__((ext_vector_type(4)));
          auto p = (__attribute__((address_space(3))) s16x4*)(st + G::HALF + row * G::ROWB +
                                                               ((d ^ G::swv(row)) << 6) + dsub * 32 + (s16 & 3) * 8);
          v[x] = bitcast<u32x2>(__builtin_amdgcn_ds_read_tr16_b64_v4i16(p));
        }
        const u32x4 vop = {v[0].x, v[0].y, v[1].x, v[1].y};
#pragma unroll
        for (int rs = 0; rs < RS; ++rs) O[rs][d] = T::mma32(vop, P[rs][k], O[rs][d]);
      }
  };

  if (kb0 < kb1) {
    if constexpr (!Q8) {
      int pid = page_of(kb0);
#pragma unroll
      for (int i = 0; i < NST - 1; ++i) {
        issue(i, kb0 + i, pid);
        pid = page_of(kb0 + i + 1);
      }
      int slot = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(wait_vm((NST - 2) * 2 * G::NI));
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        // the stage that all have read gets the block NST - 1 ahead
        issue(slot == 0 ? NST - 1 : slot - 1, kb + NST - 1, pid);
        pid = page_of(kb + NST);
        step(slot, kb);
        slot = slot == NST - 1 ? 0 : slot + 1;
      }
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(wait_vm(0));  // no copy may outlive the workgroup
      __builtin_amdgcn_sched_barrier(0);
    } else {
      load8(kb0, page_of(kb0));
      put8(0);
      load8(kb0 + 1, page_of(kb0 + 1));
      int slot = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        __syncthreads();
        put8(slot ^ 1);
        load8(kb + 2, page_of(kb + 2));
        step(slot, kb);
        slot ^= 1;
      }
    }
  }

  bool again = false;
#pragma unroll
  for (int rs = 0; rs < RS; ++rs) {
    float x, y;
    lane_pair<32>(l[rs], x, y);
    l[rs] = x + y;
    if (kb1 * G::KB > wmin) {  // masked blocks were among the unit's
      float z = 0.0f;
#pragma unroll
      for (int d = 0; d < G::ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) z = fmaf(O[rs][d][i], 0.0f, z);
      again |= !(z == 0.0f) && tok[rs] >= 0;
    }
  }
  float* slot_p = a.part + ((long long)hk * a.units + t.slot + t.part) * prompt_slot_floats(RS, HD);
  float* ml = slot_p + ROWS * HD;
  const bool any_bad = __any(bad);

  if (!__any(again)) {
#pragma unroll
    for (int rs = 0; rs < RS; ++rs) {
      if (any_bad) l[rs] = __builtin_nanf("");
      if (t.parts > 1) {
        float* dst = slot_p + (wave * RS + rs) * 32 * HD + lane * 4;
#pragma unroll
        for (int d = 0; d < G::ND; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *(f32x4*)(dst + (d * 4 + i) * 256) =
                f32x4{O[rs][d][4 * i], O[rs][d][4 * i + 1], O[rs][d][4 * i + 2], O[rs][d][4 * i + 3]};
        if (h == 0) *(float2*)(ml + ((wave * RS + rs) * 32 + col) * 2) = float2{m[rs], l[rs]};
      } else {
        const float inv = 1.0f / l[rs];
        // a row that sees no key is zero
        const float f = lim[rs] > 0 ? inv : 0.0f;
        uint16_t* o = (uint16_t*)a.o + (long long)(t.s.q0 + tok[rs]) * a.ot + head[rs] * a.oh;
#pragma unroll
        for (int d = 0; d < G::ND; ++d)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            // halves hold 4 values each of two runs of 8: exchanged, each stores one run
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int x = 0; x < 2; ++x)
                w[2 * e + x] = T::pack(O[rs][d][8 * i + 4 * e + 2 * x] * f, O[rs][d][8 * i + 4 * e + 2 * x + 1] * f);
            const auto r0 = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
            const auto r1 = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
            if (tok[rs] >= 0)
              *(u32x4*)(o + 32 * d + 16 * i + 8 * h) =
                  u32x4{(uint32_t)r0[0], (uint32_t)r1[0], (uint32_t)r0[1], (uint32_t)r1[1]};
          }
      }
    }
    return;
  }

  // Something non-finite among the sums: the wave's rows again, one at a time, over the keys
  // that each sees (lanes hold HD / 64 adjacent values).
  constexpr int E = HD / 64;
  for (int r = 0; r < 32 * RS; ++r) {
    const int R = R0 + r, i = R / a.G;
    if (i >= t.s.nq) break;
    const int hq = hk * a.G + (R - i * a.G);
    const int k1 = min(kb1 * G::KB, seen(a, t.s, i));
    const uint16_t* q = (const uint16_t*)a.q + (t.s.q0 + i) * a.qt + hq * a.qh + lane * E;
    float qv[E], o[E], mr = kNegInf, lr = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) qv[e] = T::get(q[e]), o[e] = 0.0f;
    for (int key = kb0 * G::KB; key < k1; ++key) {
      const int pid = PAGED ? table[key >> a.kv.page_shift] : 0;
      const int pc = (unsigned)pid >= (unsigned)a.kv.num_pages ? 0 : pid;
      const uint8_t* kp = base_of(a.kv.k, key, pc);
      const uint8_t* vp = base_of(a.kv.v, key, pc);
      float kv[E], vv[E], dot = 0.0f;
      if constexpr (Q8) {
        const long long off = key & ((1 << a.kv.page_shift) - 1);
        const float ks = a.kv.k.s[pc * a.kv.k.ssp + off * a.kv.k.sst + hk * a.kv.k.ssh];
        const float vs = a.kv.v.s[pc * a.kv.v.ssp + off * a.kv.v.sst + hk * a.kv.v.ssh];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          kv[e] = (float)((const int8_t*)kp)[lane * E + e] * ks;
          vv[e] = (float)((const int8_t*)vp)[lane * E + e] * vs;
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          kv[e] = T::get(((const uint16_t*)kp)[lane * E + e]);
          vv[e] = T::get(((const uint16_t*)vp)[lane * E + e]);
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) dot = fmaf(qv[e], kv[e], dot);
#pragma unroll
      for (int x = 1; x < 64; x <<= 1) dot += __shfl_xor(dot, x);
      const float s = dot * a.c;
      const float mn = fmaxf(mr, s), ms = mn == kNegInf ? 0.0f : mn;
      const float al = exp2_(mr - ms), p = exp2_(s - ms);
      mr = mn;
      lr = lr * al + p;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = o[e] * al + p * vv[e];
    }
    if (any_bad) lr = __builtin_nanf("");
    if (t.parts > 1) {
      float* dst = slot_p + (wave * RS + r / 32) * 32 * HD;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = lane * E + e;
        dst[((d / 32) * 4 + (d % 32) / 8) * 256 + ((r % 32) + 32 * ((d % 8) / 4)) * 4 + d % 4] = o[e];
      }
      if (lane == 0) *(float2*)(ml + ((wave * RS) * 32 + r) * 2) = float2{mr, lr};
    } else {
      uint16_t* out = (uint16_t*)a.o + (long long)(t.s.q0 + i) * a.ot + hq * a.oh + lane * E;
      const bool none = seen(a, t.s, i) == 0;
#pragma unroll
      for (int e = 0; e < E; ++e) out[e] = to_out16(none ? 0.0f : o[e] / lr, T::DT);
    }
  }
}

// Joins a cut tile's parts in key order: a workgroup takes one row set of 32.
template <typename T, int HD, int RS>
__global__ __launch_bounds__(kPromptThreads) void prompt_join_kernel(const PromptArgs a) {
  constexpr int ROWS = prompt_rows(RS);
  constexpr int SETS = 4 * RS;
  const int set = (int)blockIdx.x % SETS, u = (int)blockIdx.x / SETS;
  const int hk = u % a.HKV;
  Tile t;
  if (!find_tile<ROWS, false>(a, u / a.HKV, t) || t.parts == 1) return;
  const int tid = (int)threadIdx.x;
  const int R = t.tile * ROWS + set * 32 + (tid & 31);
  const int i = R / a.G;
  if (i >= t.s.nq) return;
  const long long sf = prompt_slot_floats(RS, HD);
  const float* p0 = a.part + ((long long)hk * a.units + t.slot) * sf;
  const float* ml = p0 + ROWS * HD + (set * 32 + (tid & 31)) * 2;
  float M = kNegInf;
  for (int s = 0; s < t.parts; ++s) M = fmaxf(M, ml[s * sf]);
  const float Ms = M == kNegInf ? 0.0f : M;
  constexpr int F = HD * 8 / kPromptThreads;  // float4s of a thread
  f32x4 o[F];
  float l = 0.0f;
#pragma unroll
  for (int f = 0; f < F; ++f) o[f] = f32x4{0, 0, 0, 0};
  for (int s = 0; s < t.parts; ++s) {
    const float e = exp2_(ml[s * sf] - Ms);
    l += ml[s * sf + 1] * e;
    const float* p = p0 + s * sf + set * 32 * HD + tid * 4;
#pragma unroll
    for (int f = 0; f < F; ++f) o[f] += *(const f32x4*)(p + f * kPromptThreads * 4) * e;
  }
  const float inv = seen(a, t.s, i) > 0 ? 1.0f / l : 0.0f;
  uint16_t* out = (uint16_t*)a.o + (long long)(t.s.q0 + i) * a.ot + (hk * a.G + (R - i * a.G)) * a.oh;
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const int x = (tid + f * kPromptThreads) / 64;  // (32-wide block, run of 8)
    const int d = (x / 4) * 32 + (x % 4) * 8 + 4 * ((tid & 63) >> 5);
    *(u32x2*)(out + d) = u32x2{T::pack(o[f][0] * inv, o[f][1] * inv), T::pack(o[f][2] * inv, o[f][3] * inv)};
  }
}

template <typename T, int HD, int RS, bool Q8, bool PAGED>
hipError_t prompt_go(const PromptArgs& a, hipStream_t st) {
  const size_t lds = (size_t)prompt_stages<Q8>() * PGeo<HD>::STAGE;
  auto kern = prompt_kernel<T, HD, RS, Q8, PAGED>;
  static const hipError_t attr = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                     (int)lds);
  if (attr != hipSuccess) return attr;
  hipLaunchKernelGGL(kern, dim3(grid_of(a.HKV, a.units)), dim3(kPromptThreads), lds, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.target == 0) return e;
  hipLaunchKernelGGL((prompt_join_kernel<T, HD, RS>), dim3((unsigned)(a.tiles * a.HKV * 4 * RS)),
                     dim3(kPromptThreads), 0, st, a);
  return hipGetLastError();
}

template <typename T, int HD, int RS>
hipError_t prompt_src(const PromptArgs& a, hipStream_t st) {
  if (!a.kv.table) return prompt_go<T, HD, RS, false, false>(a, st);
  if (a.kv.k.s) return prompt_go<T, HD, RS, true, true>(a, st);
  return prompt_go<T, HD, RS, false, true>(a, st);
}

template <typename T>
hipError_t prompt_dispatch(const PromptArgs& a, int hd, int rs, hipStream_t st) {
  if (hd == 256) return rs == 2 ? prompt_src<T, 256, 2>(a, st) : prompt_src<T, 256, 1>(a, st);
  if (hd == 128) return rs == 2 ? prompt_src<T, 128, 2>(a, st) : prompt_src<T, 128, 1>(a, st);
  return rs == 2 ? prompt_src<T, 64, 2>(a, st) : prompt_src<T, 64, 1>(a, st);
}

}  // namespace

}  // namespace qlin
