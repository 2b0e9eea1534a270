// Penalties for repeated tokens, biases and a mask on rows of logits.
//
//   y = x                                   in 32 bits
//   y = y > 0 ? y / r : y * r               where the row's history holds the token
//   y = (y - f c) - p                       where its answer holds it c > 0 times
//   y = y + bias                            where the row gives the token one
//   y = -inf                                where the mask does not allow it
//
// Each step is rounded to 32 bits once (the product f c too: no fused multiply-add), so that the result is
// the formula's to the bit, and once to the output's type.
//
// Bound by HBM: a row is read and written once.  A workgroup takes a run of tokens of one row.  Its logits are
// loaded first; while they are on their way it reads the row's history and biases whole and notes in LDS those
// that fall into its run, a word for each token: how often it came behind the prompt (bits 0 .. 18), the last
// place among the biases (19 .. 30) and whether the prompt holds it (31); two words where histories or biases
// are too long for that.  Each run reads the whole history, so many rows (and long histories) take longer
// runs in larger workgroups: 64 rows of 248320 16-bit logits to 32 bits with histories of 8192 tokens 32 us, without
// any 22 (4.3 TB/s).  Larger runs yet (16384, 1024 threads: 37) leave a CU two workgroups that wait for each other's barriers.
#include "attn_dev.h"
#include "step_dev.h"

namespace qlin {

namespace {

constexpr uint32_t kInPrompt = 0x80000000u, kCount = (1u << 19) - 1u;
constexpr int kPlace = 19;
constexpr long long kManyLogits = 3 << 20;
constexpr int kLongHistory = 2048;
constexpr uint32_t kPlaces = 0xFFFu;

// A token's word: a thread looks at eight words by 16-byte reads; in plain order a read of threads 8 .. 15 meets
// one of 0 .. 7 in the same banks (3.5 M cycles of conflicts in the 32 us above, 0.01 M so; the call 1.2 us less).
__device__ __forceinline__ uint32_t word_of(uint32_t i) { return i ^ (i >> 4 & 4u); }

// WORDS: of LDS for a token: 1 (all in one), 2 (a count, and a place), or 0 (no history, no biases).
template <int XDT, int ODT, int WORDS, int THREADS, int IT>
__global__ __launch_bounds__(THREADS) void logits_kernel(const LogitsArgs a) {
#pragma clang fp contract(off)
  constexpr int RUN = THREADS * 8 * IT;
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  const int tiles = (a.V + RUN - 1) / RUN;
  const int b = (int)blockIdx.x / tiles, v0 = ((int)blockIdx.x - b * tiles) * RUN;
  const int tid = (int)threadIdx.x;
  const int n = min(RUN, a.V - v0);
  const uint8_t* x = (const uint8_t*)a.x + (b * a.xs + v0) * (XDT == DT_F32 ? 4 : 2);
  uint8_t* o = (uint8_t*)a.o + (b * a.os + v0) * (ODT == DT_F32 ? 4 : 2);

  Row8<XDT> r[IT];
  uint64_t allowed[IT];  // a byte of each token, or its bits in the lowest byte
  const uint8_t* mask = nullptr;
  if (a.mask) mask = (const uint8_t*)a.mask + (a.mask_bytes ? b * a.ms + v0 : b * a.ms * 4 + v0 / 8);
  auto load_row = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int i = (it * THREADS + tid) * 8;
      if (i + 8 <= n) {
        r[it].load(x, i);
        if (mask) {
          if (a.mask_bytes) __builtin_memcpy(&allowed[it], mask + i, 8);
          else allowed[it] = mask[i / 8];
        }
      }
    }
  };

  const bool history = WORDS > 0 && a.tokens, biases = WORDS > 0 && a.nb > 0;
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  if constexpr (WORDS > 0) {
    // a first batch of the history and of the biases is loaded before its length is known
    constexpr int N = 8;  // loads in flight
    constexpr uint32_t kNone = ~0u;
    uint32_t id[N], bid = kNone;
    auto at_of = [&](long long id) { return id >= v0 && id < v0 + n ? (uint32_t)(id - v0) : kNone; };
    auto load = [&](int i0) __attribute__((always_inline)) {
      if (a.tokens64) {
        long long w[N];
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = ((const long long*)a.tokens)[b * a.ts + min(i0 + e * THREADS, a.L - 1)];
#pragma unroll
        for (int e = 0; e < N; ++e) id[e] = at_of(w[e]);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) id[e] = (uint32_t)((const int*)a.tokens)[b * a.ts + min(i0 + e * THREADS, a.L - 1)] - (uint32_t)v0;
      }
    };
    if (history) load(tid);
    if (biases) bid = (uint32_t)a.bias_ids[b * a.bis + min(tid, a.nb - 1)] - (uint32_t)v0;
    __builtin_amdgcn_sched_barrier(0);  // (loads come back in order: the row is not waited for until it is needed)
    load_row();
    __builtin_amdgcn_sched_barrier(0);
    const int len = history ? (a.lens ? min(max(a.lens[b], 0), a.L) : a.L) : 0;
    const int prompt = history && a.prompt_lens ? a.prompt_lens[b] : 0;
    if (history) rep = a.rep.at(b), pres = a.pres.at(b), freq = a.freq.at(b);
#pragma unroll
    for (int i = 0; i < 2 * IT * WORDS; ++i) *(u32x4*)(lds + (i * THREADS + tid) * 4) = u32x4{0, 0, 0, 0};
    __syncthreads();
    for (int i0 = tid; i0 < len;) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int i = i0 + e * THREADS;
        if (i >= len || id[e] >= (uint32_t)n) continue;
        if (i < prompt) atomicOr(lds + word_of(id[e]), kInPrompt);
        else atomicAdd(lds + word_of(id[e]), 1u);
      }
      i0 += THREADS * N;
      if (i0 < len) load(i0);
    }
    for (int i = tid; biases && i < a.nb;) {
      if (bid < (uint32_t)n) {
        const uint32_t mine = (uint32_t)i + 1u;
        if constexpr (WORDS == 2) {
          atomicMax(lds + RUN + word_of(bid), mine);
        } else {
          uint32_t* word = lds + word_of(bid);
          uint32_t old = *word;
          while ((old >> kPlace & kPlaces) < mine) {
            const uint32_t was = atomicCAS(word, old, (old & ~(kPlaces << kPlace)) | mine << kPlace);
            if (was == old) break;
            old = was;
          }
        }
      }
      i += THREADS;
      if (i < a.nb) bid = (uint32_t)a.bias_ids[b * a.bis + i] - (uint32_t)v0;
    }
    __syncthreads();
  }

  if constexpr (WORDS == 0) load_row();

  auto adjusted = [&](float y, uint32_t w, uint32_t at) {
    const uint32_t c = w & (WORDS == 1 ? kCount : ~kInPrompt);
    if (w & (kInPrompt | c)) {
      y = y > 0.0f ? y / rep : y * rep;
      if (c) {
        y = y - freq * (float)c;
        y = y - pres;
      }
    }
    if (at) y = y + a.bias[b * a.bs + (at - 1u)];
    return y;
  };
  auto value = [&](float y, uint32_t w, uint32_t at, bool ok) {
    if constexpr (WORDS == 1) y = adjusted(y, w, w >> kPlace & kPlaces);
    if constexpr (WORDS == 2) y = adjusted(y, w, at);
    return ok ? y : -__builtin_inff();
  };
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int i = (it * THREADS + tid) * 8;
    if (i >= n) continue;
    if (i + 8 <= n) {
      float y[8];
      u32x4 w[2] = {}, at[2] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t from = word_of((uint32_t)i + 4u * h);
        if constexpr (WORDS > 0) w[h] = *(const u32x4*)(lds + from);
        if constexpr (WORDS == 2) at[h] = *(const u32x4*)(lds + RUN + from);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool ok = !mask || (a.mask_bytes ? (allowed[it] >> (8 * e)) & 0xFFu : (allowed[it] >> e) & 1u);
        y[e] = value(r[it].get(e), w[e / 4][e % 4], at[e / 4][e % 4], ok);
      }
      store8<ODT>(o, i, y);
    } else {
      for (int e = 0; i + e < n; ++e) {
        const bool ok = !mask || (a.mask_bytes ? mask[i + e] != 0 : mask[i / 8] >> e & 1);
        const uint32_t from = word_of((uint32_t)(i + e));
        store1<ODT>(o, i + e, value(load1<XDT>(x, i + e), WORDS > 0 ? lds[from] : 0u, WORDS == 2 ? lds[RUN + from] : 0u, ok));
      }
    }
  }
}

template <int XDT, int ODT, int WORDS, int THREADS, int IT>
hipError_t go(const LogitsArgs& a, hipStream_t st) {
  constexpr int RUN = THREADS * 8 * IT;
  auto kern = logits_kernel<XDT, ODT, WORDS, THREADS, IT>;
  constexpr size_t lds = (size_t)RUN * 4 * WORDS;
  const long long tiles = ((long long)a.V + RUN - 1) / RUN;
  hipLaunchKernelGGL(kern, dim3((unsigned)(tiles * a.B)), dim3(THREADS), lds, st, a);
  return hipGetLastError();
}

template <int XDT, int ODT>
hipError_t launch(const LogitsArgs& a, hipStream_t st) {
  if (!a.tokens && a.nb == 0) return go<XDT, ODT, 0, 256, 1>(a, st);
  // (what a word holds; 248320 bf16 logits, one / two words: 4094 / 4095 biases of one row 7.5 / 6.4 us, of 64 33.8 / 45.5;
  // histories of 2^19 - 1 / 2^19 tokens of one row 81 / 143, of eight 115 / 204)
  if (a.L > (int)kCount || a.nb >= (int)kPlaces) return go<XDT, ODT, 2, 256, 1>(a, st);
  // (a whole history to every run: 512-token histories of few rows 4.0 us in short runs and 5.4 in long ones, 8192 tokens
  // of 64 rows 42 and 33)
  if ((long long)a.B * a.V >= kManyLogits) return go<XDT, ODT, 1, 512, 2>(a, st);
  if (a.L > kLongHistory) return go<XDT, ODT, 1, 512, 1>(a, st);
  return go<XDT, ODT, 1, 256, 1>(a, st);
}

template <int XDT>
hipError_t launch_x(const LogitsArgs& a, hipStream_t st) {
  if (a.odt == DT_F32) return launch<XDT, DT_F32>(a, st);
  if (a.odt == DT_BF16) return launch<XDT, DT_BF16>(a, st);
  return launch<XDT, DT_F16>(a, st);
}

}  // namespace

hipError_t launch_logits(const LogitsArgs& a, hipStream_t st) {
  if (a.xdt == DT_F32) return launch_x<DT_F32>(a, st);
  if (a.xdt == DT_BF16) return launch_x<DT_BF16>(a, st);
  return launch_x<DT_F16>(a, st);
}

}  // namespace qlin
