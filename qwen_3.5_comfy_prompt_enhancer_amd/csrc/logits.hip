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
// that fall into its run: a word of each token counts its places in the answer (the highest bit: one in the
// prompt), another holds the last place among the biases.
#include "step_dev.h"

namespace qlin {

namespace {

constexpr int kThreads = 256;
constexpr uint32_t kInPrompt = 0x80000000u;

template <int XDT, int ODT, int IT>
__global__ __launch_bounds__(kThreads) void logits_kernel(const LogitsArgs a) {
#pragma clang fp contract(off)
  constexpr int RUN = kThreads * 8 * IT;
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
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int i = (it * kThreads + tid) * 8;
    if (i + 8 <= n) {
      r[it].load(x, i);
      if (mask) {
        if (a.mask_bytes) __builtin_memcpy(&allowed[it], mask + i, 8);
        else allowed[it] = mask[i / 8];
      }
    }
  }

  const bool history = a.tokens != nullptr, biases = a.nb > 0;
  uint32_t* count = lds;
  uint32_t* place = lds + (history ? RUN : 0);
  if (history || biases) {
    for (int i = tid * 4; i < RUN * ((int)history + (int)biases); i += kThreads * 4) *(u32x4*)(lds + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
  }
  if (history) {
    const int len = a.lens ? min(max(a.lens[b], 0), a.L) : a.L;
    const int prompt = a.prompt_lens ? a.prompt_lens[b] : 0;
    auto note = [&](int i, long long id) {
      const long long at = id - v0;
      if (at < 0 || at >= n) return;
      if (i < prompt) atomicOr(count + at, kInPrompt);
      else atomicAdd(count + at, 1u);
    };
    constexpr int N = 8;  // loads in flight
    for (int i0 = tid; i0 < len; i0 += kThreads * N) {
      long long id[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const long long at = b * a.ts + min(i0 + e * kThreads, len - 1);
        id[e] = a.tokens64 ? ((const long long*)a.tokens)[at] : (long long)((const int*)a.tokens)[at];
      }
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i0 + e * kThreads < len) note(i0 + e * kThreads, id[e]);
    }
  }
  if (biases) {
    for (int i = tid; i < a.nb; i += kThreads) {
      const long long at = (long long)a.bias_ids[b * a.bis + i] - v0;
      if (at >= 0 && at < n) atomicMax(place + at, (uint32_t)i + 1u);
    }
  }
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  if (history) rep = a.rep.at(b), pres = a.pres.at(b), freq = a.freq.at(b);
  if (history || biases) __syncthreads();

  auto value = [&](float y, uint32_t c, uint32_t at, bool ok) {
    if (c) {
      y = y > 0.0f ? y / rep : y * rep;
      c &= ~kInPrompt;
      if (c) {
        y = y - freq * (float)c;
        y = y - pres;
      }
    }
    if (at) y = y + a.bias[b * a.bs + (at - 1u)];
    return ok ? y : -__builtin_inff();
  };
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int i = (it * kThreads + tid) * 8;
    if (i >= n) continue;
    if (i + 8 <= n) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool ok = !mask || (a.mask_bytes ? (allowed[it] >> (8 * e)) & 0xFFu : (allowed[it] >> e) & 1u);
        y[e] = value(r[it].get(e), history ? count[i + e] : 0u, biases ? place[i + e] : 0u, ok);
      }
      store8<ODT>(o, i, y);
    } else {
      for (int e = 0; i + e < n; ++e) {
        const bool ok = !mask || (a.mask_bytes ? mask[i + e] != 0 : mask[i / 8] >> e & 1);
        store1<ODT>(o, i + e, value(load1<XDT>(x, i + e), history ? count[i + e] : 0u, biases ? place[i + e] : 0u, ok));
      }
    }
  }
}

template <int XDT, int ODT>
hipError_t launch(const LogitsArgs& a, hipStream_t st) {
  const int arrays = (a.tokens ? 1 : 0) + (a.nb > 0 ? 1 : 0);
  constexpr int IT = 4, RUN = kThreads * 8 * IT;
  static_assert(RUN >= kLogitsRun, "");
  const long long tiles = (a.V + RUN - 1) / RUN;
  hipLaunchKernelGGL((logits_kernel<XDT, ODT, IT>), dim3((unsigned)(tiles * a.B)), dim3(kThreads),
                     (size_t)RUN * 4 * arrays, st, a);
  return hipGetLastError();
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
