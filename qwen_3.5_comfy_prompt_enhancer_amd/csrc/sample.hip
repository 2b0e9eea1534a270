// One token of each row of logits: the k largest, cut by probability mass and by the share of the
// largest, drawn by a uniform number; and its log probability among the whole row.
//
//   x_0 >= x_1 >= ... the row's k largest (of equal ones the lowest index first)
//   w_i = exp((x_i - x_0) / T), kept while w_0 + ... + w_{i-1} < top_p (w_0 + ... + w_{k-1}) and w_i >= min_p
//   token: the first i with w_0 + ... + w_i > u (sum of the kept)
//   log p = (x - max) - log sum_j exp(x_j - max) over the row
//
// Bound by HBM for many rows, by latency for few: a row is read once, by several workgroups.  A workgroup
// takes tiles of 8192 logits, 32 to a thread, in registers.  The k-th largest of its 256 threads' maxima is a
// bound that the tile's k largest do not fall below, and at most 32 k values reach (about k in
// practice), as keys of (value, index) differ; those go to LDS and are put in order by counting, for each,
// the larger ones.  The last workgroup of a row to arrive puts the rows' lists in order the same way and
// draws.  Weights and their sums are of 64 bits (k numbers: a draw next to a border then falls as the formula
// says), the row's sum of exponentials of 32.
#include "step_dev.h"

namespace qlin {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;

// Order of a logit: larger for a larger one, 0 for -inf and for no number (neither is ever drawn).
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = bitcast<uint32_t>(x + 0.0f);  // (-0 as 0)
  const uint32_t u = (b >> 31) ? ~b : b | 0x80000000u;
  return x > kNegInf ? u : 0u;
}
__device__ __forceinline__ float value_of(uint32_t u) { return bitcast<float>((u >> 31) ? u & 0x7FFFFFFFu : ~u); }
__device__ __forceinline__ uint64_t key_of(uint32_t u, uint32_t i) { return u ? ((uint64_t)u << 32) | ~i : 0ull; }

// exp(x - m) of x <= m, with exp(0) for two infinities of one sign but for -inf, whose part is none.
__device__ __forceinline__ float weight_of(float x, float m) {
  if (x == m) return x == kNegInf ? 0.0f : 1.0f;
  return __builtin_amdgcn_exp2f((x - m) * kLog2e);
}

struct Lds {
  uint64_t cand[kSampleMost * 32 + kSampleMost];
  uint64_t most[kThreads];    // the threads' largest
  uint64_t list[kSampleMost];
  double w[kSampleMost];
  float m[kWaves], s[kWaves];
  uint64_t bound;
  int n, last;
};

// The k-th largest of the threads' keys (they differ), or 0 where there are fewer.
__device__ __forceinline__ uint64_t kth(Lds& L, uint64_t mine, int k) {
  const int tid = (int)threadIdx.x;
  L.most[tid] = mine;
  if (tid == 0) L.bound = 0ull;
  __syncthreads();
  int rank = 0;
#pragma unroll 16
  for (int i = 0; i < kThreads; ++i) rank += L.most[i] > mine;
  if (rank == k - 1 && mine) L.bound = mine;
  __syncthreads();
  const uint64_t r = L.bound;
  __syncthreads();
  return r;
}

// L.list: the k largest of the n keys in L.cand (n <= 32 k + k), in order; 0 behind the last.
__device__ __forceinline__ void sort_list(Lds& L, int n, int k) {
  const int tid = (int)threadIdx.x;
  constexpr int PER = (kSampleMost * 33 + kThreads - 1) / kThreads;
  // (counting takes n^2 / 256 steps: first the same bound again, over the keys as they lie now)
  for (int round = 0; round < 2 && n > 2 * kThreads; ++round) {
    uint64_t v[PER], top = 0ull;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      v[e] = tid + e * kThreads < n ? L.cand[tid + e * kThreads] : 0ull;
      top = v[e] > top ? v[e] : top;
    }
    const uint64_t low = kth(L, top, k);
    if (tid == 0) L.n = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (v[e] && v[e] >= low) L.cand[atomicAdd(&L.n, 1)] = v[e];
    __syncthreads();
    n = L.n;
    __syncthreads();
  }
  for (int i = tid; i < k; i += kThreads) L.list[i] = 0ull;
  __syncthreads();
  for (int i = tid; i < n; i += kThreads) {
    const uint64_t mine = L.cand[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += L.cand[j] > mine;
    if (rank < k && mine) L.list[rank] = mine;
  }
  __syncthreads();
}

__device__ __forceinline__ double scan64(double v) {  // inclusive, over a wave
  const int lane = (int)threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double o = __shfl_up(v, d, 64);
    if (lane >= d) v += o;
  }
  return v;
}

// Draws from L.list, of a row whose maximum and sum of exponentials are M and S.
__device__ __forceinline__ void draw(const SampleArgs& a, Lds& L, int b, float M, float S) {
  const int lane = (int)threadIdx.x;
  if (lane >= 64) return;
  const double x0 = (double)value_of((uint32_t)(L.list[0] >> 32)), T = fmax((double)a.temp.at(b), 0.0);
  const double top_p = (double)a.top_p.at(b), min_p = (double)a.min_p.at(b), u = (double)a.u[b];
  // two keys a lane
  bool there[2];
  double w[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * lane + e;
    const uint64_t key = i < a.k ? L.list[i] : 0ull;
    const double x = (double)value_of((uint32_t)(key >> 32));
    there[e] = key != 0ull;
    w[e] = !key ? 0.0 : x == x0 ? 1.0 : exp((x - x0) / T);
  }
  const double c1 = scan64(w[0] + w[1]), last = __shfl_up(c1, 1, 64), before = lane ? last : 0.0, c0 = before + w[0];
  const double most = top_p * __shfl(c1, 63, 64);
  // the kept ones are the first n, their sums those of all
  const uint64_t cut0 = __ballot(!(there[0] && before < most && w[0] >= min_p));
  const uint64_t cut1 = __ballot(!(there[1] && c0 < most && w[1] >= min_p));
  auto first = [](uint64_t even, uint64_t odd) {
    return min(even ? 2 * __builtin_ctzll(even) : 128, odd ? 2 * __builtin_ctzll(odd) + 1 : 128);
  };
  const int n = max(1, first(cut0, cut1));
  const double s0 = __shfl(c0, (n - 1) / 2, 64), s1 = __shfl(c1, (n - 1) / 2, 64);
  const double goal = u * (n % 2 ? s0 : s1);
  const int at = min(first(__ballot(c0 > goal), __ballot(c1 > goal)), n - 1);
  if (lane) return;
  const uint64_t key = L.list[at];
  const long long token = L.list[0] ? (long long)(uint32_t)~(uint32_t)key : -1;
  if (a.tokens64) ((long long*)a.tokens)[b] = token;
  else ((int*)a.tokens)[b] = (int)token;
  if (a.logp) {
    const float x = value_of((uint32_t)(key >> 32));
    a.logp[b] = token < 0 ? kNegInf : (float)((x == M ? 0.0 : (double)x - (double)M) - log((double)S));
  }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs a) {
  constexpr int IT = kSampleTile / kThreads / 8;
  __shared__ Lds L;
  const int tid = (int)threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int b = (int)blockIdx.x / a.chunks, chunk = (int)blockIdx.x - b * a.chunks;
  const uint8_t* row = (const uint8_t*)a.x + b * a.xs * (DT == DT_F32 ? 4 : 2);
  const int tiles = (a.V + kSampleTile - 1) / kSampleTile;

  float m = kNegInf, s = 0.0f;
  for (int tile = chunk; tile < tiles; tile += a.chunks) {
    const int v0 = tile * kSampleTile, n = min(kSampleTile, a.V - v0);
    const uint8_t* x = row + (long long)v0 * (DT == DT_F32 ? 4 : 2);
    Row8<DT> r[IT];
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int i = (it * kThreads + tid) * 8;
      if (i + 8 <= n) r[it].load(x, i);
    }
    uint32_t o[IT * 8];
    float top = kNegInf;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int i = (it * kThreads + tid) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = kNegInf;
        if (i + 8 <= n) v = r[it].get(e);
        else if (i + e < n) v = load1<DT>(x, i + e);
        o[it * 8 + e] = order_of(v);
        top = fmaxf(top, v);  // (the other one of a number and no number)
      }
    }
    // sum of exponentials, against the thread's own maximum
    const float mn = fmaxf(m, top);
    s = s > 0.0f ? s * weight_of(m, mn) : 0.0f;
    uint64_t mine = 0ull;
#pragma unroll
    for (int e = 0; e < IT * 8; ++e) {
      if (o[e]) s += weight_of(value_of(o[e]), mn);
      const uint64_t key = key_of(o[e], (uint32_t)(v0 + (e / 8 * kThreads + tid) * 8 + e % 8));
      mine = key > mine ? key : mine;
    }
    m = mn;
    uint64_t low = kth(L, mine, a.k);
    const bool more = tile != chunk;
    if (more && L.list[a.k - 1] > low) low = L.list[a.k - 1];
    // candidates, and what earlier tiles left
    if (tid == 0) L.n = more ? a.k : 0;
    if (more)
      for (int i = tid; i < a.k; i += kThreads) L.cand[i] = L.list[i];
    __syncthreads();
    if (mine >= low && mine) {
#pragma unroll
      for (int e = 0; e < IT * 8; ++e) {
        const uint64_t key = key_of(o[e], (uint32_t)(v0 + (e / 8 * kThreads + tid) * 8 + e % 8));
        if (key && key >= low) L.cand[atomicAdd(&L.n, 1)] = key;
      }
    }
    __syncthreads();
    const int found = L.n;
    __syncthreads();
    sort_list(L, found, a.k);
  }
  // the row's maximum and sum
  auto join = [&](float m2, float s2) {
    const float mn = fmaxf(m, m2);
    s = (s > 0.0f ? s * weight_of(m, mn) : 0.0f) + (s2 > 0.0f ? s2 * weight_of(m2, mn) : 0.0f);
    m = mn;
  };
  auto join_all = [&]() {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) join(__shfl_xor(m, d, 64), __shfl_xor(s, d, 64));
    if (lane == 0) L.m[wave] = m, L.s[wave] = s;
    __syncthreads();
    m = L.m[0], s = L.s[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) join(L.m[w], L.s[w]);
    __syncthreads();
  };
  join_all();
  if (a.chunks == 1) {
    draw(a, L, b, m, s);
    return;
  }
  uint64_t* keys = a.keys + (long long)b * a.chunks * a.k;
  uint64_t* stats = a.stats + (long long)b * a.chunks;
  for (int i = tid; i < a.k; i += kThreads)
    __hip_atomic_store(keys + chunk * a.k + i, L.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (tid == 0)
    __hip_atomic_store(stats + chunk, (uint64_t)bitcast<uint32_t>(m) << 32 | bitcast<uint32_t>(s), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __syncthreads();
  if (tid == 0) {
    const unsigned prev = __hip_atomic_fetch_add(a.cnt + b, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    L.last = prev == (unsigned)(a.chunks - 1);
    if (L.last) __hip_atomic_store(a.cnt + b, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!L.last) return;
  const int n = a.chunks * a.k;
  for (int i = tid; i < n; i += kThreads)
    L.cand[i] = __hip_atomic_load(keys + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  m = kNegInf, s = 0.0f;
  for (int i = tid; i < a.chunks; i += kThreads) {
    const uint64_t v = __hip_atomic_load(stats + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    join(bitcast<float>((uint32_t)(v >> 32)), bitcast<float>((uint32_t)v));
  }
  __syncthreads();
  join_all();
  sort_list(L, n, a.k);
  draw(a, L, b, m, s);
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.B * a.chunks)), block(kThreads);
  if (a.xdt == DT_F32) hipLaunchKernelGGL(sample_kernel<DT_F32>, grid, block, 0, st, a);
  else if (a.xdt == DT_BF16) hipLaunchKernelGGL(sample_kernel<DT_BF16>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(sample_kernel<DT_F16>, grid, block, 0, st, a);
  return hipGetLastError();
}

}  // namespace qlin
