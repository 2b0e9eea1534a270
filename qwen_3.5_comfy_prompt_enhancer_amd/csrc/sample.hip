// One token of each row of logits: the k largest, cut by probability mass and by the share of the
// largest, drawn by a uniform number; and its log probability among the whole row.
//
//   x_0 >= x_1 >= ... the row's k largest (of equal ones the lowest index first)
//   w_i = exp((x_i - x_0) / T), kept while w_0 + ... + w_{i-1} < top_p (w_0 + ... + w_{k-1}) and w_i >= min_p
//   token: the first i with w_0 + ... + w_i > u (sum of the kept); of T = 0 the first
//   log p = (x - max) - log sum_j exp(x_j - max) over the row
//
// Bound by HBM for many rows, by latency for few: a row is read once, by several workgroups, each of which takes
// a part of it, 32 or 64 logits of a thread, for the maximum and the sum of exponentials of each thread.  The k-th
// largest of its 256 threads' maxima (to 20 bits, rounded down) is a bound that the part's k largest do not fall
// below, and in practice little more than k logits reach; the threads whose maximum does leave theirs in LDS, from
// their registers (longer parts are read again; for all parts that took 29 us where this takes 25).  64 rows of 248320
// fp32 logits take 25 us for k = 50 (2.5 TB/s; 8 us of a workgroup's time go to reading and summing, 5 to the search, 7
// of the row's last one to the join), one row 11.4.  (Lists kept in registers as tiles come took 104 and 27.)  Where
// many of equal value reach it (a mask of the type's lowest value), the bound goes on with their index.  The last
// workgroup of a row to arrive does the same with all parts' candidates, puts what reaches the bound in order by
// counting, for each, the larger ones, and draws.  Weights and their sums are of 64 bits (k numbers: a draw next to a
// border then falls as the formula says), the row's sum of exponentials of 32.
#include "attn_dev.h"
#include "step_dev.h"

namespace qlin {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kCandidates = 1024;
constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;

// Order of a logit: larger for a larger one, 0 for -inf (which is never drawn).
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = bitcast<uint32_t>(x + 0.0f);  // (-0 as 0)
  return x > -kInf ? b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u) : 0u;
}
constexpr uint32_t kLowest = 0x00800000u;  // of the lowest finite number
__device__ __forceinline__ float value_of(uint32_t u) { return bitcast<float>((u >> 31) ? u & 0x7FFFFFFFu : ~u); }

// exp(x - m) of x <= m, with exp(0) for two infinities of one sign but for -inf, whose part is none.
__device__ __forceinline__ float weight_of(float x, float m) {
  if (x == m) return x == -kInf ? 0.0f : 1.0f;
  return __builtin_amdgcn_exp2f((x - m) * kLog2e);
}

struct Lds {
  uint64_t cand[kCandidates];
  uint64_t list[kSampleMost];
  uint32_t top[kThreads];
  float m[kWaves], s[kWaves];
  int n, last;
};

// The k-th largest of the 256 numbers o (four of each lane, the same on all waves), its bits below `last`
// cleared.  For few, that of 64 or 128 groups' largest is close enough (no larger, and less work).
__device__ __forceinline__ uint32_t bound_of(const uint32_t (&o)[4], int k, uint32_t last) {
  const uint32_t p = max(o[0], o[1]), q = max(o[2], o[3]);
  auto search = [&](auto count) {
    uint32_t t = 0u;
    for (uint32_t bit = 0x80000000u; bit >= last; bit >>= 1) {
      const uint32_t c = t | bit;
      if (count(c) >= k) t = c;
      if (bit == 1u) break;
    }
    return t;
  };
  auto lanes = [](bool yes) { return __builtin_popcountll(__ballot(yes)); };
  if (k <= 24) return search([&](uint32_t c) { return lanes(max(p, q) >= c); });
  if (k <= 56) return search([&](uint32_t c) { return lanes(p >= c) + lanes(q >= c); });
  return search([&](uint32_t c) { return lanes(o[0] >= c) + lanes(o[1] >= c) + lanes(o[2] >= c) + lanes(o[3] >= c); });
}

// Each thread's number, on all waves: four of each lane.  (L.top is read by the time the next barrier is passed.)
__device__ __forceinline__ void share_tops(Lds& L, uint32_t mine, uint32_t (&o)[4]) {
  const int tid = (int)threadIdx.x;
  L.top[tid] = mine;
  if (tid == 0) L.n = 0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = L.top[(tid & 63) + 64 * e];
}

__device__ __forceinline__ void add(Lds& L, uint64_t key, uint64_t low) {
  if (key < low) return;
  const int at = atomicAdd(&L.n, 1);
  if (at < kCandidates) L.cand[at] = key;
}

// The k largest of a workgroup's keys (order, ~index), which differ, and maybe a few more, to L.cand: how many.
// top: the largest order of this thread's keys; scan(f) calls f(key) for each of them (0: none); quick(order) adds
// those from that order on to L.cand.
template <typename Quick, typename Scan>
__device__ __forceinline__ int gather(Lds& L, int k, uint32_t top, Quick quick, Scan scan) {
  const int tid = (int)threadIdx.x;
  uint32_t o[4];
  share_tops(L, top, o);
  const uint32_t rough = max(bound_of(o, k, 0x1000u), kLowest);
  auto collect = [&](uint64_t low, bool some) {
    if (some) scan([&](uint64_t key) { add(L, key, low); });
    __syncthreads();
    return L.n;
  };
  if (top >= rough) quick(rough);
  __syncthreads();
  int n = L.n;
  if (n <= kCandidates) return n;
  // Many of (nearly) equal value: the k-th largest of the threads' largest keys, order and index.
  uint64_t most = 0ull;
  scan([&](uint64_t key) { most = max(most, key); });
  const uint32_t t = bound_of(o, k, 1u);
  __syncthreads();
  share_tops(L, top > t ? ~0u : top == t ? (uint32_t)most : 0u, o);
  uint64_t low = max((uint64_t)t << 32 | bound_of(o, k, 1u), (uint64_t)1);
  n = collect(low, most >= low);
  if (n <= kCandidates) return n;
  // In few threads: the k-th largest key itself, by its bits.
  low = 0ull;
  for (uint64_t bit = 1ull << 63; bit; bit >>= 1) {
    const uint64_t c = low | bit;
    int mine = 0;
    scan([&](uint64_t key) { mine += key >= c; });
    __syncthreads();
    if (tid == 0) L.n = 0;
    __syncthreads();
    if (mine) atomicAdd(&L.n, mine);
    __syncthreads();
    if (L.n >= k) low = c;
  }
  __syncthreads();
  if (tid == 0) L.n = 0;
  __syncthreads();
  return collect(max(low, (uint64_t)1), true);
}

// L.list: the k largest of the n keys (order, ~index) in L.cand, which differ, in order; 0 behind the last.
// Several threads count for a key where keys are few.
__device__ __forceinline__ void sort_list(Lds& L, int n, int k) {
  const int tid = (int)threadIdx.x;
  for (int i = n + tid; i < k; i += kThreads) L.list[i] = 0ull;
  const int share = n <= 32 ? 8 : n <= 64 ? 4 : n <= 128 ? 2 : 1;
  for (int i = tid / share; i < n; i += kThreads) {  // (a key's threads are neighbours: all or none)
    const uint64_t mine = L.cand[i];
    int rank = 0;
#pragma unroll 8
    for (int j = tid % share; j < n; j += share) rank += L.cand[j] > mine;
    for (int d = 1; d < share; d *= 2) rank += __shfl_xor(rank, d, 64);
    if (rank < k) L.list[rank] = mine;
  }
  __syncthreads();
}

__device__ __forceinline__ double scan64(double v) {  // inclusive, over a wave
  auto add = [&](auto ctrl, auto rows) {
    const uint64_t u = bitcast<uint64_t>(v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
    v += bitcast<double>((uint64_t)hi << 32 | lo);
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});  // row_shr 1, 2, 4, 8
  add(integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
  add(integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
  add(integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
  add(integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});  // row_bcast 15, 31
  add(integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});
  return v;
}
__device__ __forceinline__ double lane64(double v, int at) {  // one lane's, on all
  const uint64_t u = bitcast<uint64_t>(v);
  return bitcast<double>((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), at) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, at));
}

// Draws from L.list, of a row whose maximum and sum of exponentials are M and S (the first wave).
__device__ __forceinline__ void draw(const SampleArgs& a, const Lds& L, int b, float M, float S, float temp, float top_p,
                                     float min_p, float u) {
  const int lane = (int)threadIdx.x;
  const double x0 = (double)value_of((uint32_t)(L.list[0] >> 32)), T = fmax((double)temp, 0.0);
  // two keys a lane
  bool there[2];
  double w[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = 2 * lane + e;
    const uint64_t key = i < a.k ? L.list[i] : 0ull;
    const double x = (double)value_of((uint32_t)(key >> 32));
    there[e] = key != 0ull;
    // (beside an infinite one nothing weighs: in front of the quotient, which is no number where T is infinite too)
    w[e] = !key ? 0.0 : x == x0 ? 1.0 : x0 == (double)kInf ? 0.0 : exp((x - x0) / T);
  }
  const double c1 = scan64(w[0] + w[1]);
  const double prev = __shfl_up(c1, 1, 64), from = lane ? prev : 0.0, mid = from + w[0];
  const double most = (double)top_p * lane64(c1, 63);
  // the kept ones are the first n, their sums those of all
  const uint64_t cut0 = __ballot(!(there[0] && from < most && w[0] >= (double)min_p));
  const uint64_t cut1 = __ballot(!(there[1] && mid < most && w[1] >= (double)min_p));
  auto first = [](uint64_t even, uint64_t odd) {
    return min(even ? 2 * __builtin_ctzll(even) : 128, odd ? 2 * __builtin_ctzll(odd) + 1 : 128);
  };
  // (temperature 0: the first alone, as its equals weigh 1 too; infinite ones share the row at any temperature)
  const int n = T == 0.0 && x0 < (double)kInf ? 1 : max(1, first(cut0, cut1));
  const double goal = (double)u * (n % 2 ? lane64(mid, (n - 1) / 2) : lane64(c1, (n - 1) / 2));
  const int at = min(first(__ballot(mid > goal), __ballot(c1 > goal)), n - 1);
  if (lane) return;
  const uint64_t key = L.list[at];
  const long long token = L.list[0] ? (long long)(uint32_t)~(uint32_t)key : -1;
  if (a.tokens64) ((long long*)a.tokens)[b] = token;
  else ((int*)a.tokens)[b] = (int)token;
  if (a.logp) {
    const float x = value_of((uint32_t)(key >> 32));
    a.logp[b] = token < 0 ? -kInf : (float)((x == M ? 0.0 : (double)x - (double)M) - log((double)S));
  }
}

// SHORT: rows of up to 2048 logits, which come one by one, so that all threads have some; else IT runs of eight of a
// thread at a time.
template <int DT, bool SHORT, int IT>
__global__ __launch_bounds__(kThreads, IT > 4 ? 4 : 6) void sample_kernel(const SampleArgs a) {
  constexpr int N = IT * 8;
  __shared__ Lds L;
  const int tid = (int)threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int b = (int)blockIdx.x / a.chunks, chunk = (int)blockIdx.x - b * a.chunks;
  const uint8_t* row = (const uint8_t*)a.x + b * a.xs * (DT == DT_F32 ? 4 : 2);
  // (on their way while the row is read)
  const float temp = a.temp.at(b), top_p = a.top_p.at(b), min_p = a.min_p.at(b), u = a.u[b];

  // This workgroup's part of the row: whole runs of 8.
  const int len = (int)((((long long)a.V + a.chunks - 1) / a.chunks + 7) & ~7LL);
  const int v0 = (int)min((long long)chunk * len, (long long)a.V), n = min(len, a.V - v0);
  const uint8_t* x = row + (long long)v0 * (DT == DT_F32 ? 4 : 2);
  // N of this thread's logits, from place i0 of the part on: f(y, place), of places behind the end -inf
  auto some = [&](int i0, auto f) __attribute__((always_inline)) {
    if constexpr (SHORT) {
      float y[N];
#pragma unroll
      for (int e = 0; e < N; ++e) y[e] = load1<DT>(x, min(i0 + e * kThreads + tid, n - 1));
#pragma unroll
      for (int e = 0; e < N; ++e) f(e, i0 + e * kThreads + tid < n ? y[e] : -kInf, i0 + e * kThreads + tid);
    } else {
      Row8<DT> r[IT];
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const int i = i0 + (it * kThreads + tid) * 8;
        if (i + 8 <= n) r[it].load(x, i);
      }
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const int i = i0 + (it * kThreads + tid) * 8;
        if (i + 8 <= n) {
#pragma unroll
          for (int e = 0; e < 8; ++e) f(it * 8 + e, r[it].get(e), i + e);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) f(it * 8 + e, i + e < n ? load1<DT>(x, i + e) : -kInf, i + e);
        }
      }
    }
  };
  constexpr int STEP = N * kThreads;
  float m = -kInf, s = 0.0f, v[N];
  for (int i0 = 0; i0 < n; i0 += STEP) {
    float top = m;
    some(i0, [&](int e, float y, int) {
      v[e] = fmaxf(y, -kInf);  // (no number as -inf)
      top = fmaxf(top, v[e]);
    });
    // sum of exponentials, against the thread's own maximum
    if (top == kInf) {
      s = m == kInf ? s : 0.0f;
#pragma unroll
      for (int e = 0; e < N; ++e) s += v[e] == kInf ? 1.0f : 0.0f;
    } else {
      const float ms = top == -kInf ? 0.0f : top;
      s *= __builtin_amdgcn_exp2f((m - ms) * kLog2e);
#pragma unroll
      for (int e = 0; e < N; ++e) s += __builtin_amdgcn_exp2f((v[e] - ms) * kLog2e);
    }
    m = top;
  }
  auto scan = [&](auto f) {
    for (int i0 = 0; i0 < n; i0 += STEP)
      some(i0, [&](int, float y, int i) {
        const uint32_t o = order_of(fmaxf(y, -kInf));
        f(o ? (uint64_t)o << 32 | (uint32_t)~(v0 + i) : 0ull);
      });
  };
  // (a part of one step is still in registers: counted first, so that a thread takes its places at once)
  auto quick = [&](uint32_t from) {
    if (n > STEP) {
      scan([&](uint64_t key) { add(L, key, (uint64_t)from << 32); });
      return;
    }
    const float low = value_of(from);
    int c = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) c += v[e] >= low;
    int at = atomicAdd(&L.n, c);
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (v[e] >= low) {
        const int i = SHORT ? e * kThreads + tid : (e / 8 * kThreads + tid) * 8 + e % 8;
        if (at < kCandidates) L.cand[at] = (uint64_t)order_of(v[e]) << 32 | (uint32_t)~(v0 + i);
        ++at;
      }
  };
  int have = gather(L, a.k, order_of(m), quick, scan);
  // the row's maximum and sum
  auto join_all = [&]() {
    const float M = wave_max(m);
    float x, y;
    s *= weight_of(m, M);
    s += lane_xor<1>(s);
    s += lane_xor<2>(s);
    s += lane_xor<4>(s);
    s += lane_xor<8>(s);
    lane_pair<16>(s, x, y);
    s = x + y;
    lane_pair<32>(s, x, y);
    s = x + y;
    if (lane == 0) L.m[wave] = M, L.s[wave] = s;
    __syncthreads();
    m = fmaxf(fmaxf(L.m[0], L.m[1]), fmaxf(L.m[2], L.m[3]));
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s += L.s[w] * weight_of(L.m[w], m);
  };
  join_all();
  if (a.chunks == 1) {
    sort_list(L, have, a.k);
    if (wave == 0) draw(a, L, b, m, s, temp, top_p, min_p, u);
    return;
  }
  // The candidates as they are, or where they are many more than k only those.  (One of each chunk after the other:
  // the last workgroup's threads then each see some of several.)
  const int cap = sample_list(a.k);
  const uint64_t* from = L.cand;
  if (have > cap) {
    sort_list(L, have, a.k);
    from = L.list;
    have = a.k;
  }
  uint64_t* keys = a.keys + (long long)b * a.chunks * cap;
  uint64_t* stats = a.stats + (long long)b * a.chunks;
  for (int i = tid; i < cap; i += kThreads)
    __hip_atomic_store(keys + i * a.chunks + chunk, i < have ? from[i] : 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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
  // all candidates, in registers: up to 24 of a thread
  constexpr int RUN = 8, RUNS = kSampleKeys / kThreads / RUN;
  static_assert(RUNS * RUN * kThreads == kSampleKeys, "a row's keys");
  const int all = a.chunks * cap;
  uint64_t key[RUNS][RUN];
#pragma unroll
  for (int r = 0; r < RUNS; ++r) {
    if (r * RUN * kThreads >= all) break;
#pragma unroll
    for (int e = 0; e < RUN; ++e)
      key[r][e] = __hip_atomic_load(keys + min((r * RUN + e) * kThreads + tid, all - 1), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  auto all_keys = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < RUNS; ++r) {
      if (r * RUN * kThreads >= all) break;
#pragma unroll
      for (int e = 0; e < RUN; ++e) f((r * RUN + e) * kThreads + tid < all ? key[r][e] : 0ull);
    }
  };
  uint32_t top = 0u;
  all_keys([&](uint64_t key) { top = max(top, (uint32_t)(key >> 32)); });
  m = -kInf, s = 0.0f;
  for (int i = tid; i < a.chunks; i += kThreads) {
    const uint64_t v = __hip_atomic_load(stats + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const float m2 = bitcast<float>((uint32_t)(v >> 32)), mn = fmaxf(m, m2);
    s = s * weight_of(m, mn) + bitcast<float>((uint32_t)v) * weight_of(m2, mn);
    m = mn;
  }
  join_all();
  auto reach = [&](uint32_t from) { all_keys([&](uint64_t key) { add(L, key, (uint64_t)from << 32); }); };
  const int found = gather(L, a.k, top, reach, all_keys);
  sort_list(L, found, a.k);
  if (wave == 0) draw(a, L, b, m, s, temp, top_p, min_p, u);
}

}  // namespace

template <int DT>
static void launch(const SampleArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.B * a.chunks)), block(kThreads);
  if (a.V <= 8 * kThreads) hipLaunchKernelGGL((sample_kernel<DT, true, 1>), grid, block, 0, st, a);
  else if (a.V <= (long long)kSampleTile * a.chunks) hipLaunchKernelGGL((sample_kernel<DT, false, 4>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((sample_kernel<DT, false, 8>), grid, block, 0, st, a);
}

hipError_t launch_sample(const SampleArgs& a, hipStream_t st) {
  if (a.xdt == DT_F32) launch<DT_F32>(a, st);
  else if (a.xdt == DT_BF16) launch<DT_BF16>(a, st);
  else launch<DT_F16>(a, st);
  return hipGetLastError();
}

}  // namespace qlin
