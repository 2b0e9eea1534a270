// Host/device shared definitions of what lies between the vocabulary head and the next token
// (not part of the public ABI).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qlin {

// A number of each row: a vector on the device, or one number for all.
struct RowValue {
  const float* p;
  float v;
  __device__ __forceinline__ float at(int b) const { return p ? p[b] : v; }
};

// Penalties, biases and masks (logits.hip).
struct LogitsArgs {
  const void* x;
  long long xs;           // row strides, in elements
  int xdt;                // DT_*
  void* o;
  long long os;
  int odt;
  int B, V;
  const void* tokens;     // [B][L], or nullptr
  long long ts;
  int tokens64, L;
  const int* lens;        // nullptr: L
  const int* prompt_lens; // nullptr: 0
  RowValue rep, pres, freq;
  const int* bias_ids;    // [B][nb]
  long long bis;
  const float* bias;
  long long bs;
  int nb;
  const void* mask;       // nullptr: every token is allowed
  long long ms;           // row stride: words, or bytes
  int mask_bytes;         // 1: a byte for each token, 0: a bit
};
constexpr int kLogitsRun = 2048;    // tokens of a workgroup at least
hipError_t launch_logits(const LogitsArgs& a, hipStream_t st);

// Drawing a token of each row (sample.hip).
struct SampleArgs {
  const void* x;
  long long xs;
  int xdt;
  int B, V, k;
  const float* u;
  RowValue temp, top_p, min_p;
  void* tokens;
  int tokens64;
  float* logp;            // or nullptr
  int chunks;             // workgroups of a row
  uint64_t* keys;         // [B][sample_list(k)][chunks] the largest of each chunk among them
  uint64_t* stats;        // [B][chunks] maximum and sum
  unsigned* cnt;          // arrivals of each row, zero between calls
};
constexpr int kSampleTile = 8192;   // logits that a workgroup keeps in registers (or twice as many)
constexpr int kSampleMost = 128;    // largest k
constexpr int kSampleKeys = 6144;   // keys of a row's chunks at most
// keys that a chunk leaves room for
__host__ __device__ constexpr int sample_list(int k) { return k + k / 2 + 4; }
hipError_t launch_sample(const SampleArgs& a, hipStream_t st);

}  // namespace qlin
