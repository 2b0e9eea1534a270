// Host/device shared definitions of the attention layer's middle (not part of the
// public ABI): per-head norm with rotary positions into a paged cache, prompt and
// decode attention.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qlin {

// One tensor of a paged cache: 16-bit or int8 values [pages][page][heads][hd] with any
// strides (elements; the last axis is contiguous), and the fp32 scales of an int8 one
// [pages][page][heads].
struct PagedTensor {
  void* p;
  long long sp, st, sh;   // page, token and head strides
  float* s;               // nullptr: 16-bit values
  long long ssp, sst, ssh;
};

// Per-head norm, rotary positions, cache write (rope.hip).
struct RopeArgs {
  const void* q;
  long long qt, qh;       // token and head strides (elements)
  const void* k;
  long long kt, kh;
  const void* v;          // nullptr: no values
  long long vt, vh;
  void* qo;
  long long qot, qoh;
  void* ko;               // nullptr: rotated keys go to the cache only
  long long kot, koh;
  PagedTensor kc, vc;     // p == nullptr: no cache
  long long nslots;       // pages * page
  int page_shift;
  const void* slots;      // [T]
  int slots64;
  const void* pos;        // [axes][T]
  long long pos_a, pos_t;
  int pos64;
  const void* freqs;      // [rot / 2]
  int freqs64;
  const void* qw;         // norm weights [hd] or nullptr (no norm)
  const void* kw;
  int wdt;
  int one_plus;
  float eps;
  int T, HQ, HKV, hd, rot;
  int axes, sec[3], interleaved;
  int dt;                 // DT_BF16 or DT_F16
};
hipError_t launch_rope(const RopeArgs& a, hipStream_t st);

// Where attention finds keys and values: packed rows [rows][heads][hd] (table ==
// nullptr; sequence b holds rows cu[b] .. cu[b + 1] - 1) or the pages table[b][...] of a
// cache (sequence b holds len[b] keys).
struct KvSrc {
  PagedTensor k, v;
  const int* table;
  long long table_stride;
  int num_pages, max_pages, page_shift;
  const int* len;
  const int* cu;
  int rows;               // packed: rows of k and v
};

// Attention of one token per sequence (attn_decode.hip).
struct DecodeArgs {
  const void* q;
  long long qb, qh;
  void* o;
  long long ob, oh;
  KvSrc kv;
  int B, HKV, G;          // G: query heads of a key head
  int gb;                 // groups of 16 query heads of a key head
  float c;                // scale * log2(e)
  int target;             // most work units of a (key head, group) to cut into; 0: no cut
  int few;                // units that short work is cut into
  int units;              // units per (key head, group): the grid's bound
  float* part;            // unit partials
  unsigned* cnt;          // arrival counters, zero between calls
};
// A part: rows x hd sums of 32 bits, then (reference of P, sum of P, 0, 0) of each row.
__host__ __device__ constexpr int decode_slot_floats(int rows, int hd) { return rows * hd + rows * 4; }
constexpr int kDecodeBlock = 32;     // keys a wave takes at a time
constexpr int kDecodeChunk = 4;      // blocks of a unit come in multiples of this (one per wave)
constexpr int kDecodeLong = 32;      // blocks of a unit up to which fewer units are better
constexpr int kDecodeGroup = 16;     // units joined at a time
constexpr int kDecodeCounters = 32;  // counters of a (sequence, key head, group)
hipError_t launch_decode(const DecodeArgs& a, int dt, int hd, hipStream_t st);

// Attention of one token per sequence, of groups that share a prefix (attn_shared*.hip).
struct SharedArgs {
  const void* q;
  long long qb, qh;
  void* o;
  long long ob, oh;
  KvSrc pre, own;         // one cache; pre: a group's table row and length, own: a sequence's
  const int* cu;          // [G + 1] sequences of each group
  int G, B, HKV, R;       // R: query heads of a key head
  int tiles;              // 16-row tiles of a prefix's unit: 1, 2, or 8 in the wide form
  int spt;                // sequences of a prefix's unit
  float c;                // scale * log2(e)
  int target, few;        // cuts of a key head's long and short work
  int brief;              // blocks of a unit up to which work is short
  int units;              // units per key head: the grid's bound
  long long own_rows;     // rows of parts of a key head in front of the own ones
  long long rows;         // rows of parts of a key head
  float* part;            // [key head][row][hd] sums
  float* ml;              // [key head][row][2] reference and sum of P
};
constexpr int kSharedBlock = 32;     // keys a wave takes at a time
constexpr int kSharedManyRows = 1024;  // rows of a call from which a workgroup joins several
constexpr int kSharedFewRows = 256;    // rows of a call up to which a join may take 512 threads,
constexpr int kSharedManyKeys = 4096;  // for prefixes (by their table) of more keys
hipError_t launch_shared_bf16(const SharedArgs& a, int hd, hipStream_t st);
hipError_t launch_shared_f16(const SharedArgs& a, int hd, hipStream_t st);
hipError_t launch_shared_wide_bf16(const SharedArgs& a, int hd, hipStream_t st);
hipError_t launch_shared_wide_f16(const SharedArgs& a, int hd, hipStream_t st);

// Attention of packed prompts over packed keys or a paged cache (attn_prompt*.hip).
struct PromptArgs {
  const void* q;
  long long qt, qh;       // token and head strides (elements)
  void* o;
  long long ot, oh;
  KvSrc kv;               // table == nullptr: packed keys, sequence b's at kv.cu
  const int* cu;          // [B + 1] rows of q of each sequence
  int T, B, HKV, G;
  int causal;
  float c;                // scale * log2(e)
  int target;             // work units to cut the keys into; 0: no cut
  int shortest;           // blocks of the shortest cut
  int gain;               // blocks that a cut has to take off the longest tile
  int units;              // units per key head: the grid's bound
  int rows;               // rows of a tile: kPromptRows, or half as many with two key groups
  int tiles;              // row tiles per key head at most
  int join_apart;         // parts are joined by a launch of its own
  float* part;            // unit partials [key head][unit]
  unsigned* cnt;          // arrival counters of each tile, zero between calls
};
constexpr int kPromptBlock = 32;     // keys of a step
constexpr int kPromptFewTiles = 96;  // tiles of all key heads up to which short cuts pay
constexpr int kPromptHalves = 272;   // halved tiles of all key heads up to which tiles are halved
constexpr int kPromptFill = 3000;    // (tile, block) pairs that fill the chip with whole tiles
constexpr int kPromptJoinApart = 256;  // row tiles of all key heads up to which a second launch joins
constexpr int kPromptCounters = 32;  // counters of a (key head, row tile)
constexpr int kPromptRows = 128;     // rows of a tile: tokens x the query heads of a key head
// a unit's partial: sums of its rows, then (reference of P, sum of P) of each
__host__ __device__ constexpr long long prompt_slot_floats(int hd, int rows) { return (long long)rows * (hd + 2); }
hipError_t launch_prompt(const PromptArgs& a, int dt, int hd, hipStream_t st);
hipError_t launch_prompt_bf16(const PromptArgs& a, int hd, hipStream_t st);
hipError_t launch_prompt_f16(const PromptArgs& a, int hd, hipStream_t st);

}  // namespace qlin
