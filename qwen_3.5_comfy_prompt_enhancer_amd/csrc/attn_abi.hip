// extern "C" entry points of the attention operators (declared in include/qlin_attn.h): checks
// of arguments and launch plans.
#include <math.h>
#include <stdlib.h>

#include <algorithm>

#include "../../include/qlin_attn.h"
#include "../../include/qlin_candidates.h"
#include "abi_check.h"
#include "attn_internal.h"
#include "qlin_dev.h"

using namespace qlin;

namespace {

constexpr int kMaxRows = (1 << 24) - 1;       // tokens of a call (rows of a key head stay below 2^31), and its
                                              // workgroups (a launch has less than 2^32 threads)
constexpr int kMaxHeads = 1 << 16;
constexpr int kMaxSeqs = 1 << 16;             // sequences of a call: every workgroup scans them for its own
constexpr int kMaxGroup = 64;                 // query heads of a key head
constexpr long long kMaxKeys = 1LL << 30;     // keys of a sequence
constexpr long long kMaxTokenStride = 1LL << 26;  // eight rows' offset stays in 32 bits
constexpr long long kMaxStride = (1LL << 31) - 16;  // of heads and pages: in bytes below 2^32

// One 16-bit (es = 2) or int8 tensor: n of the outer strides (that of an axis of one is never used).
// `write`: rows must not overlap.
int check_tensor(const char* fn, const char* name, const void* p, int es, int hd, long long n0, long long s0,
                 long long n1, long long s1, bool write) {
  const int mult = es == 1 ? 16 : 8;
  if (!p) return fail(QLIN_ERR_INVALID, "%s: null %s", fn, name);
  if (n0 <= 1) s0 = 0;
  if (n1 <= 1) s1 = 0;
  if (!aligned(p, 16) || s0 % mult || s1 % mult || s0 < 0 || s1 < 0)
    return fail(QLIN_ERR_UNSUPPORTED, "%s: %s must be 16-byte aligned with strides that are multiples of %d", fn, name,
                mult);
  if (s0 > kMaxTokenStride || s1 > kMaxStride)
    return fail(QLIN_ERR_UNSUPPORTED, "%s: strides of %s above %lld (rows) or %lld (heads)", fn, name, kMaxTokenStride,
                kMaxStride);
  if (write && ((n0 > 1 && s0 < hd) || (n1 > 1 && s1 < hd)))
    return fail(QLIN_ERR_INVALID, "%s: rows of %s overlap", fn, name);
  return QLIN_OK;
}

int check_heads(const char* fn, int hq, int hkv, int hd, int dtype) {
  if (hq <= 0 || hkv <= 0 || hq % hkv != 0)
    return fail(QLIN_ERR_INVALID, "%s: %d query heads must be a multiple of %d key heads", fn, hq, hkv);
  if (hq / hkv > kMaxGroup)
    return fail(QLIN_ERR_UNSUPPORTED, "%s: more than %d query heads to a key head", fn, kMaxGroup);
  if (hq > kMaxHeads) return fail(QLIN_ERR_UNSUPPORTED, "%s: more than %d query heads", fn, kMaxHeads);
  if (hd != 64 && hd != 128 && hd != 256)
    return fail(QLIN_ERR_UNSUPPORTED, "%s: head size %d (need 64, 128 or 256)", fn, hd);
  if (dtype != QLIN_BF16 && dtype != QLIN_F16)
    return fail(QLIN_ERR_UNSUPPORTED, "%s: dtype %d (need bf16 or fp16)", fn, dtype);
  return QLIN_OK;
}

int check_apart(const char* fn, const void* q, const void* out) {
  if (q == out) return fail(QLIN_ERR_INVALID, "%s: out must not be q (queries are read while others' outputs are written)", fn);
  return QLIN_OK;
}

int check_seqs(const char* fn, int B) {
  if (B > kMaxSeqs) return fail(QLIN_ERR_UNSUPPORTED, "%s: more than %d sequences", fn, kMaxSeqs);
  return QLIN_OK;
}

int check_grid(const char* fn, long long workgroups) {
  if (workgroups > kMaxRows) return fail(QLIN_ERR_UNSUPPORTED, "%s: too many rows for one launch", fn);
  return QLIN_OK;
}

int check_scale(const char* fn, float scale) {
  if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(QLIN_ERR_INVALID, "%s: scale must be positive", fn);
  return QLIN_OK;
}

int check_cache(const char* fn, const qlin_paged_kv* c, int hkv, int hd, int dtype, bool write, PagedTensor& k,
                PagedTensor& v) {
  if (!c) return fail(QLIN_ERR_INVALID, "%s: null cache", fn);
  if (c->dtype != QLIN_I8 && c->dtype != dtype)
    return fail(QLIN_ERR_UNSUPPORTED, "%s: cache dtype %d (need int8 or the queries' type)", fn, c->dtype);
  if (c->page < 16 || c->page > 1024 || (c->page & (c->page - 1)))
    return fail(QLIN_ERR_UNSUPPORTED, "%s: page of %d tokens (need a power of two from 16 to 1024)", fn, c->page);
  if (c->num_pages <= 0) return fail(QLIN_ERR_INVALID, "%s: a cache of no pages", fn);
  const bool q8 = c->dtype == QLIN_I8;
  const int es = q8 ? 1 : 2, mult = q8 ? 16 : 8;
  QA_TRY(check_tensor(fn, "k_cache", c->k, es, hd, c->page, c->k_token, hkv, c->k_head, write));
  QA_TRY(check_tensor(fn, "v_cache", c->v, es, hd, c->page, c->v_token, hkv, c->v_head, write));
  if (c->num_pages > 1) {
    if (c->k_page % mult || c->v_page % mult || c->k_page < 0 || c->v_page < 0)
      return fail(QLIN_ERR_UNSUPPORTED, "%s: page strides must be multiples of %d", fn, mult);
    if (c->k_page > kMaxStride || c->v_page > kMaxStride)
      return fail(QLIN_ERR_UNSUPPORTED, "%s: page strides above %lld", fn, kMaxStride);
    if (write && (c->k_page < hd || c->v_page < hd))
      return fail(QLIN_ERR_INVALID, "%s: pages of the cache overlap", fn);
  }
  if (q8) {
    if (!c->k_s || !c->v_s) return fail(QLIN_ERR_INVALID, "%s: an int8 cache needs k_s and v_s", fn);
    if (!aligned(c->k_s, 4) || !aligned(c->v_s, 4))
      return fail(QLIN_ERR_UNSUPPORTED, "%s: scales must be 4-byte aligned", fn);
    const int64_t st[6] = {c->ks_page, c->ks_token, c->ks_head, c->vs_page, c->vs_token, c->vs_head};
    const int n[3] = {c->num_pages, c->page, hkv};
    for (int i = 0; i < 6; ++i) {
      if (n[i % 3] <= 1) continue;
      if (st[i] < 0 || st[i] > (i % 3 == 1 ? kMaxTokenStride : kMaxStride / 2))
        return fail(QLIN_ERR_UNSUPPORTED, "%s: stride of the scales negative or too large", fn);
      if (write && st[i] < 1) return fail(QLIN_ERR_INVALID, "%s: scales of the cache overlap", fn);
    }
  } else if (c->k_s || c->v_s) {
    return fail(QLIN_ERR_INVALID, "%s: a 16-bit cache has no scales", fn);
  }
  k = PagedTensor{c->k, c->k_page, c->k_token, c->k_head, c->k_s, c->ks_page, c->ks_token, c->ks_head};
  v = PagedTensor{c->v, c->v_page, c->v_token, c->v_head, c->v_s, c->vs_page, c->vs_token, c->vs_head};
  return QLIN_OK;
}

int shift_of(int page) { return __builtin_ctz((unsigned)page); }

int check_paged(const char* fn, const qlin_paged_kv* cache, const int* table, int64_t table_stride, int max_pages,
                const int* kv_len, int hkv, int hd, int dtype, KvSrc& kv) {
  QA_TRY(check_cache(fn, cache, hkv, hd, dtype, false, kv.k, kv.v));
  if (max_pages == 0) table = kv_len;  // (a table of no pages is never read: no sequence has a key)
  if (!table || !kv_len) return fail(QLIN_ERR_INVALID, "%s: null page table or lengths", fn);
  if (!aligned(table, 4) || !aligned(kv_len, 4))
    return fail(QLIN_ERR_UNSUPPORTED, "%s: table and kv_len must be 4-byte aligned", fn);
  if (max_pages < 0 || table_stride < 0) return fail(QLIN_ERR_INVALID, "%s: negative page table size", fn);
  if ((long long)max_pages * cache->page > kMaxKeys)
    return fail(QLIN_ERR_UNSUPPORTED, "%s: more than %lld keys a sequence", fn, kMaxKeys);
  kv.table = table;
  kv.table_stride = table_stride;
  kv.num_pages = cache->num_pages;
  kv.max_pages = max_pages;
  kv.page_shift = shift_of(cache->page);
  kv.len = kv_len;
  kv.cu = nullptr;
  kv.rows = 0;
  return QLIN_OK;
}

// A cache's keys, values and scales.
struct CacheRegions {
  Region r[4];
  int n;
};
CacheRegions cache_regions(const qlin_paged_kv* c, int hkv, int hd) {
  const int es = c->dtype == QLIN_I8 ? 1 : 2;
  CacheRegions x = {{region("k_cache", c->k, es, hd, c->num_pages, c->k_page, c->page, c->k_token, hkv, c->k_head),
                     region("v_cache", c->v, es, hd, c->num_pages, c->v_page, c->page, c->v_token, hkv, c->v_head)},
                    2};
  if (c->dtype == QLIN_I8) {
    x.r[2] = region("k_s", c->k_s, 4, 1, c->num_pages, c->ks_page, c->page, c->ks_token, hkv, c->ks_head);
    x.r[3] = region("v_s", c->v_s, 4, 1, c->num_pages, c->vs_page, c->page, c->vs_token, hkv, c->vs_head);
    x.n = 4;
  }
  return x;
}
int check_cache_apart(const char* fn, const Region& a, const qlin_paged_kv* c, int hkv, int hd) {
  const CacheRegions x = cache_regions(c, hkv, hd);
  for (int i = 0; i < x.n; ++i) QA_TRY(check_regions(fn, a, x.r[i]));
  return QLIN_OK;
}

// Row tiles and key cuts of a prompt call.
int plan_prompt(const char* fn, PromptArgs& a, int hd, long long max_keys, void* ws, size_t ws_bytes) {
  char* part;
  size_t avail;
  QA_TRY(workspace_parts(fn, ws, ws_bytes, &part, &avail));
  // Units: about as many as run at once (two, three or four workgroups a CU by head size), fewer
  // where their sums are the larger; 8192 tokens, 256 values, 384 / 448 / 512 / 640 units: 315 (not
  // cut) / 258 / 265 / 283 us; 8192 tokens of 8 heads, 128 values, not cut / 384 / 448 / 512 / 576 / 640:
  // 196 / 193 / 170 / 181 / 174 / 165, 64 values, not cut / 448 / 512 / 640 / 768: 138 / 115 / 122 / 110 / 112.
  a.rows = kPromptRows;
  long long target = hd == 256 ? 448 : hd == 128 ? 512 : 640;
  // Few tiles (of 16-bit keys) are halved, two groups of waves sharing their keys: 512 tokens 20.8
  // -> 18.6 us, four prompts of 512 24.7 -> 19.9.  Beyond a halved tile for each CU, or with work
  // enough to fill the chip with whole ones (by what the host knows of it), that only moves twice the
  // keys (2048 tokens 44.5 -> 49.9, four chunks of 700 over 3000 keys 69 -> 94); sequences of few
  // rows leave half of a whole tile empty.  A CU then holds one workgroup, and units stay below
  // the CUs (100-token chunks, 192 / 256 units: 25.5 / 35.4).
  const long long rows = (long long)a.T * a.G, halves = (rows * 2 / kPromptRows + a.B) * a.HKV;
  const long long blocks = a.kv.table ? max_keys / kPromptBlock : max_keys / a.B / kPromptBlock / (a.causal ? 2 : 1);
  if (!a.kv.k.s && halves <= kPromptHalves &&
      (rows <= (long long)a.B * kPromptRows / 2 || halves * blocks / 2 <= kPromptFill)) {
    a.rows = kPromptRows / 2;
    target = 192;
  }
  if (const char* e = getenv("QLIN_PROMPT_UNITS")) {  // for tuning runs
    if (atoi(e) >= 0) target = atoi(e);
  }
  const long long tiles = (long long)a.T * a.G / a.rows + a.B, all = tiles * a.HKV;
  const long long slot = prompt_slot_floats(hd, a.rows) * 4;
  // A cut costs about as much as seven blocks, and gives less where most of the chip has a tile
  // already: so many blocks it has to take off the longest tile (128-row tiles; uncut / cut: 192
  // of 32 blocks 41 / 41 us, 188 of 47 56 / 48; 512 of 64 89 / 104, of 128 165 / 168, 534 of up to
  // 125 158 / 148, 314 of 157 171 / 129; halved tiles: 100 of 25 blocks 25.0 / 23.4, 116 of 29
  // 27.2 / 24.5, 264 of up to 29 28 / 37).
  const bool halved = a.rows < kPromptRows;
  a.shortest = all <= kPromptFewTiles ? 8 : all <= kPromptJoinApart ? 12 : 16;
  a.gain = all <= kPromptFewTiles ? 4 : halved ? 13 : all <= kPromptJoinApart ? 20 : 52;
  if (max_keys < (long long)(a.shortest + a.gain) * kPromptBlock) target = 0;
  // every unit of a key head has a slot: at most 2 target / HKV + tiles of them (and two more for
  // what the device's 32-bit estimate rounds)
  target = std::min(target, ((long long)avail / slot / a.HKV - tiles - 3) * a.HKV / 2);
  if (target <= a.HKV || all * kPromptCounters * 4 > (long long)counter_bytes()) target = 0;
  a.target = (int)target;
  a.tiles = (int)tiles;
  // A second launch joins where parts are many (see prompt_join_kernel): not where sequences of the average
  // length are too short for a cut (a launch that finds nothing to join costs 3 us), with an eighth for
  // batches of which only the longest is cut (1100, 950 and 800 tokens, this line / without the eighth: 37.8 /
  // 47.3 us, 1300, 900 and 600 37.2 / 44.3, three of 950, which are not cut, 41.4 / 38.4), nor for halved
  // tiles of small heads, whose few small parts their last one joins as quickly (1300 tokens, a
  // launch / the last part: 64 values 15.2 / 13.4 us, 128 20.2 / 18.4, 256 31.8 / 32.8).
  const long long average = a.kv.table ? max_keys : max_keys / a.B;
  a.join_apart = all <= kPromptJoinApart && average >= (long long)(a.shortest + a.gain) * kPromptBlock * 7 / 8 &&
                 (a.kv.table || hd == 256 || a.rows == kPromptRows);
  const long long units = tiles + (target ? (2 * target + a.HKV - 1) / a.HKV + 2 : 0);
  // (the grid is rounded up to the XCDs; few key heads share them)
  QA_TRY(check_grid(fn, units * a.HKV + 8));
  a.units = (int)units;
  a.part = (float*)part;
  a.cnt = (unsigned*)ws;
  return QLIN_OK;
}

// Row tiles and units of a decode step over shared prefixes.
int plan_shared(const char* fn, SharedArgs& a, int hd, int page, char* part, size_t avail) {
  const long long rows = (long long)((a.B + a.G - 1) / a.G) * a.R;  // of a prefix, on average
  // 17 to 32 rows take one unit of two tiles, or two of one, which read the keys twice (the second time from the L2) but
  // come two to a CU (of 256 values) and more even.  One / two tiles, us: of 256 values prefixes of 62 MB together 24.0 /
  // 26.3, 125 MB 33.7 / 40.2, 195 MB 52.4 / 44.0; of 128 one of 31 MB 16.4 / 17.1, 46 MB 18.8 / 19.0, 93 MB 30.2 / 26.0, six of
  // 23 MB 17.5 / 18.2, 70 MB 31.0 / 24.4; of 64 one of 11 MB 11.5 / 12.1, 23 MB 14.5 / 14.2, 48 MB 21.1 / 19.4, six of 17 MB
  // 14.0 / 13.9, 35 MB 21.6 / 17.8.  int8 keys are cheaper read than two tiles are kept in registers.
  // The average group's rows choose: one of 57 sequences beside seven of one takes 16-row tiles, and its prefix is loaded
  // for each of them, from the L2 but for the first (8 + 2 heads of 256 behind 8000 tokens each: 48.8 us, in two calls 28.2
  // and 26.7; eight of eight 34.7).
  const long long keys = std::max(1, a.pre.max_pages) * (long long)page, own = std::max(1, a.own.max_pages) * (long long)page;
  const bool q8 = a.own.k.s != nullptr;
  const long long bytes = (long long)a.G * keys * a.HKV * hd * 4;
  const bool two = rows > 16 && !q8 && bytes > (hd == 256 ? 160LL << 20 : 24LL << 20);
  a.tiles = a.R > 16 || rows > 32 ? 8 : two ? 2 : 1;
  a.spt = 16 * a.tiles / a.R;
  // One workgroup a CU as long as that makes units of at most `brief` blocks: more of them read no faster and leave more
  // sums to join (8 sequences behind 32000 tokens of 256 values, 256 / 512 units: 23.8 / 29.2 us).  Where vector work bounds
  // a wide unit (int8 keys, 64 values), three: 64 sequences behind 16384 tokens with 30 and with 1000 keys of their own, 512 and
  // 768 units: int8 of 256 values 48.2 / 50.6 and 70.0 / 48.1, of 128 64.0 / 57.4 and 66.6 / 65.5, of 64 60.7 / 50.9 and 62.3 /
  // 60.7, 16 bits of 64 38.2 / 34.1 and 38.2 / 39.9; not so 16 bits of 128 41.9 / 43.0 and 49.7 / 50.1, of 256 34.2 / 44.3 and
  // 52.1 / 51.2.  (512 instead of 256 for those: 40.5 and 49.5, 33.4 and 46.2; behind 50000 tokens 76.1 / 75.3, 52.8 / 55.8.
  // Where own keys are most of the work finer cuts would be better: 1000 of each behind 1000 tokens, 256 / 768 units: 45 / 31.)
  long long few = a.tiles == 8 && (q8 || hd == 64) ? 768 : 256, total = two && hd == 256 ? 256 : std::max(512LL, few);
  a.brief = q8 ? 24 : 32;
  if (const char* e = getenv("QLIN_SHARED_UNITS")) {  // for tuning runs
    if (atoi(e) > 0) few = total = atoi(e);
  }
  const long long tiles = a.B / a.spt + std::min(a.B, a.G);  // units of prefixes that are not cut
  const long long bound = tiles * ((keys + 4 * kSharedBlock - 1) / (4 * kSharedBlock)) +
                          a.B * ((own + 4 * kSharedBlock - 1) / (4 * kSharedBlock));
  long long target = std::min(std::max(1LL, total / a.HKV), bound);
  // Every unit leaves its rows' sums: a tile's and a sequence's uncut work, and at most `target` cuts.  (A group's
  // parts lie next to each other without room between them; a cut of a prefix leaves those of a tile's sequences.  Cuts are
  // whole numbers below total / chunk, in which total's rounding in 32 bits is less than a tenth.)  Fewer cuts where that is
  // more than the workspace holds.
  const long long row = (long long)hd * 4 + 8, cut = std::min(a.spt, a.B);
  target = std::min(target, ((long long)avail / row / a.HKV / a.R - 2LL * a.B) / (cut + 1));
  if (target < 1)
    return fail(QLIN_ERR_UNSUPPORTED, "%s: %d sequences of %d query heads are more than the workspace holds sums of", fn,
                a.B, a.HKV * a.R);
  a.target = (int)target;
  a.few = (int)std::min(std::max(1LL, few / a.HKV), target);
  a.own_rows = (target * cut + a.B) * a.R;
  a.rows = a.own_rows + (target + a.B) * a.R;
  const long long units = target + tiles + a.B + 2;
  QA_TRY(check_grid(fn, units * a.HKV));
  QA_TRY(check_grid(fn, (long long)a.B * a.HKV * a.R));
  a.units = (int)units;
  a.part = (float*)part;
  a.ml = (float*)(part + (long long)a.HKV * a.rows * hd * 4);
  return QLIN_OK;
}

}  // namespace

extern "C" {

int qlin_qk_norm_rope(const qlin_rope* r, const qlin_paged_kv* cache, void* stream) {
  const char* fn = "qlin_qk_norm_rope";
  set_error(QLIN_OK, "");
  if (!r) return fail(QLIN_ERR_INVALID, "%s: null arguments", fn);
  if (r->T < 0) return fail(QLIN_ERR_INVALID, "%s: negative size", fn);
  QA_TRY(check_heads(fn, r->q_heads, r->kv_heads, r->hd, r->dtype));
  if (r->rot < 0 || r->rot > r->hd || r->rot % 16)
    return fail(QLIN_ERR_UNSUPPORTED, "%s: %d rotated values (need a multiple of 16 up to the head size)", fn, r->rot);
  if (r->axes < 1 || r->axes > 3) return fail(QLIN_ERR_UNSUPPORTED, "%s: %d position axes (need 1 to 3)", fn, r->axes);
  int sum = 0;
  for (int i = 0; i < r->axes; ++i) {
    if (r->sections[i] < 0) return fail(QLIN_ERR_INVALID, "%s: negative section", fn);
    sum += r->sections[i];
    if (r->interleaved && i > 0 && r->sections[i] > 0 && r->axes * (r->sections[i] - 1) + i >= r->rot / 2)
      return fail(QLIN_ERR_INVALID, "%s: axis %d has no %d turns among %d frequencies", fn, i, r->sections[i],
                  r->rot / 2);
  }
  if (sum != r->rot / 2)
    return fail(QLIN_ERR_INVALID, "%s: sections add up to %d, not %d frequencies", fn, sum, r->rot / 2);
  if (r->T == 0) return QLIN_OK;
  if (r->T > kMaxRows) return fail(QLIN_ERR_UNSUPPORTED, "%s: more than %d tokens", fn, kMaxRows);
  QA_TRY(check_tensor(fn, "q", r->q, 2, r->hd, r->T, r->q_token, r->q_heads, r->q_head, false));
  QA_TRY(check_tensor(fn, "k", r->k, 2, r->hd, r->T, r->k_token, r->kv_heads, r->k_head, false));
  QA_TRY(check_tensor(fn, "q_out", r->q_out, 2, r->hd, r->T, r->qo_token, r->q_heads, r->qo_head, true));
  if (r->k_out) QA_TRY(check_tensor(fn, "k_out", r->k_out, 2, r->hd, r->T, r->ko_token, r->kv_heads, r->ko_head, true));
  if (!r->k_out && !cache) return fail(QLIN_ERR_INVALID, "%s: neither k_out nor a cache for the keys", fn);
  if (r->rot > 0 && (!r->pos || !r->freqs)) return fail(QLIN_ERR_INVALID, "%s: null positions or frequencies", fn);
  if (!aligned(r->pos, r->pos_64 ? 8 : 4) || !aligned(r->freqs, r->freqs_64 ? 8 : 4))
    return fail(QLIN_ERR_UNSUPPORTED, "%s: positions and frequencies must be aligned to their size", fn);
  if (r->q_w || r->k_w) {
    if (r->w_dtype != QLIN_BF16 && r->w_dtype != QLIN_F16 && r->w_dtype != QLIN_F32)
      return fail(QLIN_ERR_UNSUPPORTED, "%s: norm weight dtype %d", fn, r->w_dtype);
    if (!aligned(r->q_w, 16) || !aligned(r->k_w, 16))
      return fail(QLIN_ERR_UNSUPPORTED, "%s: norm weights must be 16-byte aligned", fn);
  }
  RopeArgs a = {};
  if (cache) {
    if (!r->v || !r->slots) return fail(QLIN_ERR_INVALID, "%s: a cache needs values and slots", fn);
    if (!aligned(r->slots, r->slots_64 ? 8 : 4))
      return fail(QLIN_ERR_UNSUPPORTED, "%s: slots must be aligned to their size", fn);
    QA_TRY(check_tensor(fn, "v", r->v, 2, r->hd, r->T, r->v_token, r->kv_heads, r->v_head, false));
    QA_TRY(check_cache(fn, cache, r->kv_heads, r->hd, r->dtype, true, a.kc, a.vc));
    a.page_shift = shift_of(cache->page);
    a.nslots = (long long)cache->num_pages * cache->page;
  }
  a.q = r->q, a.qt = r->q_token, a.qh = r->q_head;
  a.k = r->k, a.kt = r->k_token, a.kh = r->k_head;
  a.v = cache ? r->v : nullptr, a.vt = r->v_token, a.vh = r->v_head;
  a.qo = r->q_out, a.qot = r->qo_token, a.qoh = r->qo_head;
  a.ko = r->k_out, a.kot = r->ko_token, a.koh = r->ko_head;
  a.slots = r->slots, a.slots64 = r->slots_64;
  a.pos = r->pos, a.pos_a = r->pos_axis, a.pos_t = r->pos_token, a.pos64 = r->pos_64;
  a.freqs = r->freqs, a.freqs64 = r->freqs_64;
  a.qw = r->q_w, a.kw = r->k_w, a.wdt = r->w_dtype, a.one_plus = r->one_plus, a.eps = r->eps;
  a.T = r->T, a.HQ = r->q_heads, a.HKV = r->kv_heads, a.hd = r->hd, a.rot = r->rot;
  a.axes = r->axes, a.interleaved = r->interleaved, a.dt = r->dtype;
  for (int i = 0; i < 3; ++i) a.sec[i] = i < r->axes ? r->sections[i] : 0;
  // What is written, and what it may be: q_out q itself, k_out k itself (each head is read before it is
  // written, by the same threads).
  const Region q = region("q", r->q, 2, r->hd, r->T, r->q_token, r->q_heads, r->q_head);
  const Region k = region("k", r->k, 2, r->hd, r->T, r->k_token, r->kv_heads, r->k_head);
  const Region v = region("v", a.v, 2, r->hd, r->T, r->v_token, r->kv_heads, r->v_head);
  const Region qo = region("q_out", r->q_out, 2, r->hd, r->T, r->qo_token, r->q_heads, r->qo_head);
  const Region ko = region("k_out", r->k_out, 2, r->hd, r->T, r->ko_token, r->kv_heads, r->ko_head);
  auto same = [](const Region& x, const Region& y) { return x.p == y.p && x.s[0] == y.s[0] && x.s[1] == y.s[1]; };
  QA_TRY(check_region(fn, qo));
  if (!same(qo, q)) QA_TRY(check_regions(fn, qo, q));
  QA_TRY(check_regions(fn, qo, k));
  QA_TRY(check_regions(fn, qo, v));
  if (r->k_out) {
    QA_TRY(check_region(fn, ko));
    if (!same(ko, k)) QA_TRY(check_regions(fn, ko, k));
    QA_TRY(check_regions(fn, ko, q));
    QA_TRY(check_regions(fn, ko, v));
    QA_TRY(check_regions(fn, ko, qo));
  }
  if (cache) {
    const CacheRegions x = cache_regions(cache, r->kv_heads, r->hd);
    for (int i = 0; i < x.n; ++i) {
      QA_TRY(check_region(fn, x.r[i]));
      for (const Region* y : {&q, &k, &v, &qo, &ko}) QA_TRY(check_regions(fn, *y, x.r[i]));
      for (int j = 0; j < i; ++j) QA_TRY(check_regions(fn, x.r[j], x.r[i]));
    }
  }
  return status(fn, launch_rope(a, (hipStream_t)stream));
}

int qlin_attn_prompt(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                     const void* v, int64_t v_token, int64_t v_head, const int* cu_q, const int* cu_k, void* out,
                     int64_t o_token, int64_t o_head, int T, int Tk, int B, int q_heads, int kv_heads, int hd,
                     int dtype, float scale, int causal, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "qlin_attn_prompt";
  set_error(QLIN_OK, "");
  if (T < 0 || Tk < 0 || B < 0) return fail(QLIN_ERR_INVALID, "%s: negative size", fn);
  QA_TRY(check_heads(fn, q_heads, kv_heads, hd, dtype));
  QA_TRY(check_scale(fn, scale));
  if (T == 0 || B == 0) return QLIN_OK;
  if (T > kMaxRows || Tk > kMaxRows) return fail(QLIN_ERR_UNSUPPORTED, "%s: more than %d tokens", fn, kMaxRows);
  QA_TRY(check_seqs(fn, B));
  if (!cu_q || !cu_k) return fail(QLIN_ERR_INVALID, "%s: null row bounds", fn);
  if (!aligned(cu_q, 4) || !aligned(cu_k, 4))
    return fail(QLIN_ERR_UNSUPPORTED, "%s: row bounds must be 4-byte aligned", fn);
  QA_TRY(check_tensor(fn, "q", q, 2, hd, T, q_token, q_heads, q_head, false));
  QA_TRY(check_tensor(fn, "out", out, 2, hd, T, o_token, q_heads, o_head, true));
  QA_TRY(check_apart(fn, q, out));
  if (Tk > 0) {
    QA_TRY(check_tensor(fn, "k", k, 2, hd, Tk, k_token, kv_heads, k_head, false));
    QA_TRY(check_tensor(fn, "v", v, 2, hd, Tk, v_token, kv_heads, v_head, false));
  }
  PromptArgs a = {};
  a.q = q, a.qt = q_token, a.qh = q_head;
  a.o = out, a.ot = o_token, a.oh = o_head;
  a.kv.k = PagedTensor{const_cast<void*>(k), 0, k_token, k_head, nullptr, 0, 0, 0};
  a.kv.v = PagedTensor{const_cast<void*>(v), 0, v_token, v_head, nullptr, 0, 0, 0};
  a.kv.cu = cu_k, a.kv.rows = Tk;
  a.cu = cu_q, a.T = T, a.B = B, a.HKV = kv_heads, a.G = q_heads / kv_heads;
  a.causal = causal, a.c = scale * 1.44269504088896340736f;
  QA_TRY(plan_prompt(fn, a, hd, Tk, workspace, workspace_bytes));
  const Region to = region("out", out, 2, hd, T, o_token, q_heads, o_head);
  QA_TRY(check_region(fn, to));
  QA_TRY(check_regions(fn, to, region("q", q, 2, hd, T, q_token, q_heads, q_head)));
  if (Tk > 0) {
    QA_TRY(check_regions(fn, to, region("k", k, 2, hd, Tk, k_token, kv_heads, k_head)));
    QA_TRY(check_regions(fn, to, region("v", v, 2, hd, Tk, v_token, kv_heads, v_head)));
  }
  return status(fn, launch_prompt(a, dtype, hd, (hipStream_t)stream));
}

int qlin_attn_prompt_paged(const void* q, int64_t q_token, int64_t q_head, const qlin_paged_kv* cache,
                           const int* table, int64_t table_stride, int max_pages, const int* kv_len, const int* cu_q,
                           void* out, int64_t o_token, int64_t o_head, int T, int B, int q_heads, int kv_heads,
                           int hd, int dtype, float scale, int causal, void* workspace, size_t workspace_bytes,
                           void* stream) {
  const char* fn = "qlin_attn_prompt_paged";
  set_error(QLIN_OK, "");
  if (T < 0 || B < 0) return fail(QLIN_ERR_INVALID, "%s: negative size", fn);
  QA_TRY(check_heads(fn, q_heads, kv_heads, hd, dtype));
  QA_TRY(check_scale(fn, scale));
  if (T == 0 || B == 0) return QLIN_OK;
  if (T > kMaxRows) return fail(QLIN_ERR_UNSUPPORTED, "%s: more than %d tokens", fn, kMaxRows);
  QA_TRY(check_seqs(fn, B));
  if (!cu_q) return fail(QLIN_ERR_INVALID, "%s: null row bounds", fn);
  if (!aligned(cu_q, 4)) return fail(QLIN_ERR_UNSUPPORTED, "%s: row bounds must be 4-byte aligned", fn);
  QA_TRY(check_tensor(fn, "q", q, 2, hd, T, q_token, q_heads, q_head, false));
  QA_TRY(check_tensor(fn, "out", out, 2, hd, T, o_token, q_heads, o_head, true));
  QA_TRY(check_apart(fn, q, out));
  PromptArgs a = {};
  QA_TRY(check_paged(fn, cache, table, table_stride, max_pages, kv_len, kv_heads, hd, dtype, a.kv));
  a.q = q, a.qt = q_token, a.qh = q_head;
  a.o = out, a.ot = o_token, a.oh = o_head;
  a.cu = cu_q, a.T = T, a.B = B, a.HKV = kv_heads, a.G = q_heads / kv_heads;
  a.causal = causal, a.c = scale * 1.44269504088896340736f;
  QA_TRY(plan_prompt(fn, a, hd, (long long)max_pages * cache->page, workspace, workspace_bytes));
  const Region to = region("out", out, 2, hd, T, o_token, q_heads, o_head);
  QA_TRY(check_region(fn, to));
  QA_TRY(check_regions(fn, to, region("q", q, 2, hd, T, q_token, q_heads, q_head)));
  QA_TRY(check_cache_apart(fn, to, cache, kv_heads, hd));
  return status(fn, launch_prompt(a, dtype, hd, (hipStream_t)stream));
}

int qlin_attn_decode(const void* q, int64_t q_seq, int64_t q_head, const qlin_paged_kv* cache, const int* table,
                     int64_t table_stride, int max_pages, const int* kv_len, void* out, int64_t o_seq,
                     int64_t o_head, int B, int q_heads, int kv_heads, int hd, int dtype, float scale,
                     void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "qlin_attn_decode";
  set_error(QLIN_OK, "");
  if (B < 0) return fail(QLIN_ERR_INVALID, "%s: negative size", fn);
  QA_TRY(check_heads(fn, q_heads, kv_heads, hd, dtype));
  QA_TRY(check_scale(fn, scale));
  if (B == 0) return QLIN_OK;
  QA_TRY(check_seqs(fn, B));
  QA_TRY(check_tensor(fn, "q", q, 2, hd, B, q_seq, q_heads, q_head, false));
  QA_TRY(check_tensor(fn, "out", out, 2, hd, B, o_seq, q_heads, o_head, true));
  QA_TRY(check_apart(fn, q, out));
  DecodeArgs a = {};
  QA_TRY(check_paged(fn, cache, table, table_stride, max_pages, kv_len, kv_heads, hd, dtype, a.kv));
  char* part;
  size_t avail;
  QA_TRY(workspace_parts(fn, workspace, workspace_bytes, &part, &avail));
  a.q = q, a.qb = q_seq, a.qh = q_head;
  a.o = out, a.ob = o_seq, a.oh = o_head;
  a.B = B, a.HKV = kv_heads, a.G = q_heads / kv_heads;
  a.gb = (a.G + 15) / 16;
  a.c = scale * 1.44269504088896340736f;
  const long long hg = (long long)kv_heads * a.gb;
  const long long blocks = ((long long)max_pages * cache->page + kDecodeBlock - 1) / kDecodeBlock;
  const long long bound = std::max(1LL, B * ((blocks + kDecodeChunk - 1) / kDecodeChunk));
  long long few = 256, total = 1536;
  if (const char* e = getenv("QLIN_DECODE_UNITS")) {  // for tuning runs
    if (atoi(e) > 0) few = total = atoi(e);
  }
  long long target = std::min(std::max(1LL, total / hg), bound);
  const long long slot = (long long)decode_slot_floats(std::min(16, a.G), hd) * 4;
  // without room for the parts (very many sequences) every sequence is one unit
  if ((target + B + 2) * hg * slot > (long long)avail || B * hg * kDecodeCounters * 4 > (long long)counter_bytes())
    target = 0;
  QA_TRY(check_grid(fn, (target + B + 2) * hg));
  const Region to = region("out", out, 2, hd, B, o_seq, q_heads, o_head);
  QA_TRY(check_region(fn, to));
  QA_TRY(check_regions(fn, to, region("q", q, 2, hd, B, q_seq, q_heads, q_head)));
  QA_TRY(check_cache_apart(fn, to, cache, kv_heads, hd));
  a.target = (int)target;
  a.few = (int)std::min(std::max(1LL, few / hg), std::max(1LL, target));
  a.units = (int)(target + B + (target ? 2 : 0));  // (two for what the device's estimate rounds)
  a.part = (float*)part;
  a.cnt = (unsigned*)workspace;
  return status(fn, launch_decode(a, dtype, hd, (hipStream_t)stream));
}

int qlin_attn_decode_shared(const void* q, int64_t q_seq, int64_t q_head, const qlin_paged_kv* cache,
                            const int* prefix_table, int64_t prefix_table_stride, int max_prefix_pages,
                            const int* prefix_len, const int* cu_seq, int G, const int* table, int64_t table_stride,
                            int max_pages, const int* kv_len, void* out, int64_t o_seq, int64_t o_head, int B,
                            int q_heads, int kv_heads, int hd, int dtype, float scale, void* workspace,
                            size_t workspace_bytes, void* stream) {
  const char* fn = "qlin_attn_decode_shared";
  set_error(QLIN_OK, "");
  if (B < 0 || G < 0) return fail(QLIN_ERR_INVALID, "%s: negative size", fn);
  QA_TRY(check_heads(fn, q_heads, kv_heads, hd, dtype));
  QA_TRY(check_scale(fn, scale));
  if (B == 0 || G == 0) return QLIN_OK;
  QA_TRY(check_seqs(fn, B));
  if (G > kMaxSeqs) return fail(QLIN_ERR_UNSUPPORTED, "%s: more than %d groups", fn, kMaxSeqs);
  if (!cu_seq) return fail(QLIN_ERR_INVALID, "%s: null sequence bounds", fn);
  if (!aligned(cu_seq, 4)) return fail(QLIN_ERR_UNSUPPORTED, "%s: sequence bounds must be 4-byte aligned", fn);
  QA_TRY(check_tensor(fn, "q", q, 2, hd, B, q_seq, q_heads, q_head, false));
  QA_TRY(check_tensor(fn, "out", out, 2, hd, B, o_seq, q_heads, o_head, true));
  QA_TRY(check_apart(fn, q, out));
  SharedArgs a = {};
  QA_TRY(check_paged(fn, cache, prefix_table, prefix_table_stride, max_prefix_pages, prefix_len, kv_heads, hd, dtype,
                     a.pre));
  QA_TRY(check_paged(fn, cache, table, table_stride, max_pages, kv_len, kv_heads, hd, dtype, a.own));
  const Region to = region("out", out, 2, hd, B, o_seq, q_heads, o_head);
  QA_TRY(check_region(fn, to));
  QA_TRY(check_regions(fn, to, region("q", q, 2, hd, B, q_seq, q_heads, q_head)));
  QA_TRY(check_cache_apart(fn, to, cache, kv_heads, hd));
  // (the second launch reads lengths and bounds again, beside workgroups that write)
  const Region in[5] = {region("prefix_table", max_prefix_pages ? prefix_table : nullptr, 4, max_prefix_pages, G, prefix_table_stride, 1, 0),
                        region("table", max_pages ? table : nullptr, 4, max_pages, B, table_stride, 1, 0),
                        region("prefix_len", prefix_len, 4, G, 1, 0, 1, 0), region("kv_len", kv_len, 4, B, 1, 0, 1, 0),
                        region("cu_seq", cu_seq, 4, G + 1, 1, 0, 1, 0)};
  for (const Region& r : in) QA_TRY(check_regions(fn, to, r));
  char* part;
  size_t avail;
  QA_TRY(workspace_parts(fn, workspace, workspace_bytes, &part, &avail));
  a.q = q, a.qb = q_seq, a.qh = q_head;
  a.o = out, a.ob = o_seq, a.oh = o_head;
  a.cu = cu_seq, a.G = G, a.B = B, a.HKV = kv_heads, a.R = q_heads / kv_heads;
  a.c = scale * 1.44269504088896340736f;
  QA_TRY(plan_shared(fn, a, hd, cache->page, part, avail));
  return status(fn, dtype == QLIN_BF16 ? launch_shared_bf16(a, hd, (hipStream_t)stream)
                                       : launch_shared_f16(a, hd, (hipStream_t)stream));
}

}  // extern "C"
