// extern "C" entry points of what lies between the vocabulary head and the next token (declared in
// include/qlin_candidates.h): checks of arguments and launch plans.
#include <algorithm>
#include <cmath>

#include "../../include/qlin_candidates.h"
#include "abi_check.h"
#include "qlin_dev.h"
#include "step_internal.h"

using namespace qlin;

namespace {

constexpr int kMaxRows = 1 << 16;
constexpr int kMaxTokens = 1 << 30;                   // of a vocabulary or a history
constexpr long long kMaxGrid = (1 << 24) - 1;         // a launch has less than 2^32 threads

int bytes_of(int dt) { return dt == QLIN_F32 ? 4 : 2; }

// Rows of n elements of es bytes at stride (elements); `write`: rows must not overlap.
int check_rows(const char* fn, const char* name, const void* p, int es, long long n, long long rows, long long stride,
               bool write) {
  if (!p) return fail(QLIN_ERR_INVALID, "%s: null %s", fn, name);
  if (!aligned(p, (size_t)es)) return fail(QLIN_ERR_UNSUPPORTED, "%s: %s must be %d-byte aligned", fn, name, es);
  if (rows > 1 && (stride < 0 || (write && stride < n)))
    return fail(QLIN_ERR_INVALID, "%s: rows of %s overlap", fn, name);
  return QLIN_OK;
}

int check_float(const char* fn, const char* name, int dt) {
  if (dt != QLIN_F32 && dt != QLIN_BF16 && dt != QLIN_F16)
    return fail(QLIN_ERR_UNSUPPORTED, "%s: %s of dtype %d (need bf16, fp16 or fp32)", fn, name, dt);
  return QLIN_OK;
}

int check_sizes(const char* fn, int B, int V) {
  if (B < 0 || V < 0) return fail(QLIN_ERR_INVALID, "%s: negative size", fn);
  if (B > kMaxRows) return fail(QLIN_ERR_UNSUPPORTED, "%s: more than %d rows", fn, kMaxRows);
  if (V > kMaxTokens) return fail(QLIN_ERR_UNSUPPORTED, "%s: a vocabulary of more than %d tokens", fn, kMaxTokens);
  return QLIN_OK;
}

// A number of each row, or one for all (`least` .. `most`, finite).
int check_value(const char* fn, const char* name, const float* p, float v, float least, float most) {
  if (p) return aligned(p, 4) ? QLIN_OK : fail(QLIN_ERR_UNSUPPORTED, "%s: %s must be 4-byte aligned", fn, name);
  if (!(v >= least && v <= most) || !std::isfinite(v))
    return fail(QLIN_ERR_INVALID, "%s: %s must be from %g to %g", fn, name, least, most);
  return QLIN_OK;
}

constexpr float kAny = 3.4028235e38f;

}  // namespace

extern "C" {

int qlin_logits_process(const qlin_logits* r, void* stream) {
  const char* fn = "qlin_logits_process";
  set_error(QLIN_OK, "");
  if (!r) return fail(QLIN_ERR_INVALID, "%s: null arguments", fn);
  QA_TRY(check_sizes(fn, r->B, r->V));
  QA_TRY(check_float(fn, "logits", r->dtype));
  QA_TRY(check_float(fn, "out", r->out_dtype));
  if (r->history < 0 || r->biases < 0) return fail(QLIN_ERR_INVALID, "%s: negative size", fn);
  if (r->history > kMaxTokens || r->biases > kMaxTokens)
    return fail(QLIN_ERR_UNSUPPORTED, "%s: more than %d tokens of a row's history or biases", fn, kMaxTokens);
  QA_TRY(check_value(fn, "repetition", r->repetition, r->repetition_all, 1.1754944e-38f, kAny));
  QA_TRY(check_value(fn, "presence", r->presence, r->presence_all, -kAny, kAny));
  QA_TRY(check_value(fn, "frequency", r->frequency, r->frequency_all, -kAny, kAny));
  if (r->B == 0 || r->V == 0) return QLIN_OK;
  const int xb = bytes_of(r->dtype), ob = bytes_of(r->out_dtype);
  QA_TRY(check_rows(fn, "logits", r->logits, xb, r->V, r->B, r->logits_row, false));
  QA_TRY(check_rows(fn, "out", r->out, ob, r->V, r->B, r->out_row, true));
  const bool tokens = r->tokens && r->history > 0, bias = r->biases > 0, bits = r->mask && !r->mask_bytes;
  const int tb = r->tokens_64 ? 8 : 4;
  if (r->history > 0) QA_TRY(check_rows(fn, "tokens", r->tokens, tb, r->history, r->B, r->tokens_row, false));
  if (!aligned(r->lens, 4) || !aligned(r->prompt_lens, 4))
    return fail(QLIN_ERR_UNSUPPORTED, "%s: lengths must be 4-byte aligned", fn);
  if (bias) {
    QA_TRY(check_rows(fn, "bias_ids", r->bias_ids, 4, r->biases, r->B, r->bias_ids_row, false));
    QA_TRY(check_rows(fn, "bias", r->bias, 4, r->biases, r->B, r->bias_row, false));
  }
  const int words = (int)(((long long)r->V + 31) / 32);
  if (r->mask) QA_TRY(check_rows(fn, "mask", r->mask, bits ? 4 : 1, bits ? words : r->V, r->B, r->mask_row, false));
  // What is written is apart from what is read, but that it may be the logits themselves.
  const Region to = region("out", r->out, ob, r->V, r->B, r->out_row, 1, 0);
  const bool same = r->out == r->logits && r->dtype == r->out_dtype && (r->B == 1 || r->out_row == r->logits_row);
  if (!same) QA_TRY(check_regions(fn, to, region("logits", r->logits, xb, r->V, r->B, r->logits_row, 1, 0)));
  if (tokens) {
    QA_TRY(check_regions(fn, to, region("tokens", r->tokens, tb, r->history, r->B, r->tokens_row, 1, 0)));
    const struct { const char* name; const void* p; } each[5] = {{"lens", r->lens}, {"prompt_lens", r->prompt_lens},
        {"repetition", r->repetition}, {"presence", r->presence}, {"frequency", r->frequency}};
    for (const auto& x : each) QA_TRY(check_regions(fn, to, region(x.name, x.p, 4, r->B, 1, 0, 1, 0)));
  }
  if (bias) {
    QA_TRY(check_regions(fn, to, region("bias_ids", r->bias_ids, 4, r->biases, r->B, r->bias_ids_row, 1, 0)));
    QA_TRY(check_regions(fn, to, region("bias", r->bias, 4, r->biases, r->B, r->bias_row, 1, 0)));
  }
  if (r->mask)
    QA_TRY(check_regions(fn, to, region("mask", r->mask, bits ? 4 : 1, bits ? words : r->V, r->B, r->mask_row, 1, 0)));
  LogitsArgs a = {};
  a.x = r->logits, a.xs = r->logits_row, a.xdt = r->dtype;
  a.o = r->out, a.os = r->out_row, a.odt = r->out_dtype;
  a.B = r->B, a.V = r->V;
  if (tokens) {
    a.tokens = r->tokens, a.ts = r->tokens_row, a.tokens64 = r->tokens_64, a.L = r->history;
    a.lens = r->lens, a.prompt_lens = r->prompt_lens;
  }
  a.rep = RowValue{r->repetition, r->repetition_all};
  a.pres = RowValue{r->presence, r->presence_all};
  a.freq = RowValue{r->frequency, r->frequency_all};
  if (bias) a.bias_ids = r->bias_ids, a.bis = r->bias_ids_row, a.bias = r->bias, a.bs = r->bias_row, a.nb = r->biases;
  a.mask = r->mask, a.ms = r->mask_row, a.mask_bytes = r->mask_bytes;
  const long long tiles = ((long long)a.V + kLogitsRun - 1) / kLogitsRun;
  if (tiles * a.B > kMaxGrid) return fail(QLIN_ERR_UNSUPPORTED, "%s: too many logits for one launch", fn);
  return status(fn, launch_logits(a, (hipStream_t)stream));
}

int qlin_sample(const void* logits, int dtype, int64_t logits_row, int B, int V, int top_k, const float* u,
                const float* temperature, float temperature_all, const float* top_p, float top_p_all,
                const float* min_p, float min_p_all, void* tokens, int tokens_64, float* logprobs, void* workspace,
                size_t workspace_bytes, void* stream) {
  const char* fn = "qlin_sample";
  set_error(QLIN_OK, "");
  QA_TRY(check_sizes(fn, B, V));
  QA_TRY(check_float(fn, "logits", dtype));
  if (top_k < 1 || top_k > kSampleMost)
    return fail(QLIN_ERR_UNSUPPORTED, "%s: top_k %d (need 1 to %d)", fn, top_k, kSampleMost);
  QA_TRY(check_value(fn, "temperature", temperature, temperature_all, 0.0f, kAny));
  QA_TRY(check_value(fn, "top_p", top_p, top_p_all, 0.0f, kAny));
  QA_TRY(check_value(fn, "min_p", min_p, min_p_all, 0.0f, kAny));
  if (B == 0) return QLIN_OK;
  if (V == 0) return fail(QLIN_ERR_INVALID, "%s: an empty vocabulary", fn);
  QA_TRY(check_rows(fn, "logits", logits, bytes_of(dtype), V, B, logits_row, false));
  QA_TRY(check_rows(fn, "u", u, 4, B, 1, 0, false));
  const int tb = tokens_64 ? 8 : 4;
  QA_TRY(check_rows(fn, "tokens", tokens, tb, B, 1, 0, true));
  if (!aligned(logprobs, 4)) return fail(QLIN_ERR_UNSUPPORTED, "%s: logprobs must be 4-byte aligned", fn);
  const Region x = region("logits", logits, bytes_of(dtype), V, B, logits_row, 1, 0);
  const Region to = region("tokens", tokens, tb, B, 1, 0, 1, 0), lo = region("logprobs", logprobs, 4, B, 1, 0, 1, 0);
  const Region in[5] = {x, region("u", u, 4, B, 1, 0, 1, 0), region("temperature", temperature, 4, B, 1, 0, 1, 0),
                        region("top_p", top_p, 4, B, 1, 0, 1, 0), region("min_p", min_p, 4, B, 1, 0, 1, 0)};
  for (const Region& i : in) {
    QA_TRY(check_regions(fn, to, i));
    QA_TRY(check_regions(fn, lo, i));
  }
  QA_TRY(check_regions(fn, to, lo));
  char* part;
  size_t avail;
  QA_TRY(workspace_parts(fn, workspace, workspace_bytes, &part, &avail));
  SampleArgs a = {};
  a.x = logits, a.xs = logits_row, a.xdt = dtype;
  a.B = B, a.V = V, a.k = std::min(top_k, V);
  a.u = u;
  a.temp = RowValue{temperature, temperature_all};
  a.top_p = RowValue{top_p, top_p_all};
  a.min_p = RowValue{min_p, min_p_all};
  a.tokens = tokens, a.tokens64 = tokens_64, a.logp = logprobs;
  // A workgroup for each part of a row that a workgroup keeps in registers, fewer where their lists would be more than
  // one can join or than the workspace holds.  Long parts where they fill the chip: fewer lists, and all workgroups at
  // once (248320 fp32 logits, parts of 8192 / 16384: one row 11.4 / 13, 16 rows 20.2 / 18.9 us, 64 33.7 / 26.4; 64 rows of
  // 100003 19.0 / 19.4, 8 13.4 / 15.1).
  const long long tiles = ((long long)V + kSampleTile - 1) / kSampleTile, half = (tiles + 1) / 2;
  const long long keys = sample_list(a.k), list = 8 * (keys + 1);
  const long long parts = half > 8 && half * B >= 256 ? half : tiles;
  const long long chunks = std::min({parts, (long long)kSampleKeys / keys, (long long)avail / list / B, kMaxGrid / B});
  if (chunks < 1) return fail(QLIN_ERR_WORKSPACE, "%s: workspace too small for %d rows", fn, B);
  a.chunks = (int)chunks;
  a.keys = (uint64_t*)part;
  a.stats = (uint64_t*)part + (long long)B * chunks * keys;
  a.cnt = (unsigned*)workspace;  // (kMaxRows of them are a quarter of the counters there are)
  return status(fn, launch_sample(a, (hipStream_t)stream));
}

}  // extern "C"
