// What the entry points of the attention operators and of the steps behind the vocabulary head check
// and report with.
#pragma once

#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>

#include "../../include/qlin.h"
#include "qlin_internal.h"

namespace qlin {

namespace {

int fail(int code, const char* fmt, ...) {
  char msg[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  return set_error(code, msg);
}

int status(const char* fn, hipError_t e) {
  if (e == hipSuccess) return QLIN_OK;
  return fail(QLIN_ERR_HIP, "%s: HIP error %d (%s)", fn, (int)e, hipGetErrorString(e));
}

#define QA_TRY(expr)                \
  do {                              \
    const int rc_ = (expr);         \
    if (rc_ != QLIN_OK) return rc_; \
  } while (0)

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// A tensor's bytes: runs of `width` at every sum of indexes times strides (bytes; an axis of one has 0).
struct Region {
  const char* name;
  const char* p;
  long long width;
  long long n[3], s[3];
  long long end() const {
    long long e = width;
    for (int i = 0; i < 3; ++i) e += (n[i] - 1) * s[i];
    return e;
  }
};

Region region(const char* name, const void* p, int es, int run, long long n0, long long s0, long long n1, long long s1,
              long long n2 = 1, long long s2 = 0) {
  return Region{name, (const char*)p, (long long)es * run, {n0, n1, n2},
                {n0 > 1 ? s0 * es : 0, n1 > 1 ? s1 * es : 0, n2 > 1 ? s2 * es : 0}};
}

// Sums c + sum k_i s_i with lo_i <= k_i <= hi_i: whether one lies between -before and after (both
// excluded).  Axes come from the longest stride to the shortest; of each only the few multiples are tried
// that the shorter ones can still bring there.  Layouts that take more than `budget` tries (strides of
// about the same length, over long axes) are taken to overlap.
struct Sums {
  struct Axis { long long s, lo, hi; } ax[6];
  int axes = 0;
  long long before, after;
  int budget = 4096;

  void add(long long s, long long lo, long long hi) {
    if (s == 0 || (lo == 0 && hi == 0)) return;
    for (int i = 0; i < axes; ++i)
      if (ax[i].s == s) {
        ax[i].lo += lo, ax[i].hi += hi;
        return;
      }
    int at = axes++;
    for (; at > 0 && ax[at - 1].s < s; --at) ax[at] = ax[at - 1];
    ax[at] = Axis{s, lo, hi};
  }
  static long long floor_div(long long a, long long b) { return a / b - (a % b < 0); }
  bool meet(long long c, int i = 0, bool zero = false) {  // zero: all k 0 so far, which does not count
    if (i == axes) return !zero && c > -before && c < after;
    if (--budget < 0) return true;
    long long least = 0, most = 0;
    for (int j = i + 1; j < axes; ++j) least += ax[j].lo * ax[j].s, most += ax[j].hi * ax[j].s;
    const long long k0 = std::max(ax[i].lo, -floor_div(c + most + before - 1, ax[i].s));
    const long long k1 = std::min(ax[i].hi, floor_div(after - 1 - c - least, ax[i].s));
    for (long long k = k0; k <= k1; ++k)
      if (meet(c + k * ax[i].s, i + 1, zero && k == 0)) return true;
    return false;
  }
};

int check_regions(const char* fn, const Region& a, const Region& b) {
  if (!a.p || !b.p || a.p + a.end() <= b.p || b.p + b.end() <= a.p) return QLIN_OK;
  Sums d;
  d.before = a.width, d.after = b.width;
  for (int i = 0; i < 3; ++i) {
    d.add(a.s[i], 0, a.n[i] - 1);
    d.add(b.s[i], -(b.n[i] - 1), 0);
  }
  if (d.meet(a.p - b.p)) return fail(QLIN_ERR_INVALID, "%s: %s overlaps %s", fn, a.name, b.name);
  return QLIN_OK;
}

// Whether runs of one region share bytes.
int check_region(const char* fn, const Region& a) {
  Sums d;
  d.before = d.after = a.width;
  for (int i = 0; i < 3; ++i)
    if (a.n[i] > 1) {
      if (a.s[i] < a.width) return fail(QLIN_ERR_INVALID, "%s: rows of %s overlap", fn, a.name);
      for (int j = 0; j < i; ++j)  // (two axes of one stride: index (0, 1) is (1, 0))
        if (a.n[j] > 1 && a.s[j] == a.s[i]) return fail(QLIN_ERR_INVALID, "%s: rows of %s overlap", fn, a.name);
      d.add(a.s[i], 1 - a.n[i], a.n[i] - 1);
    }
  if (d.meet(0, 0, true)) return fail(QLIN_ERR_INVALID, "%s: rows of %s overlap", fn, a.name);
  return QLIN_OK;
}

// The partial sums' place in the workspace, behind its counters and exchange slots.
int workspace_parts(const char* fn, void* ws, size_t bytes, char** part, size_t* avail) {
  const size_t base = counter_bytes() + poll_bytes();
  if (!ws || bytes < base) return fail(QLIN_ERR_WORKSPACE, "%s: workspace missing or too small", fn);
  if (!aligned(ws, 256)) return fail(QLIN_ERR_INVALID, "%s: workspace must be 256-byte aligned", fn);
  *part = (char*)ws + base;
  *avail = bytes - base;
  return QLIN_OK;
}

}  // namespace

}  // namespace qlin
