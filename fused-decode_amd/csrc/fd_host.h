// Host-side argument checking and error reporting shared by the C ABI entry
// points. Every check runs before any HIP call, so a rejected call launches
// nothing and can be tested without a GPU.
#pragma once

#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <cmath>

#include "fused_decode.h"

namespace fd {

inline thread_local char g_last_error[512] = "";

inline int set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return code;
}

inline bool check_act_dtype(int dt) {
  if (dt == FD_F16 || dt == FD_BF16) return true;
  set_error(FD_EINVAL, "act_dtype must be FD_F16 or FD_BF16, got %d", dt);
  return false;
}

inline bool check_any_dtype(int dt, const char* what) {
  if (dt == FD_F16 || dt == FD_BF16 || dt == FD_F32) return true;
  set_error(FD_EINVAL, "%s must be FD_F16, FD_BF16 or FD_F32, got %d", what, dt);
  return false;
}

inline bool check_rows(const fd_rows& l, const char* what) {
  if (l.a < 0 || l.b < 0 || l.c < 0 || l.n < 0) {
    set_error(FD_EINVAL, "%s layout has a negative size", what);
    return false;
  }
  if (l.sa < 0 || l.sb < 0 || l.sc < 0 || l.col < 0) {
    set_error(FD_EINVAL, "%s layout has a negative stride", what);
    return false;
  }
  return true;
}

inline bool same_grid(const fd_rows& x, const fd_rows& o, const char* what) {
  if (x.a != o.a || x.b != o.b || x.c != o.c || x.n != o.n) {
    set_error(FD_EINVAL, "%s cannot be indexed with the same row grid as the input", what);
    return false;
  }
  return true;
}

// Whether two elements of a layout lie at one address: strides that broadcast, windows that run into each other.
// Sorted by stride, dimensions that each step past all that the smaller ones reach hold no such two, which is every
// view that slices and transposes make. For the rest (no more than four, of sizes > 1) it is the question
// whether some steps, not all zero and less than each size, add up to nothing: answered by search, and by yes where
// the search is longer than kMeetSearch.
struct RowDim {
  int64_t size, step;
};
constexpr int kMeetSearch = 1 << 16;

// `at` + steps of dims[0 .. n) = 0, with a step taken somewhere (`moved`: there was one).
inline bool steps_cancel(const RowDim* dims, int n, int64_t at, bool moved, int& budget) {
  if (n == 0) return at == 0 && moved;
  int64_t rest = 0;
  for (int i = 1; i < n; ++i) rest += (dims[i].size - 1) * dims[i].step;
  const int64_t step = dims[0].step, most = dims[0].size - 1;
  for (int64_t k = moved ? -most : 0; k <= most; ++k) {  // the negative of an answer is one: the first step is >= 0
    const int64_t to = at + k * step;
    if (to > rest) break;
    if (to < -rest) {
      const int64_t skip = (-rest - to + step - 1) / step;
      k += skip - 1;
      continue;
    }
    if (--budget < 0 || steps_cancel(dims + 1, n - 1, to, moved || k != 0, budget)) return true;
  }
  return false;
}

inline bool rows_meet(const fd_rows& l) {
  const RowDim all[4] = {{l.a, l.sa}, {l.b, l.sb}, {l.c, l.sc}, {l.n, l.col}};
  RowDim dims[4];  // by falling stride
  int n = 0;
  for (const RowDim& d : all) {
    if (d.size <= 0) return false;
    if (d.size == 1) continue;
    if (d.step == 0) return true;
    int i = n++;
    for (; i > 0 && dims[i - 1].step < d.step; --i) dims[i] = dims[i - 1];
    dims[i] = d;
  }
  int64_t reach = 0;
  bool nested = true;
  for (int i = n - 1; i >= 0; --i) {
    nested = nested && dims[i].step > reach;
    reach += (dims[i].size - 1) * dims[i].step;
  }
  int budget = kMeetSearch;
  return !nested && steps_cancel(dims, n, 0, false, budget);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// True when the byte ranges [a, a + na) and [b, b + nb) share a byte.
inline bool overlaps(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
  return na > 0 && nb > 0 && pa < pb + (uintptr_t)nb && pb < pa + (uintptr_t)na;
}

// Bytes from the first to past the last of rows x cols elements at r * sr + c * sc
// (strides >= 0).
inline int64_t span_bytes(int64_t rows, int64_t cols, int64_t sr, int64_t sc, int64_t elem_bytes) {
  return rows > 0 && cols > 0 ? ((rows - 1) * sr + (cols - 1) * sc + 1) * elem_bytes : 0;
}

inline int dtype_bytes(int dt) { return dt == FD_F32 ? 4 : 2; }

// True when an epilogue that reads row_add at other elements than the one it then
// writes could meet the output: row_add [M,N] and y share memory, and row_add is not
// y's own elements in y's order.
inline bool row_add_meets(const void* row_add, int row_dtype, int64_t srm, int64_t srn, const void* y, int act_dtype,
                          int64_t sym, int64_t syn, int64_t M, int64_t N) {
  if (!row_add || !overlaps(row_add, span_bytes(M, N, srm, srn, dtype_bytes(row_dtype)), y,
                            span_bytes(M, N, sym, syn, dtype_bytes(act_dtype))))
    return false;
  const bool same = row_add == y && row_dtype == act_dtype && (M == 1 || srm == sym) && (N == 1 || srn == syn);
  return !same;
}

// The MLP entry points write y and mid while hidden is still to be read (the
// down projection adds hidden as its residual, and from M = 5 y first holds the
// normalised rows): none of the three may share memory.
inline int check_mlp_buffers(const void* y, const void* mid, const void* hidden, int64_t M,
                             int64_t H, int64_t I, int elem_bytes) {
  const int64_t nh = M * H * elem_bytes, ni = M * I * elem_bytes;
  if (overlaps(y, nh, hidden, nh)) return set_error(FD_EINVAL, "y must not overlap hidden");
  if (overlaps(mid, ni, hidden, nh) || overlaps(mid, ni, y, nh))
    return set_error(FD_EINVAL, "mid must not overlap y or hidden");
  return FD_OK;
}

// True when every row of `l` is a run of n contiguous elements whose start is
// 16-byte aligned and n is a multiple of 8 (so 16-byte vectors tile the row).
inline bool rows_vectorizable(const void* p, const fd_rows& l, int elem_bytes) {
  const int64_t v = 16 / elem_bytes;
  if (!aligned16(p) || l.n % v != 0) return false;
  if (l.n > 1 && l.col != 1) return false;
  if (l.a > 1 && l.sa % v != 0) return false;
  if (l.b > 1 && l.sb % v != 0) return false;
  if (l.c > 1 && l.sc % v != 0) return false;
  return true;
}

// Row sums of squares handed between launches (a producer GEMV's per-tile sums
// of its squared outputs, read by the next RMSNorm): the checks of a *_sumsq
// entry point's `ss_in` (ceil(H/16) tiles of the norm input's width H) and
// `ss_out`. `mfma`: whether this call runs the MFMA kernels that read or write
// them.
inline int check_sumsq(bool mfma, const float* ss_in, int64_t ss_tiles, int64_t H, const float* ss_out) {
  if (!mfma)
    return set_error(FD_EUNSUPPORTED, "row sums of squares are for the MFMA kernels (kind=dot, M >= 5)");
  if (ss_in) {
    if (ss_tiles != (H + 15) / 16)
      return set_error(FD_EINVAL, "ss_tiles must be ceil(H / 16) = %lld, got %lld", (long long)((H + 15) / 16),
                       (long long)ss_tiles);
    if (!aligned16(ss_in)) return set_error(FD_EUNSUPPORTED, "ss_in must be 16-byte aligned");
  }
  if (ss_out && !aligned16(ss_out)) return set_error(FD_EUNSUPPORTED, "ss_out must be 16-byte aligned");
  return FD_OK;
}

inline int check_launch() {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(FD_ELAUNCH, "HIP launch failed: %s", hipGetErrorString(e));
  return FD_OK;
}

}  // namespace fd
