// The two norms around a block: after its output, and before the next one, with the block's residual between them.
//
//   z = x * post_w * rsqrt(mean(x^2) + eps)
//   t = residual + residual_scale * gate * z          (float32); residual_out = round(t)
//   y = round(t * w * rsqrt(mean(t^2) + eps))
//
// t is float32 from its first product to y, and rounded once for residual_out. The gate is one a channel, one a row or
// one an element: a row layout of its own, with strides of 0 where it is broadcast.
//
// One pass over memory: a row stays in registers from its loads to the stores, packed as x and the residual until t
// takes their place. Two sums over a row, each with one exchange between lanes and, where a row is a workgroup's, one
// between waves.
//
// A sum of squares leaves float32's range before its root does: rows of bfloat16 values above about 1e19, and below
// 1e-14 where eps is as small as their squares. Its values then take a power of two (off_range) that cancels.
//
// Many rows are bound by HBM (8192 x 4096 bfloat16, a gate a channel: 49 us, 5.5 TB/s, half of it writes), few by a launch's
// start and end (1 x 4096: 2.8 us).
//
// Two kernels:
//   norm_pair_kernel     - unit column strides, rows of any alignment, 8 <= n <= 32768: LPR lanes a row.
//   norm_pair_gen_kernel - any strides and any n: a workgroup a row, three times over the row.
#include <numeric>
#include <type_traits>

#include "fd_device.h"
#include "fd_gemv.h"
#include "fd_host.h"

namespace fd {

enum GateMode { GATE_NONE = 0, GATE_SAME = 1, GATE_F32 = 2, GATE_ROW = 3 };  // vectors of T, of float32; one a row

// The power of two that a row's values take so that the sum of their squares stays in range, 1 where it is (a sum past
// the top is at least 2^128; one below 2^-90 matters beside eps only where that is below 2^-60).
__device__ __forceinline__ float sum_off_range(float ss, float eps) {
  if (!(ss <= 3.40282347e38f)) return 0x1p-80f;
  return ss < 0x1p-90f && eps < 0x1p-60f ? 0x1p80f : 1.f;
}

template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (L > 32) v = xlane_sum<32>(v);
  if constexpr (L > 16) v = xlane_sum<16>(v);
  v = xlane_sum<8>(v);
  v = xlane_sum<4>(v);
  v = xlane_sum<2>(v);
  return xlane_sum<1>(v);
}

// Sum over a row's LPR lanes, in every lane; `part` holds a value a wave and is written after all have read what it held.
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* part) {
  v = lanes_sum<(LPR > kWave ? kWave : LPR)>(v);
  if constexpr (LPR > kWave) {
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < LPR / kWave; ++i) v += part[i];
  }
  return v;
}

struct PairArgs {
  void *y, *ro;
  const void *x, *r, *gate, *pw, *w;
  int gate_dtype, pw_dtype, w_dtype;
  int64_t pw_stride, w_stride;
  fd_rows lx, lr, lg, ly, lro;
  int64_t rows;
  float scale, eps;
  hipStream_t st;
};

struct PairRows {  // the operands' strides on the row grid
  RowStrides x, r, g, y, ro;
};

template <typename T, typename W, int GATE, int LPR, int VPL>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void norm_pair_kernel(T* y, T* ro, const T* x, const T* r,
                                                                          const void* gate, int gate_dtype,
                                                                          const W* pw, const W* w, RowGrid grid,
                                                                          PairRows l, int n, uint32_t row0,
                                                                          uint32_t rows, float scale, float eps) {
  typedef typename Vec8<T>::type V8;
  typedef typename std::conditional<GATE == GATE_F32, float, T>::type G;
  constexpr int NT = LPR > 256 ? LPR : 256, RPB = NT / LPR, NWAVE = LPR / kWave;
  constexpr bool VEC = GATE == GATE_SAME || GATE == GATE_F32;
  __shared__ float part[NWAVE > 1 ? 4 * NWAVE : 1];
  const int lane = threadIdx.x % LPR;
  const uint32_t row = row0 + blockIdx.x * RPB + threadIdx.x / LPR;
  const bool live = row < rows;
  const int nv = (n + 7) / 8;
  const RowPos p = row_pos(grid, live ? row : 0);
  const T* xr = x + row_off(l.x, p);
  const T* rr = r + row_off(l.r, p);
  const G* gr = VEC ? static_cast<const G*>(gate) + row_off(l.g, p) : nullptr;
  // Where n % 8 != 0 the last vector lies at n - 8; its first elements are the vector before it's too: they are left out
  // of the sums and written twice with one value.
  auto first = [&](int v) { return v * 8 + 8 <= n ? v * 8 : n - 8; };
  V8 a[VPL], b[VPL];
  RawAny<W> pv[VPL];
  RawAny<G> gv[VEC ? VPL : 1];
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int k = first(j * LPR + lane);
    a[j] = load8_any<T>(xr + k);
    b[j] = load8_any<T>(rr + k);
  }
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int k = first(j * LPR + lane);
    pv[j].load(pw + k);
    if constexpr (VEC) gv[j].load(gr + k);
  }
  float f = scale;
  if constexpr (GATE == GATE_ROW) f *= load_any(gate, gate_dtype, row_off(l.g, p));
  auto squares = [&](auto value) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      const int v = j * LPR + lane;
      int skip = v < nv ? v * 8 - first(v) : 8;  // elements that another vector holds, or that lie past the row
      asm volatile("" : "+v"(skip));             // compared where it is used, not kept as 8 VPL masks
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float q = i >= skip ? value(j, i) : 0.f;
        ss += q * q;
      }
    }
    return ss;
  };
  // 1 / rms of a row's values
  auto inverse = [&](auto value, float* at) {
    float ss = row_sum<LPR>(squares(value), at);
    const float pre = sum_off_range(ss, eps);  // the same in all of the row's lanes
    if (pre != 1.f) ss = row_sum<LPR>(squares([&](int j, int i) { return value(j, i) * pre; }), at + NWAVE);
    return rsqrtf(ss / (float)n + eps * pre * pre) * pre;
  };
  f *= inverse([&](int j, int i) { return to_f32(a[j][i]); }, part);
  float t[VPL][8];
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float z = to_f32(a[j][i]) * f * pv[j][i];
      if constexpr (VEC) z *= gv[VEC ? j : 0][i];
      t[j][i] = to_f32(b[j][i]) + z;
    }
  }
  RawAny<W> wv[VPL];
#pragma unroll
  for (int j = 0; j < VPL; ++j) wv[j].load(w + first(j * LPR + lane));
  const float inv = inverse([&](int j, int i) { return t[j][i]; }, part + 2 * NWAVE);
  if (!live) return;
  T* yr = y + row_off(l.y, p);
  T* ror = ro + row_off(l.ro, p);
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int v = j * LPR + lane, k = first(v);
    if (v >= nv) continue;
    V8 o, s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i] = from_f32<T>(t[j][i]);
      o[i] = from_f32<T>(t[j][i] * inv * wv[j][i]);
    }
    store8_any<T>(ror + k, s);
    store8_any<T>(yr + k, o);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void norm_pair_gen_kernel(T* y, T* ro, const T* x, const T* r, const void* gate,
                                                            int gate_dtype, const void* pw, int pw_dtype,
                                                            int64_t pw_stride, const void* w, int w_dtype,
                                                            int64_t w_stride, RowGrid grid, PairRows l, int64_t n,
                                                            uint32_t row0, float scale, float eps) {
  __shared__ float part[4][4];
  const RowPos p = row_pos(grid, row0 + blockIdx.x);
  const T* xr = x + row_off(l.x, p);
  const T* rr = r + row_off(l.r, p);
  const int64_t g0 = row_off(l.g, p);
  auto inverse = [&](auto value, int at) {
    auto squares = [&](float pre) {
      float ss = 0.f;
      for (int64_t k = threadIdx.x; k < n; k += 256) {
        const float q = value(k) * pre;
        ss += q * q;
      }
      return ss;
    };
    float ss = row_sum<256>(squares(1.f), part[at]);
    const float pre = sum_off_range(ss, eps);
    if (pre != 1.f) ss = row_sum<256>(squares(pre), part[at + 1]);
    return rsqrtf(ss / (float)n + eps * pre * pre) * pre;
  };
  const float f = scale * inverse([&](int64_t k) { return to_f32(xr[k * l.x.col]); }, 0);
  auto sum = [&](int64_t k) {
    float z = to_f32(xr[k * l.x.col]) * f * load_any(pw, pw_dtype, k * pw_stride);
    if (gate) z *= load_any(gate, gate_dtype, g0 + k * l.g.col);
    return to_f32(rr[k * l.r.col]) + z;
  };
  const float inv = inverse(sum, 2);
  T* yr = y + row_off(l.y, p);
  T* ror = ro + row_off(l.ro, p);
  for (int64_t k = threadIdx.x; k < n; k += 256) {
    const float t = sum(k);
    ror[k * l.ro.col] = from_f32<T>(t);
    yr[k * l.y.col] = from_f32<T>(t * inv * load_any(w, w_dtype, k * w_stride));
  }
}

namespace {

// launch(first row, workgroups) over all rows, `per` a workgroup of `threads`: a launch has fewer than 2^32 threads.
template <typename F>
void pair_launches(int64_t rows, int per, int threads, F&& launch) {
  const int64_t most = (int64_t)(0xffffffffu / (unsigned)threads) * per;
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t some = rows - r < most ? rows - r : most;
    launch((uint32_t)r, dim3((unsigned)((some + per - 1) / per)));
  }
}

PairRows pair_rows(const PairArgs& a) {
  return PairRows{row_strides(a.lx), row_strides(a.lr), row_strides(a.lg), row_strides(a.ly), row_strides(a.lro)};
}

template <typename T, typename W, int GATE, int LPR, int VPL>
void launch_pair(const PairArgs& a) {
  constexpr int NT = LPR > 256 ? LPR : 256, RPB = NT / LPR;
  pair_launches(a.rows, RPB, NT, [&](uint32_t row0, dim3 blocks) {
    hipLaunchKernelGGL((norm_pair_kernel<T, W, GATE, LPR, VPL>), blocks, dim3(NT), 0, a.st, static_cast<T*>(a.y),
                       static_cast<T*>(a.ro), static_cast<const T*>(a.x), static_cast<const T*>(a.r), a.gate,
                       a.gate_dtype, static_cast<const W*>(a.pw), static_cast<const W*>(a.w), row_grid(a.lx),
                       pair_rows(a), (int)a.lx.n, row0, (uint32_t)a.rows, a.scale, a.eps);
  });
}

constexpr int64_t kPairMaxN = 32768;  // 512 lanes of eight vectors

// Lanes of a row and vectors of eight a lane: 16 lanes up to 128 elements, a wave up to 1024, 256 lanes up to 8192, then 512,
// so that a row stays in registers. Captured, bfloat16, a gate a channel, us of one row and of many (33 million elements),
// beside other lanes:
//
//   elements      rule              other lanes
//   64            16: 3.0   63      64: 3.0   195
//   256           64: 3.0   59      16: 3.8    54
//   512           64: 2.9   44.5    16: 4.1    46
//   1024          64: 3.3   45     256: 3.1    55
//   2048         256: 3.2   48      64: 4.1    47
//   4096         256: 3.6   49      64: 5.7    60     512: 3.5   47
//   8192         256: 4.6   48     512: 4.0    50
//   16384        512: 5.2   55     256: 6.3    64    1024: 5.2   57
//   32768        512: 8.1   56    1024: 8.4    59
template <typename T, typename W, int GATE>
void pick_pair(const PairArgs& a) {
  const int64_t nv = (a.lx.n + 7) / 8;
  if (nv <= 16) return launch_pair<T, W, GATE, 16, 1>(a);
  if (nv <= 64) return launch_pair<T, W, GATE, 64, 1>(a);
  if (nv <= 128) return launch_pair<T, W, GATE, 64, 2>(a);
  if (nv <= 256) return launch_pair<T, W, GATE, 256, 1>(a);
  if (nv <= 512) return launch_pair<T, W, GATE, 256, 2>(a);
  if (nv <= 1024) return launch_pair<T, W, GATE, 256, 4>(a);
  if (nv <= 2048) return launch_pair<T, W, GATE, 512, 4>(a);
  launch_pair<T, W, GATE, 512, 8>(a);
}

template <typename T, typename W>
void pick_gate(const PairArgs& a) {
  constexpr int same = std::is_same<T, f16>::value ? FD_F16 : FD_BF16;
  if (!a.gate) return pick_pair<T, W, GATE_NONE>(a);
  if (a.lg.col == 0) return pick_pair<T, W, GATE_ROW>(a);
  if (a.gate_dtype == same) return pick_pair<T, W, GATE_SAME>(a);
  pick_pair<T, W, GATE_F32>(a);
}

template <typename T>
int dispatch_pair(const PairArgs& a) {
  constexpr int same = std::is_same<T, f16>::value ? FD_F16 : FD_BF16;
  const bool unit = a.lx.n >= 8 && a.lx.n <= kPairMaxN && a.lx.col == 1 && a.lr.col == 1 && a.ly.col == 1 &&
                    a.lro.col == 1 && a.pw_stride == 1 && a.w_stride == 1 && a.pw_dtype == a.w_dtype &&
                    (a.w_dtype == same || a.w_dtype == FD_F32) &&
                    (!a.gate || a.lg.col == 0 || (a.lg.col == 1 && (a.gate_dtype == same || a.gate_dtype == FD_F32)));
  if (unit && a.w_dtype == same)
    pick_gate<T, T>(a);
  else if (unit)
    pick_gate<T, float>(a);
  else
    pair_launches(a.rows, 1, 256, [&](uint32_t row0, dim3 blocks) {
      hipLaunchKernelGGL((norm_pair_gen_kernel<T>), blocks, dim3(256), 0, a.st, static_cast<T*>(a.y),
                         static_cast<T*>(a.ro), static_cast<const T*>(a.x), static_cast<const T*>(a.r), a.gate,
                         a.gate_dtype, a.pw, a.pw_dtype, a.pw_stride, a.w, a.w_dtype, a.w_stride, row_grid(a.lx),
                         pair_rows(a), a.lx.n, row0, a.scale, a.eps);
    });
  return check_launch();
}

int64_t pair_bytes(const fd_rows& l, int elem) {
  return l.a && l.b && l.c && l.n
             ? ((l.a - 1) * l.sa + (l.b - 1) * l.sb + (l.c - 1) * l.sc + (l.n - 1) * l.col + 1) * elem
             : 0;
}

// Whether operands share a byte. Rows of unit column stride begin at multiples of the greatest common divisor of all row
// strides from their bases, so they lie beside each other (halves of a wider buffer's rows) where the bases are a row
// apart within it, both ways round.
bool pair_meet(const void* pa, const fd_rows& la, int ea, const void* pb, const fd_rows& lb, int eb) {
  if (!overlaps(pa, pair_bytes(la, ea), pb, pair_bytes(lb, eb))) return false;
  if (la.n > 1 && (la.col != 1 || lb.col != 1)) return true;
  int64_t step = 0;
  for (const fd_rows* l : {&la, &lb}) {
    const int e = l == &la ? ea : eb;
    if (l->a > 1) step = std::gcd(step, l->sa * e);
    if (l->b > 1) step = std::gcd(step, l->sb * e);
    if (l->c > 1) step = std::gcd(step, l->sc * e);
  }
  if (step == 0) return true;
  const int64_t apart = (int64_t)(reinterpret_cast<uintptr_t>(pb) - reinterpret_cast<uintptr_t>(pa)) % step;
  const int64_t d = apart < 0 ? apart + step : apart;
  return !(d >= la.n * ea && d + lb.n * eb <= step);
}

bool pair_same(const fd_rows& a, const fd_rows& b) {
  return (a.a == 1 || a.sa == b.sa) && (a.b == 1 || a.sb == b.sb) && (a.c == 1 || a.sc == b.sc) &&
         (a.n == 1 || a.col == b.col);
}

}  // namespace
}  // namespace fd

using namespace fd;

extern "C" int fd_norm_add_norm(void* y, void* residual_out, const void* x, const void* residual, const void* gate,
                                int gate_dtype, const void* post_w, int post_w_dtype, int64_t post_w_stride,
                                const void* w, int w_dtype, int64_t w_stride, const fd_rows* lx, const fd_rows* lr,
                                const fd_rows* lg, const fd_rows* ly, const fd_rows* lro, float residual_scale,
                                float eps, int act_dtype, void* stream) {
  if (!check_act_dtype(act_dtype) || !check_any_dtype(post_w_dtype, "post_w_dtype") ||
      !check_any_dtype(w_dtype, "w_dtype") || (gate && !check_any_dtype(gate_dtype, "gate_dtype")))
    return FD_EINVAL;
  if (!y || !residual_out || !x || !residual || !post_w || !w || !lx || !lr || !ly || !lro || (gate && !lg))
    return set_error(FD_EINVAL, "null pointer argument");
  if (!check_rows(*lx, "x") || !check_rows(*lr, "residual") || !check_rows(*ly, "y") ||
      !check_rows(*lro, "residual_out") || (gate && !check_rows(*lg, "gate")) || !same_grid(*lx, *lr, "residual") ||
      !same_grid(*lx, *ly, "y") || !same_grid(*lx, *lro, "residual_out") || (gate && !same_grid(*lx, *lg, "gate")))
    return FD_EINVAL;
  if (post_w_stride < 0 || w_stride < 0) return set_error(FD_EINVAL, "negative stride");
  if (!(eps >= 0.f) || eps == INFINITY) return set_error(FD_EINVAL, "eps must be a finite value >= 0");
  if (!(std::fabs(residual_scale) <= 3.40282347e38f))
    return set_error(FD_EINVAL, "residual_scale must be a finite value");
  const PairArgs a{y, residual_out, x, residual, gate, post_w, w, gate_dtype, post_w_dtype, w_dtype, post_w_stride,
                   w_stride, *lx, *lr, gate ? *lg : *lx, *ly, *lro, lx->a * lx->b * lx->c, residual_scale, eps,
                   static_cast<hipStream_t>(stream)};
  const int64_t n = lx->n;
  if (a.rows == 0 || n == 0) return FD_OK;
  if (a.rows > 0x7fffffffLL) return set_error(FD_EUNSUPPORTED, "too many rows (>= 2^31)");
  // outputs are stored while other rows are still read
  if (rows_meet(*ly) || rows_meet(*lro)) return set_error(FD_EINVAL, "an output's elements must not share memory");
  const int64_t npw = ((n - 1) * post_w_stride + 1) * dtype_bytes(post_w_dtype);
  const int64_t nw = ((n - 1) * w_stride + 1) * dtype_bytes(w_dtype);
  if (pair_meet(y, *ly, 2, residual_out, *lro, 2)) return set_error(FD_EINVAL, "the outputs must not overlap each other");
  const void* out[2] = {y, residual_out};
  const fd_rows* lo[2] = {ly, lro};
  for (int i = 0; i < 2; ++i) {
    const int64_t len = pair_bytes(*lo[i], 2);
    if (overlaps(out[i], len, post_w, npw) || overlaps(out[i], len, w, nw) ||
        (gate && pair_meet(out[i], *lo[i], 2, gate, *lg, dtype_bytes(gate_dtype))))
      return set_error(FD_EINVAL, "an output must not overlap a weight or the gate");
    if ((pair_meet(out[i], *lo[i], 2, x, *lx, 2) && !(out[i] == x && pair_same(*lo[i], *lx))) ||
        (pair_meet(out[i], *lo[i], 2, residual, *lr, 2) && !(out[i] == residual && pair_same(*lo[i], *lr))))
      return set_error(FD_EINVAL, "an output must not overlap an input, other than as x or residual itself");
  }
  return act_dtype == FD_F16 ? dispatch_pair<f16>(a) : dispatch_pair<bf16>(a);
}
