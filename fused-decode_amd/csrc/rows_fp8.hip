// Rows to OCP E4M3 codes with one float32 scale a row, for the products whose
// activations are 8 bits wide: the row itself, its RMSNorm, or the RMSNorm of its
// sum with a residual.
//
//   t = x                    (quantize_rows, rms_norm_fp8)
//   t = x + r (float32); ro = round(t)                 (add_rms_norm_fp8)
//   y = t                    (quantize_rows), else  y = t * w * rsqrt(mean(t^2) + eps)
//   scale = max(max|y| * (1/448), 2^-126), 1 where max|y| is 0
//   code = e4m3(y / scale), round to nearest even
//
// y is float32 and never rounded to the activation type. A row whose max|y| is not
// finite has a NaN scale and NaN codes: a product with it is NaN, not a row of
// saturated values. max|y| is found on the float32 bits without their sign, whose
// integer order puts an infinity above every number and a NaN above that. The scale is
// never subnormal, so its reciprocal is finite.
//
// A sum of squares leaves float32's range before its root does: rows of bfloat16 values above about 1e19, and
// below 1e-14 where eps is as small as their squares. Such a row is read again, an element at a time, with t times a
// power of two (off_range) that cancels in t * rsqrt(mean(t^2) + eps). That stands behind the stores, which such a
// row leaves out (its inputs may be its outputs), where no register waits for it: a second sweep of the registers cost
// every row some (2048 x 14336 norm 16.7 -> 20.8 us), the same code before the stores too (300 x 20000 7.4 -> 8.6).
//
// One pass over memory: a row stays in registers, packed, from its loads to its codes.
// max|y| = max|t * w| * rsqrt(...), so the sum of squares and the maximum come from one
// sweep and one exchange between lanes.
//
// Many rows are bound by HBM (8192 x 4096, add and norm: 38.7 us, 6.1 TB/s, half of them
// writes; 2048 x 14336 quantised: 16.4 us, 5.4 TB/s), few by a launch's start and end (1 x 4096:
// 2.6 us of device time). Codes are read by the product that follows, not by this kernel: their
// stores are nontemporal.
//
// Two kernels:
//   rows_fp8_kernel     - unit column stride, rows of any alignment, 8 <= n <= 32768: LPR
//                         lanes a row (part of a wave, a wave or a workgroup).
//   rows_fp8_gen_kernel - any strides and any n: a workgroup a row, twice over the row.
#include <atomic>
#include <type_traits>

#include "fd_device.h"
#include "fd_gemv.h"
#include "fd_host.h"

namespace fd {

enum RowsMode { ROWS_PLAIN = 0, ROWS_NORM = 1, ROWS_ADD = 2 };

constexpr float kE4m3Max = 448.f;
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126

// |v| as bits whose unsigned order is that of the magnitudes, NaN on top.
__device__ __forceinline__ uint32_t mag_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

template <int MASK>
__device__ __forceinline__ uint32_t xlane_umax(uint32_t v) {
  if constexpr (MASK >= 16) {
    const auto r = MASK == 32 ? __builtin_amdgcn_permlane32_swap(v, v, false, false)
                              : __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const uint32_t r0 = r[0], r1 = r[1];
    return r0 > r1 ? r0 : r1;
  } else {
    const uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, XlaneDpp<MASK>::ctrl, 0xf, 0xf, false);
    return v > o ? v : o;
  }
}

// Sum and maximum over groups of L lanes (a power of two of at most 64), in every lane.
template <int L, bool SUM>
__device__ __forceinline__ void lanes_reduce(float& ss, uint32_t& mx) {
#define FD_STEP(MASK)                      \
  if constexpr (L > MASK) {                \
    if constexpr (SUM) ss = xlane_sum<MASK>(ss); \
    mx = xlane_umax<MASK>(mx);             \
  }
  FD_STEP(32) FD_STEP(16) FD_STEP(8) FD_STEP(4) FD_STEP(2) FD_STEP(1)
#undef FD_STEP
}

// The power of two that a row's values take so that the sum of their squares stays in range, 1 where it is. A sum
// past the top is at least 2^128, 2^-32 with 2^-80 on the values, where squares that then underflow are too small to
// count. One below 2^-90 matters beside eps only where that is below 2^-60; its values, below 2^-45, take 2^80, and
// the square of the smallest bfloat16 value becomes 2^-106. NaN and infinite values stay what they are.
__device__ __forceinline__ float off_range(float ss, float eps) {
  if (!(ss <= 3.40282347e38f)) return 0x1p-80f;
  return ss < 0x1p-90f && eps < 0x1p-60f ? 0x1p80f : 1.f;
}

// What a row's sums make of its values: code = e4m3(v * inv * r), or NaN.
struct CodeScale {
  float inv, scale, r;
  bool bad;
};
__device__ __forceinline__ CodeScale row_scale(float inv, uint32_t mx) {
  CodeScale q;
  q.inv = inv;
  const float top = __builtin_bit_cast(float, mx) * inv;
  q.bad = mag_bits(top) >= 0x7f800000u;
  q.scale = q.bad ? __builtin_bit_cast(float, 0x7fc00000u)
                  : top > 0.f ? fmaxf(top * (1.f / kE4m3Max), kMinScale) : 1.f;
  q.r = 1.f / q.scale;
  return q;
}

// Four values to four codes. Every |v| is at most 448 (1 + 2^-22), which rounds to 448.
__device__ __forceinline__ uint32_t pack4(const float (&v)[4], bool bad) {
  int p = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  p = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], p, true);
  return bad ? 0x7f7f7f7fu : (uint32_t)p;
}

// y / scale from the reciprocal, rounded as a division rounds it: the quotient's error is
// below one unit, and one step of correction leaves the nearest float (the correction of
// Markstein's division theorem; subnormal remainders only meet quotients far below the
// smallest code; the sign is y's, which the correction of a negative zero loses). Without it
// one code in about 10^6 rounds to its neighbour.
__device__ __forceinline__ float quotient(float y, const CodeScale& q) {
  const float a = y * q.r;
  return __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-a, q.scale, y), q.r, a), y);
}

// A row an element at a time by LPR lanes, of which this is lane l: the sum of squares and the maximum of its values
// times `pre`, in every lane. `sums` and `tops` hold a value a wave where a row is a whole workgroup's.
template <int LPR, bool NORM, typename Value, typename Weight>
__device__ __forceinline__ void element_sums(Value value, Weight weight, int64_t n, float pre, int l, float& ss,
                                             uint32_t& mx, float* sums, uint32_t* tops) {
  ss = 0.f;
  mx = 0;
  for (int64_t k = l; k < n; k += LPR) {
    const float f = value(k) * pre;
    if constexpr (NORM) ss += f * f;
    const uint32_t m = mag_bits(NORM ? f * weight(k) : f);
    mx = m > mx ? m : mx;
  }
  lanes_reduce<(LPR > kWave ? kWave : LPR), NORM>(ss, mx);
  if constexpr (LPR > kWave) {
    __syncthreads();  // what they held has been read
    if (l % kWave == 0) {
      sums[l / kWave] = ss;
      tops[l / kWave] = mx;
    }
    __syncthreads();
    ss = 0.f;
    for (int i = 0; i < LPR / kWave; ++i) {
      ss += sums[i];
      mx = tops[i] > mx ? tops[i] : mx;
    }
  }
}

// The codes of such a row, and its sum with the residual.
template <typename T, int MODE, int LPR, typename Value, typename Weight>
__device__ __forceinline__ void element_codes(uint8_t* codes, T* ro, int64_t ro_col, Value value, Weight weight,
                                              int64_t n, float pre, int l, const CodeScale& q) {
  for (int64_t k = l; k < n; k += LPR) {
    const float f = value(k);
    if constexpr (MODE == ROWS_ADD) ro[k * ro_col] = from_f32<T>(f);
    const float v = MODE != ROWS_PLAIN ? f * pre * weight(k) * q.inv * q.r : quotient(f, q);
    codes[k] = q.bad ? 0x7f : (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false);
  }
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_any __attribute__((aligned(1)));

template <typename T, typename W, int MODE, int LPR, int VPL>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void rows_fp8_kernel(
    uint8_t* codes, float* scale, T* ro, const T* x, const T* r, const W* w, RowGrid grid, RowStrides lx, RowStrides lr,
    RowStrides lro, int n, uint32_t row0, uint32_t rows, float eps) {
  typedef typename Vec8<T>::type V8;
  constexpr int NT = LPR > 256 ? LPR : 256, RPB = NT / LPR, NWAVE = LPR / kWave;
  constexpr bool ADD = MODE == ROWS_ADD, NORM = MODE != ROWS_PLAIN;
  const int l = threadIdx.x % LPR;
  const uint32_t row = row0 + blockIdx.x * RPB + threadIdx.x / LPR;
  const bool live = row < rows;
  const int nv = (n + 7) / 8;
  const RowPos p = row_pos(grid, live ? row : 0);
  const T* xr = x + row_off(lx, p);
  const T* rr = ADD ? r + row_off(lr, p) : nullptr;
  // Where n % 8 != 0 the last vector lies at n - 8; its first elements are the vector
  // before it's too: they are left out of the sum and written twice with one value.
  auto first = [&](int v) { return v * 8 + 8 <= n ? v * 8 : n - 8; };
  V8 a[VPL], b[ADD ? VPL : 1];
  RawAny<W> wv[NORM ? VPL : 1];
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int k = first(j * LPR + l);
    a[j] = load8_any<T>(xr + k);
    if constexpr (ADD) b[j] = load8_any<T>(rr + k);
  }
  if constexpr (NORM) {
#pragma unroll
    for (int j = 0; j < VPL; ++j) wv[j].load(w + first(j * LPR + l));
  }
  auto value = [&](int j, int i) {
    const float f = to_f32(a[j][i]);
    return ADD ? f + to_f32(b[ADD ? j : 0][i]) : f;
  };
  float ss = 0.f;
  uint32_t mx = 0;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int v = j * LPR + l, skip = v < nv ? v * 8 - first(v) : 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = value(j, i);
      if constexpr (NORM) {
        const float q = i >= skip ? f : 0.f;
        ss += q * q;
        const uint32_t m = mag_bits(f * wv[j][i]);
        mx = m > mx ? m : mx;  // vectors past the row hold its last elements again
      } else {
        const uint32_t m = mag_bits(f);
        mx = m > mx ? m : mx;
      }
    }
  }
  lanes_reduce<(LPR > kWave ? kWave : LPR), NORM>(ss, mx);
  __shared__ float sums[NWAVE > 1 ? NWAVE : 1];
  __shared__ uint32_t tops[NWAVE > 1 ? NWAVE : 1];
  if constexpr (NWAVE > 1) {
    if (threadIdx.x % kWave == 0) {
      sums[threadIdx.x / kWave] = ss;
      tops[threadIdx.x / kWave] = mx;
    }
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < NWAVE; ++i) {
      ss += sums[i];
      mx = tops[i] > mx ? tops[i] : mx;
    }
  }
  float pre = NORM ? off_range(ss, eps) : 1.f;  // the same in all of the row's lanes
  if constexpr (NORM && LPR >= kWave)
    pre = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, pre)));
  const CodeScale q = row_scale(NORM ? rsqrtf(ss / (float)n + eps) : 1.f, mx);
  if (!live) return;
  if (l == 0) scale[row] = q.scale;
  uint8_t* cr = codes + (int64_t)row * n;
  T* ror = ADD ? ro + row_off(lro, p) : nullptr;
  const int stored = pre == 1.f ? nv : 0;  // vectors; none of a row out of range, whose inputs may be its outputs
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int k = first(j * LPR + l);
    if (j * LPR + l >= stored) continue;
    u32x2 o;
    V8 s;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = value(j, 4 * h + i);
        if constexpr (ADD) s[4 * h + i] = from_f32<T>(f);
        if constexpr (NORM)
          v[i] = f * wv[j][4 * h + i] * q.inv * q.r;
        else
          v[i] = quotient(f, q);
      }
      o[h] = pack4(v, q.bad);
    }
    if constexpr (ADD) store8_any<T>(ror + k, s);
    __builtin_nontemporal_store(o, reinterpret_cast<u32x2_any*>(cr + k));
  }
  if constexpr (NORM) {
    if (pre != 1.f) {  // in all of the row's lanes, so in every lane that meets at a barrier
      uint32_t at = row;
      int lane = l;
      if constexpr (LPR > kWave) at = __builtin_amdgcn_readfirstlane(at);
      asm volatile("" : "+v"(lane));  // made here, not ahead in registers that the sweep needs
      const RowPos p = row_pos(grid, at);
      const T* xr = x + row_off(lx, p);
      const T* rr = ADD ? r + row_off(lr, p) : nullptr;
      auto element = [&](int64_t k) { return ADD ? to_f32(xr[k]) + to_f32(rr[k]) : to_f32(xr[k]); };
      auto weight = [&](int64_t k) { return to_f32(w[k]); };
      element_sums<LPR, NORM>(element, weight, n, pre, lane, ss, mx, sums, tops);
      const CodeScale q = row_scale(rsqrtf(ss / (float)n + eps * pre * pre), mx);
      if (lane == 0) scale[at] = q.scale;
      element_codes<T, MODE, LPR>(codes + (int64_t)at * n, ADD ? ro + row_off(lro, p) : nullptr, 1, element, weight, n,
                                  pre, lane, q);
    }
  }
}

template <typename T, int MODE>
__global__ __launch_bounds__(256) void rows_fp8_gen_kernel(uint8_t* codes, float* scale, T* ro, const T* x, const T* r,
                                                           const void* w, int w_dtype, int64_t w_stride, RowGrid grid,
                                                           RowStrides lx, RowStrides lr, RowStrides lro, int64_t n,
                                                           uint32_t row0, float eps) {
  constexpr bool ADD = MODE == ROWS_ADD, NORM = MODE != ROWS_PLAIN;
  __shared__ float sums[4];
  __shared__ uint32_t tops[4];
  const uint32_t row = row0 + blockIdx.x;
  const RowPos p = row_pos(grid, row);
  const T* xr = x + row_off(lx, p);
  const T* rr = ADD ? r + row_off(lr, p) : nullptr;
  auto value = [&](int64_t k) {
    const float f = to_f32(xr[k * lx.col]);
    return ADD ? f + to_f32(rr[k * lr.col]) : f;
  };
  auto weight = [&](int64_t k) { return load_any(w, w_dtype, k * w_stride); };
  float ss, pre = 1.f;
  uint32_t mx;
  element_sums<256, NORM>(value, weight, n, pre, (int)threadIdx.x, ss, mx, sums, tops);
  if constexpr (NORM) {
    pre = off_range(ss, eps);
    if (pre != 1.f) element_sums<256, NORM>(value, weight, n, pre, (int)threadIdx.x, ss, mx, sums, tops);
  }
  const CodeScale q = row_scale(NORM && n ? rsqrtf(ss / (float)n + eps * pre * pre) : 1.f, mx);
  if (threadIdx.x == 0) scale[row] = q.scale;
  element_codes<T, MODE, 256>(codes + (int64_t)row * n, ADD ? ro + row_off(lro, p) : nullptr, lro.col, value, weight, n,
                              pre, (int)threadIdx.x, q);
}

namespace {

struct RowsArgs {
  void *codes, *ro;
  float* scale;
  const void *x, *r, *w;
  int w_dtype;
  int64_t w_stride;
  fd_rows lx, lr, lro;
  int64_t rows;
  float eps;
  hipStream_t st;
};

// launch(first row, workgroups) over all rows, `per` a workgroup of `threads`: a launch has fewer than 2^32 threads.
template <typename F>
void row_launches(int64_t rows, int per, int threads, F&& launch) {
  const int64_t most = (int64_t)(0xffffffffu / (unsigned)threads) * per;
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t some = rows - r < most ? rows - r : most;
    launch((uint32_t)r, dim3((unsigned)((some + per - 1) / per)));
  }
}

template <typename T, typename W, int MODE, int LPR, int VPL>
void launch_rows(const RowsArgs& a) {
  constexpr int NT = LPR > 256 ? LPR : 256, RPB = NT / LPR;
  row_launches(a.rows, RPB, NT, [&](uint32_t row0, dim3 blocks) {
    hipLaunchKernelGGL((rows_fp8_kernel<T, W, MODE, LPR, VPL>), blocks, dim3(NT), 0, a.st,
                       static_cast<uint8_t*>(a.codes), a.scale, static_cast<T*>(a.ro), static_cast<const T*>(a.x),
                       static_cast<const T*>(a.r), static_cast<const W*>(a.w), row_grid(a.lx), row_strides(a.lx),
                       row_strides(a.lr), row_strides(a.lro), (int)a.lx.n, row0, (uint32_t)a.rows, a.eps);
  });
}

constexpr int64_t kRowsMaxN = 32768;  // 1024 lanes of four vectors

// Lanes of a row: one vector a lane up to 512 elements, two up to 1024, then a workgroup. Many
// rows of up to 2048 that are quantised alone, with no second operand on the way, take a wave
// each. Measured (us, bf16, add and norm / quantise; a workgroup a row, then a wave a row):
//   rows x n       workgroup        wave
//   256 x 1024     2.77 / 2.40      2.73 / 2.32
//   8192 x 1024    13.1 / 8.10      11.1 / 5.31
//   256 x 2048     2.76 / 2.40      3.41 / 2.64
//   8192 x 2048    19.4 / 10.6      21.2 / 9.36
//   256 x 4096     3.44 / 2.92      5.84 / 3.74
//   8192 x 4096    38.2 / 16.7      43.5 / 17.0
template <typename T, typename W, int MODE>
void pick_rows(const RowsArgs& a) {
  const int64_t nv = (a.lx.n + 7) / 8;
  if (nv <= 8) return launch_rows<T, W, MODE, 8, 1>(a);
  if (nv <= 16) return launch_rows<T, W, MODE, 16, 1>(a);
  if (nv <= 32) return launch_rows<T, W, MODE, 32, 1>(a);
  if (nv <= 64) return launch_rows<T, W, MODE, 64, 1>(a);
  if (nv <= 128) return launch_rows<T, W, MODE, 64, 2>(a);
  if constexpr (MODE == ROWS_PLAIN) {
    if (nv <= 256 && a.rows >= (int64_t)device_cus() * 4) return launch_rows<T, W, MODE, 64, 4>(a);
  }
  if (nv <= 256) return launch_rows<T, W, MODE, 256, 1>(a);
  if (nv <= 512) return launch_rows<T, W, MODE, 256, 2>(a);
  if (nv <= 1024) return launch_rows<T, W, MODE, 256, 4>(a);
  if (nv <= 2048) return launch_rows<T, W, MODE, 256, 8>(a);
  launch_rows<T, W, MODE, 1024, 4>(a);
}

template <typename T, int MODE>
int dispatch_rows(const RowsArgs& a) {
  constexpr int same = std::is_same<T, f16>::value ? FD_F16 : FD_BF16;
  const bool unit = a.lx.col == 1 && (MODE != ROWS_ADD || (a.lr.col == 1 && a.lro.col == 1)) &&
                    (MODE == ROWS_PLAIN || a.w_stride == 1);
  if (unit && a.lx.n >= 8 && a.lx.n <= kRowsMaxN && (MODE == ROWS_PLAIN || a.w_dtype == same))
    pick_rows<T, T, MODE>(a);
  else if (MODE != ROWS_PLAIN && unit && a.lx.n >= 8 && a.lx.n <= kRowsMaxN && a.w_dtype == FD_F32)
    pick_rows<T, typename std::conditional<MODE == ROWS_PLAIN, T, float>::type, MODE>(a);
  else
    row_launches(a.rows, 1, 256, [&](uint32_t row0, dim3 blocks) {
      hipLaunchKernelGGL((rows_fp8_gen_kernel<T, MODE>), blocks, dim3(256), 0, a.st, static_cast<uint8_t*>(a.codes),
                         a.scale, static_cast<T*>(a.ro), static_cast<const T*>(a.x), static_cast<const T*>(a.r), a.w,
                         a.w_dtype, a.w_stride, row_grid(a.lx), row_strides(a.lx), row_strides(a.lr),
                         row_strides(a.lro), a.lx.n, row0, a.eps);
    });
  return check_launch();
}

int64_t layout_bytes(const fd_rows& l) {
  return l.a && l.b && l.c && l.n
             ? ((l.a - 1) * l.sa + (l.b - 1) * l.sb + (l.c - 1) * l.sc + (l.n - 1) * l.col + 1) * 2
             : 0;
}

bool same_layout(const fd_rows& a, const fd_rows& b) {
  return (a.a == 1 || a.sa == b.sa) && (a.b == 1 || a.sb == b.sb) && (a.c == 1 || a.sc == b.sc) &&
         (a.n == 1 || a.col == b.col);
}

int rows_common(int mode, const RowsArgs& a, int act_dtype) {
  const bool add = mode == ROWS_ADD, norm = mode != ROWS_PLAIN;
  const int64_t n = a.lx.n;
  if (a.rows == 0) return FD_OK;
  if (a.rows > 0x7fffffffLL) return set_error(FD_EUNSUPPORTED, "too many rows (>= 2^31)");
  // outputs are stored while other rows are still read
  if (add && rows_meet(a.lro)) return set_error(FD_EINVAL, "residual_out's elements must not share memory");
  const int64_t nc = a.rows * n, ns = a.rows * 4, nx = layout_bytes(a.lx), nr = add ? layout_bytes(a.lr) : 0,
                nro = add ? layout_bytes(a.lro) : 0;
  const int64_t nw = norm && n ? ((n - 1) * a.w_stride + 1) * dtype_bytes(a.w_dtype) : 0;
  const void* in[3] = {a.x, a.r, a.w};
  const int64_t len[3] = {nx, nr, nw};
  for (int i = 0; i < 3; ++i)
    if (overlaps(a.codes, nc, in[i], len[i]) || overlaps(a.scale, ns, in[i], len[i]))
      return set_error(FD_EINVAL, "codes and scale must not overlap an input");
  if (overlaps(a.codes, nc, a.scale, ns) || overlaps(a.ro, nro, a.codes, nc) || overlaps(a.ro, nro, a.scale, ns))
    return set_error(FD_EINVAL, "the outputs must not overlap each other");
  if (add && (overlaps(a.ro, nro, a.w, nw) ||
              (overlaps(a.ro, nro, a.x, nx) && !(a.ro == a.x && same_layout(a.lro, a.lx))) ||
              (overlaps(a.ro, nro, a.r, nr) && !(a.ro == a.r && same_layout(a.lro, a.lr)))))
    return set_error(FD_EINVAL, "residual_out must not overlap an input, other than as x or residual itself");
  if (act_dtype == FD_F16)
    return mode == ROWS_PLAIN  ? dispatch_rows<f16, ROWS_PLAIN>(a)
           : mode == ROWS_NORM ? dispatch_rows<f16, ROWS_NORM>(a)
                               : dispatch_rows<f16, ROWS_ADD>(a);
  return mode == ROWS_PLAIN  ? dispatch_rows<bf16, ROWS_PLAIN>(a)
         : mode == ROWS_NORM ? dispatch_rows<bf16, ROWS_NORM>(a)
                             : dispatch_rows<bf16, ROWS_ADD>(a);
}

}  // namespace
}  // namespace fd

using namespace fd;

extern "C" int fd_quantize_rows_fp8(void* codes, float* scale, const void* x, const fd_rows* lx, int act_dtype,
                                    void* stream) {
  if (!check_act_dtype(act_dtype)) return FD_EINVAL;
  if (!codes || !scale || !x || !lx) return set_error(FD_EINVAL, "null pointer argument");
  if (!check_rows(*lx, "x")) return FD_EINVAL;
  const RowsArgs a{codes, nullptr, scale, x, nullptr, nullptr, act_dtype, 1, *lx, *lx, *lx, lx->a * lx->b * lx->c, 0.f,
                   static_cast<hipStream_t>(stream)};
  return rows_common(ROWS_PLAIN, a, act_dtype);
}

extern "C" int fd_rms_norm_fp8(void* codes, float* scale, const void* x, const void* w, int w_dtype, int64_t w_stride,
                               const fd_rows* lx, float eps, int act_dtype, void* stream) {
  if (!check_act_dtype(act_dtype) || !check_any_dtype(w_dtype, "w_dtype")) return FD_EINVAL;
  if (!codes || !scale || !x || !w || !lx) return set_error(FD_EINVAL, "null pointer argument");
  if (!check_rows(*lx, "x")) return FD_EINVAL;
  if (w_stride < 0) return set_error(FD_EINVAL, "negative stride");
  if (!(eps >= 0.f) || eps == INFINITY) return set_error(FD_EINVAL, "eps must be a finite value >= 0");
  const RowsArgs a{codes, nullptr, scale, x, nullptr, w, w_dtype, w_stride, *lx, *lx, *lx, lx->a * lx->b * lx->c, eps,
                   static_cast<hipStream_t>(stream)};
  return rows_common(ROWS_NORM, a, act_dtype);
}

extern "C" int fd_add_rms_norm_fp8(void* codes, float* scale, void* residual_out, const void* x, const void* residual,
                                   const void* w, int w_dtype, int64_t w_stride, const fd_rows* lx, const fd_rows* lr,
                                   const fd_rows* lro, float eps, int act_dtype, void* stream) {
  if (!check_act_dtype(act_dtype) || !check_any_dtype(w_dtype, "w_dtype")) return FD_EINVAL;
  if (!codes || !scale || !residual_out || !x || !residual || !w || !lx || !lr || !lro)
    return set_error(FD_EINVAL, "null pointer argument");
  if (!check_rows(*lx, "x") || !check_rows(*lr, "residual") || !check_rows(*lro, "residual_out") ||
      !same_grid(*lx, *lr, "residual") || !same_grid(*lx, *lro, "residual_out"))
    return FD_EINVAL;
  if (w_stride < 0) return set_error(FD_EINVAL, "negative stride");
  if (!(eps >= 0.f) || eps == INFINITY) return set_error(FD_EINVAL, "eps must be a finite value >= 0");
  const RowsArgs a{codes, residual_out, scale, x, residual, w, w_dtype, w_stride, *lx, *lr, *lro, lx->a * lx->b * lx->c,
                   eps, static_cast<hipStream_t>(stream)};
  return rows_common(ROWS_ADD, a, act_dtype);
}
