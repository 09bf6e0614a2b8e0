// Products of E4M3 activations and E4M3 weights, shared by the kernels for few and for
// many activation rows:
//
//   v[m,n] = x_scale[m] * w_scale[n] * sum_k x[m,k] * w[n,k] + bias[n]
//   y[m,n] = round(act(v[m,n]) + row_add[m,n])
//   FD_ACT_SWIGLU, w [2I,K]: y[m,j] = round(silu(v[m,j]) * v[m,I+j] + row_add[m,j])
//
// Products of two codes are exact in float32, sums, scales, the activation and row_add are
// float32, and the output is rounded once.
//
// v_mfma_f32_16x16x128_f8f6f4 takes 128 k a step: lane L holds 32 codes of row L % 16 of
// either operand. Any k order that both share gives the same sum; here lane group g = L / 16
// takes bytes 16 g and 64 + 16 g of the step's 128, so that the 16-byte reads of a group
// and of the four groups together run along a row. Weights are the A operand: a lane's four
// sums are weight rows 4 g + r of one activation row L % 16.
#pragma once

#include "fd_device.h"
#include "fd_gemv.h"
#include "fd_host.h"

namespace fd {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kStep = 128;  // k of one MFMA step

// acc += A B over one step; no block scales (both scale operands 0 select the plain form).
__device__ __forceinline__ f32x4 mfma_e4m3(const u32x4& a0, const u32x4& a1, const u32x4& b0, const u32x4& b1,
                                           f32x4 c) {
  const i32x8 a = {(int)a0[0], (int)a0[1], (int)a0[2], (int)a0[3], (int)a1[0], (int)a1[1], (int)a1[2], (int)a1[3]};
  const i32x8 b = {(int)b0[0], (int)b0[1], (int)b0[2], (int)b0[3], (int)b1[0], (int)b1[1], (int)b1[2], (int)b1[3]};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}

// One 16-byte-per-lane DMA from base + off into LDS at byte address `lds` (wave-uniform; lane L
// lands at 16 L). The s_nop is the wait state a load that reads m0 needs after the write of
// m0. (m0 is a reserved register, which the compiler warns of; the clobber still keeps it from
// reusing a value of its own across the asm.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(const uint8_t* base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base)
               : "memory", "m0");
}
// The same from a pointer a lane, nontemporal.
__device__ __forceinline__ void dma16_ptr(const uint8_t* src, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(lds), "v"(src)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// 16 bytes at any address.
__device__ __forceinline__ u32x4 load16_any(const uint8_t* p) {
  typedef u32x4 u32x4_b __attribute__((aligned(1)));
  return *reinterpret_cast<const u32x4_b*>(p);
}
// 16 bytes of a row of K >= 16 at k >= 0; zeros past K. One load wherever k is: the piece that crosses K, and one
// past it, is the row's last 16 bytes moved down.
__device__ __forceinline__ u32x4 load16_end(const uint8_t* row, int k, int K) {
  const int at = k + 16 <= K ? k : K - 16, down = k - at;
  const u32x4 v = load16_any(row + at);
  uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
  const int s = (down & 7) * 8;
  const uint64_t up = s ? hi << (64 - s) : 0;
  const uint64_t lo1 = lo >> s | up, hi1 = hi >> s;
  lo = down < 8 ? lo1 : down < 16 ? hi1 : 0;
  hi = down < 8 ? hi1 : 0;
  return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// This wave's LDS operations are done, then the workgroup's barrier; nothing moves across.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// What a product's epilogue reads beside its sums.
struct W8Epi {
  const float *xs, *ws;
  const void* bias;
  int bias_dtype;
  int64_t sb;
  int act;  // FD_ACT_*, not FD_ACT_SWIGLU, which is a kernel's form
  const void* row;
  int row_dtype;
  int64_t srm, srn;
};

// v sigmoid(u), the sigmoid from one reciprocal: exp(-u) past float32's range leaves 0.
__device__ __forceinline__ float times_sigmoid(float v, float u) {
  return v * __builtin_amdgcn_rcpf(1.f + __expf(-u));
}

// v (1 + erf(v / sqrt 2)) / 2. The lower tail of the normal distribution at -|v| is exp(-v^2 / 2) t P(t) with
// t = 1 / (1 + |v| / sqrt 8) and P a polynomial fitted to exp(z^2) erfc(z) / (2 t), z = |v| / sqrt 2, with a relative
// error below 9e-8 for z <= 13 (past that the exponential is 0). Its evaluation adds up to 2^-18, and the roundings of
// the exponential's argument up to 2^-22 v^2 / 2 (1e-6 at |v| = 3, 1e-5 at 9), relative errors on both sides; no branch
// and few instructions, where erfc's code alone was most of a kernel. The tail's |v| stops short of infinity, so that an
// infinity's is 0.
__device__ __forceinline__ float gelu(float v) {
  const float a = fminf(fabsf(v), 1e18f);
  const float t = __builtin_amdgcn_rcpf(1.f + 0.35355339f * a);
  float p = -0.0296934061f;
  p = p * t + 0.14306283f;
  p = p * t - 0.24520494f;
  p = p * t + 0.140868649f;
  p = p * t - 0.014575636f;
  p = p * t + 0.10187684f;
  p = p * t + 0.121417411f;
  p = p * t + 0.141206071f;
  p = p * t + 0.141042158f;
  const float tail = a * (__expf(-0.5f * a * a) * t * p);
  return v < 0.f ? -tail : v - tail;
}

// Values at once, so that the choice is made once. 0.5 (1 + tanh(u)) is sigmoid(2 u).
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act) {
  if (act == FD_ACT_NONE) return;
  if (act == FD_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = times_sigmoid(v[i], v[i]);
  } else if (act == FD_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];
  } else if (act == FD_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = gelu(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = times_sigmoid(v[i], 1.5957691216057308f * (v[i] + 0.044715f * v[i] * v[i] * v[i]));
  }
}

__device__ __forceinline__ float w8_bias(const W8Epi& e, int64_t n) {
  return e.bias ? load_any(e.bias, e.bias_dtype, n * e.sb) : 0.f;
}

// One output from its sum (SWIGLU: and the up row's, weight row n + half).
template <bool SWIGLU>
__device__ __forceinline__ float w8_out(const W8Epi& e, float acc, float up, int64_t m, int64_t n, int64_t half) {
  const float xs = e.xs[m];
  float v = acc * xs * e.ws[n] + w8_bias(e, n);
  if constexpr (SWIGLU) {
    v = times_sigmoid(v, v) * (up * xs * e.ws[n + half] + w8_bias(e, n + half));
  } else {
    float one[1] = {v};
    activate(one, e.act);
    v = one[0];
  }
  if (e.row) v += load_any(e.row, e.row_dtype, m * e.srm + n * e.srn);
  return v;
}

// A checked product, as the launchers take it: 16-byte aligned rows of whole 16-byte pieces but for K < 16 and M = 1.
struct W8Args {
  void* y;
  const uint8_t *x, *w;
  int M, N, K;  // N: rows of w
  int64_t sxm, swn, sym, syn;
  bool swiglu;
  W8Epi e;
  float* scratch;
  int64_t scratch_bytes;
  int act_dtype;
  hipStream_t st;
};

// One row (w8a8_one.hip): K >= 16, at any alignment.
int w8_one_launch(const W8Args& a);

// Few rows (w8a8_few.hip): whether a product fits, and its launch.
bool w8_few_fits(int64_t M, int64_t K);
void w8_few_form(int64_t M, int64_t K, int* groups, int* steps);  // of 16 activation rows; of a wave, at most
int w8_few_launch(const W8Args& a);

}  // namespace fd
