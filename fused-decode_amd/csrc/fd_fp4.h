// Products of 16-bit activations and weights held as OCP E2M1 codes, two a byte (the first in the low half), with an E8M0
// scale (2^(byte - 127), 255: NaN) for each group of 32 along K:
//
//   v[m,n] = sum_k x[m,k] * 2^(s[n, k / 32] - 127) * e2m1(w[n,k]) + bias[n]
//   y[m,n] = round(act(v[m,n]) + row_add[m,n])
//   FD_ACT_SWIGLU, w [2I,K]: y[m,j] = round(silu(v[m,j]) * v[m,I+j] + row_add[m,j])
//
// gfx950 turns two codes and a scale into two bfloat16 numbers in one instruction, and the result is exact: two bits of
// significand and bfloat16's exponents (products past them are infinite, as they are in bfloat16). So a weight needs no
// arithmetic of its own: the scale is in the matrix instruction's operand. float16 activations meet them as two bfloat16
// numbers whose sum they are exactly (11 bits of significand are 8 and 3), float32 sums of both.
//
// A row of codes is read in pieces of 16 bytes: 32 codes, one group, one scale. v_mfma_f32_16x16x32_bf16 takes 32 k a
// step, 8 of row L % 16 from each lane group g = L / 16; any k order that both operands share gives the same sum. Here a
// lane has a whole piece of its row and takes it in four steps, step j its codes 8 j .. 8 j + 7, so that the four groups'
// pieces (128 k) are four steps, and a lane's scale is one for all of them. Weights are the A operand: a lane's four sums
// are weight rows 4 g + i of activation row L % 16.
#pragma once

#include "fd_w8a8.h"

namespace fd {

constexpr int kGroupK = 32;  // k of a scale, codes of a 16-byte piece

// Two codes of byte B of `codes` with the scale whose exponent `scale` has.
template <int B>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B));
}
// Eight codes.
__device__ __forceinline__ bf16x8 fp4_to_bf16(uint32_t codes, float scale) {
  return __builtin_bit_cast(bf16x8, u32x4{fp4_pair<0>(codes, scale), fp4_pair<1>(codes, scale),
                                          fp4_pair<2>(codes, scale), fp4_pair<3>(codes, scale)});
}
// The conversion's scale of an E8M0 byte: it reads the exponent alone, 0 as 2^-127 and 255 as NaN.
__device__ __forceinline__ float e8m0_operand(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// Word J of a row's last piece without the codes past K, `left` = K % 32 of them before it: the activations are zero there,
// but 0 times what a large scale makes of a code is NaN.
template <int J>
__device__ __forceinline__ uint32_t fp4_tail_word(uint32_t codes, int left) {
  const int n = left - 8 * J;
  return n >= 8 ? codes : n <= 0 ? 0u : codes & ((1u << (4 * n)) - 1u);
}
__device__ __forceinline__ u32x4 fp4_tail(const u32x4& c, int left) {
  return u32x4{fp4_tail_word<0>(c[0], left), fp4_tail_word<1>(c[1], left), fp4_tail_word<2>(c[2], left),
               fp4_tail_word<3>(c[3], left)};
}

// float16 as two bfloat16 numbers: its first eight bits, and the three behind them, which are exact; 0 beside an infinity
// or a NaN.
__device__ __forceinline__ void split_f16(f16x8 v, bf16x8& hi, bf16x8& lo) {
  u32x4 a, b;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = (float)v[2 * i], y = (float)v[2 * i + 1];
    const uint32_t xb = __builtin_bit_cast(uint32_t, x), yb = __builtin_bit_cast(uint32_t, y);
    const float xl = x - __builtin_bit_cast(float, xb & 0xffff0000u), yl = y - __builtin_bit_cast(float, yb & 0xffff0000u);
    a[i] = __builtin_amdgcn_perm(yb, xb, 0x07060302);
    b[i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, yl), __builtin_bit_cast(uint32_t, xl), 0x07060302);
  }
  const u32x4 bits = __builtin_bit_cast(u32x4, v), top = bits & 0x7c007c00u;
  uint32_t odd = 0;  // bit 15 of a half: its exponent is all ones
#pragma unroll
  for (int i = 0; i < 4; ++i) odd |= top[i] + 0x04000400u;
  if (__builtin_amdgcn_ballot_w64(odd & 0x80008000u)) {  // rare, and the same for the whole wave
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t bad = top[i] + 0x04000400u;
      b[i] &= (bad & 0x8000u ? 0u : 0xffffu) | (bad & 0x80000000u ? 0u : 0xffff0000u);
    }
  }
  hi = __builtin_bit_cast(bf16x8, a);
  lo = __builtin_bit_cast(bf16x8, b);
}

// One 16-byte-per-lane DMA from a pointer a lane into LDS at byte address `lds` (wave-uniform; lane L lands at 16 L).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16_at(const void* src, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}
#pragma clang diagnostic pop

struct Fp4Epi {
  const void* bias;
  int bias_dtype;
  int64_t sb;
  int act;  // FD_ACT_*, not FD_ACT_SWIGLU, which is a kernel's form
  const void* row;
  int row_dtype;
  int64_t srm, srn;
};

// One output from its sum (SWIGLU: and the up row's, weight row n + half).
template <bool SWIGLU>
__device__ __forceinline__ float fp4_out(const Fp4Epi& e, float acc, float up, int64_t m, int64_t n, int64_t half) {
  float v = acc + (e.bias ? load_any(e.bias, e.bias_dtype, n * e.sb) : 0.f);
  if constexpr (SWIGLU) {
    v = times_sigmoid(v, v) * (up + (e.bias ? load_any(e.bias, e.bias_dtype, (n + half) * e.sb) : 0.f));
  } else {
    float one[1] = {v};
    activate(one, e.act);
    v = one[0];
  }
  if (e.row) v += load_any(e.row, e.row_dtype, m * e.srm + n * e.srn);
  return v;
}

// A checked product: rows of codes are 16-byte aligned runs of ceil(K / 32) pieces, x has unit stride along K.
struct Fp4Args {
  void* y;
  const void* x;
  const uint8_t *w, *ws;
  int M, N, K;  // N: rows of w
  int64_t sxm, swn, ssn, sym, syn;
  bool swiglu;
  Fp4Epi e;
  float* scratch;
  int64_t scratch_bytes;
  int act_dtype;
  hipStream_t st;
};

// One row (fp4_one.hip): any K.
int fp4_one_launch(const Fp4Args& a);

// Few rows (fp4_few.hip): whether a product fits, whether it takes less time there than in tiles, and its launch.
bool fp4_few_fits(int64_t M, int64_t K, bool swiglu);
bool fp4_few_wins(int64_t M, int64_t K, int act_dtype);
int fp4_few_launch(const Fp4Args& a);

}  // namespace fd
