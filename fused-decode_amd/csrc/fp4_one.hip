// Products with E2M1 weights for one activation row (fd_fp4.h has the mathematics): the weights stream past the
// activations through registers.
//
// A wave owns R weight rows (SWIGLU: R / 2 outputs' gate and up rows) over all of K. A chunk is 64 pieces of a row, one a
// lane: 16 bytes of codes, their scale, and the 32 activations that all rows share, which a workgroup has in LDS, quarters
// of the pieces together (a lane's 64 bytes straight from memory are a line a lane and load: 6144 x 4096 7.2 us captured
// where this takes 6.15). bfloat16 codes take their scale in the conversion; float16 ones are converted without it (they would leave
// float16's range) and a piece's sum takes it, exactly. v_dot2 adds two products in float32. Two chunks are on the way.
//
// Bound by a launch's start and end and by the instructions around the weights' stream, half of them outside of the
// products; a wave has two chunks of a K of 4096, and loads two past the end. Traced, median (least), bfloat16: 6144 x 4096
// 6.1 us (4.6; 2.2 TB/s in the median), 28672 x 4096 SWIGLU 15.6 (13.3; 4.0), 4096 x 14336 9.4 (7.8; 3.3).
#include "fd_fp4.h"

namespace fd {

// Eight activations from k on, zeros past K.
template <typename T>
__device__ __forceinline__ typename Vec8<T>::type fp4_load_x(const T* x, int k, int K) {
  typedef typename Vec8<T>::type V8;
  if (k + 8 <= K) {
    typedef V8 any __attribute__((aligned(2)));
    return *reinterpret_cast<const any*>(x + k);
  }
  V8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = k + i < K ? x[k + i] : (T)0.f;
  return v;
}

// The products of a piece: 32 codes, their scale's byte and the activations.
__device__ __forceinline__ float fp4_piece(const u32x4& c, uint32_t byte, const bf16x8 (&x)[4], float acc) {
  const float s = e8m0_operand(byte);
#pragma unroll
  for (int j = 0; j < 4; ++j) acc = dot8(fp4_to_bf16(c[j], s), x[j], acc);
  return acc;
}
__device__ __forceinline__ float fp4_piece(const u32x4& c, uint32_t byte, const f16x8 (&x)[4], float acc) {
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const u32x4 h = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c[j], 1.f, 0)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c[j], 1.f, 1)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c[j], 1.f, 2)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c[j], 1.f, 3))};
    sum = dot8(__builtin_bit_cast(f16x8, h), x[j], sum);
  }
  sum = __builtin_ldexpf(sum, (int)byte - 127);
  return acc + (byte == 255u ? __builtin_nanf("") : sum);
}

constexpr int kOneBlock = 16384;                            // k of the activations that LDS holds at once
constexpr int kOneChunk = kWave * kGroupK;                  // k of a chunk
constexpr int kOneChunks = kOneBlock / kOneChunk;

template <typename T, int R, bool SWIGLU>
__global__ __launch_bounds__(256) void fp4_one_kernel(T* y, const T* x, const uint8_t* w, const uint8_t* ws, int N, int K,
                                                      int64_t swn, int64_t ssn, int64_t syn, Fp4Epi e) {
  typedef typename Vec8<T>::type V8;
  constexpr int O = SWIGLU ? R / 2 : R;  // outputs of a wave
  extern __shared__ __align__(16) u32x4 f4_smem[];
  V8* const xs = reinterpret_cast<V8*>(f4_smem);  // [4][pieces of the block]
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int half = N / 2, cols = SWIGLU ? half : N;
  const int o0 = ((int)blockIdx.x * 4 + wave) * O;
  const int pieces = (K + kGroupK - 1) / kGroupK, chunks = (pieces + kWave - 1) / kWave, left = K % kGroupK;

  const uint8_t *wr[R], *sr[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int n = o0 + (SWIGLU ? i / 2 : i);
    const int64_t row = (n < cols ? n : cols - 1) + (int64_t)(SWIGLU && i % 2 ? half : 0);
    wr[i] = w + row * swn;
    sr[i] = ws + row * ssn;
  }
  struct Chunk {
    u32x4 c[R];
    uint32_t s[R];
  };
  auto load = [&](Chunk& b, int c) {
    const int p = c * kWave + lane, at = p < pieces ? p : 0;  // past the last: the first, times zeros
#pragma unroll
    for (int i = 0; i < R; ++i) b.c[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wr[i] + (unsigned)at * 16u));
#pragma unroll
    for (int i = 0; i < R; ++i) b.s[i] = sr[i][at];
  };
  float acc[R];
#pragma unroll
  for (int i = 0; i < R; ++i) acc[i] = 0.f;
  Chunk b0, b1;
  if (chunks > 0) {  // (a K of 0 has no memory)
    load(b0, 0);
    load(b1, 1);
  }
  // what the epilogue reads, beside the first codes
  const int o = o0 + lane;
  const bool mine = lane < O && o < cols;
  float bias = 0.f, bias2 = 0.f, add = 0.f;
  if (mine) {
    if (e.bias) bias = load_any(e.bias, e.bias_dtype, o * e.sb);
    if (SWIGLU && e.bias) bias2 = load_any(e.bias, e.bias_dtype, (o + (int64_t)half) * e.sb);
    if (e.row) add = load_any(e.row, e.row_dtype, o * e.srn);
  }
  for (int k0 = 0, c0 = 0; c0 < chunks; k0 += kOneBlock, c0 += kOneChunks) {
    const int here = chunks - c0 < kOneChunks ? chunks - c0 : kOneChunks, vectors = here * kOneChunk / 8;
    if (c0) __syncthreads();  // the block before has been read
    for (int v = tid; v < vectors; v += 256) xs[(v & 3) * (here * kWave) + v / 4] = fp4_load_x(x, k0 + v * 8, K);
    __syncthreads();
    auto multiply = [&](Chunk& b, int c) {
      if constexpr (std::is_same<T, bf16>::value) {  // (float16 codes take no scale)
        if (left && c0 + c == chunks - 1 && (c0 + c) * kWave + lane == pieces - 1) {
#pragma unroll
          for (int i = 0; i < R; ++i) b.c[i] = fp4_tail(b.c[i], left);
        }
      }
      V8 xv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) xv[j] = xs[j * (here * kWave) + c * kWave + lane];
      const bool in = (c0 + c) * kWave + lane < pieces;
#pragma unroll
      for (int i = 0; i < R; ++i) acc[i] = fp4_piece(b.c[i], in ? b.s[i] : 127u, xv, acc[i]);
    };
    // the loads run on into the next block's chunks
    for (int c = 0; c < here; c += 2) {
      multiply(b0, c);
      __builtin_amdgcn_sched_barrier(0);
      load(b0, c0 + c + 2);
      __builtin_amdgcn_sched_barrier(0);
      if (c + 1 < here) multiply(b1, c + 1);
      __builtin_amdgcn_sched_barrier(0);
      load(b1, c0 + c + 3);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) acc[i] = wave_sum(acc[i]);
  float v = 0.f, up = 0.f;
#pragma unroll
  for (int i = 0; i < O; ++i) {
    if (lane == i) {
      v = acc[SWIGLU ? 2 * i : i];
      if constexpr (SWIGLU) up = acc[2 * i + 1];
    }
  }
  if (!mine) return;
  v += bias;
  if constexpr (SWIGLU) {
    v = times_sigmoid(v, v) * (up + bias2);
  } else {
    float one[1] = {v};
    activate(one, e.act);
    v = one[0];
  }
  y[(int64_t)o * syn] = from_f32<T>(e.row ? v + add : v);
}

namespace {

template <typename T, int R, bool SWIGLU>
int fp4_one_go(const Fp4Args& a) {
  const int64_t cols = SWIGLU ? a.N / 2 : a.N, per = 4 * (SWIGLU ? R / 2 : R);  // outputs of a workgroup
  const int64_t blocks = (cols + per - 1) / per;
  const int64_t chunks = ((int64_t)a.K + kOneChunk - 1) / kOneChunk;
  const size_t lds = (size_t)(chunks < kOneChunks ? chunks : kOneChunks) * kOneChunk * 2;
  if (blocks * 256 > 0xffffffffLL) return set_error(FD_EUNSUPPORTED, "too many outputs");
  hipLaunchKernelGGL((fp4_one_kernel<T, R, SWIGLU>), dim3((unsigned)blocks), dim3(256), lds, a.st, static_cast<T*>(a.y),
                     static_cast<const T*>(a.x), a.w, a.ws, a.N, a.K, a.swn, a.ssn, a.syn, a.e);
  return FD_OK;
}

// Rows of a wave: two and four take the same time where there are many (28672 x 4096 SWIGLU 18.4, 18.5 us captured), two
// less where there are few (6144 x 4096 6.15, 6.65; 4096 x 14336 10.8, 11.3).
constexpr int kOneRows = 2;

template <typename T>
int fp4_one_pick(const Fp4Args& a) {
  return a.swiglu ? fp4_one_go<T, kOneRows, true>(a) : fp4_one_go<T, kOneRows, false>(a);
}

}  // namespace

int fp4_one_launch(const Fp4Args& a) { return a.act_dtype == FD_F16 ? fp4_one_pick<f16>(a) : fp4_one_pick<bf16>(a); }

}  // namespace fd
