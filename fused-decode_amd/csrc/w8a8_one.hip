// Products of E4M3 activations and weights for one activation row (fd_w8a8.h has the mathematics):
// the weights stream past the activations through registers.
//
// A wave owns two weight rows (SWIGLU: an output's gate and up row) over all of K, with no LDS
// and no barrier. A load takes 1 KiB of a row, 16 codes a lane; the loads of four such chunks of
// both rows and of the activations make a group, and the next group is on the way while this
// one is multiplied. Codes become pairs of float16, which holds every E4M3 value exactly, and
// v_dot2 adds two products in float32. The wave's sums meet by lane exchanges at the end. What
// the epilogue reads beside them is loaded first.
//
// Bound by the weights' stream and by a launch's start and end: 6144 x 4096 6.1 us, 28672 x 4096
// SWIGLU 19.0 (6.2 TB/s), 4096 x 14336 11.7, where the kernel for few rows, whose loads take 128
// bytes of each of 8 rows, takes 7.8, 21.1 and 12.9. Rows a wave x chunks a group, the same shapes:
// 2 x 2 6.3, 20.2, 11.6; 4 x 2 7.5, 20.6, 11.7 (fewer waves, uneven over the CUs); 2 x 8 8.3,
// 29.6, 13.1 (registers for one wave a SIMD). Two activation rows are no faster here than there.
//
// Rows have any alignment. EDGE: K is no multiple of 16, and the piece of a row that crosses K is
// its last 16 bytes moved down.
#include "fd_w8a8.h"

namespace fd {

constexpr int kOneChunk = 16 * kWave;  // codes of a row that a load of a wave takes
constexpr int kOneGroup = 4;           // chunks of a group

__device__ __forceinline__ void codes_to_f16(const u32x4& c, f16x2 (&h)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[2 * i] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.0f, false));
    h[2 * i + 1] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i], 1.0f, true));
  }
}

// An element of one of the three float types, and its value later: nothing waits for it in between.
__device__ __forceinline__ uint32_t load_raw(const void* p, int dtype, int64_t i) {
  return dtype == FD_F32 ? static_cast<const uint32_t*>(p)[i] : static_cast<const uint16_t*>(p)[i];
}
__device__ __forceinline__ float raw_f32(uint32_t v, int dtype) {
  return dtype == FD_F16 ? to_f32(__builtin_bit_cast(f16, (uint16_t)v))
                         : __builtin_bit_cast(float, dtype == FD_F32 ? v : v << 16);
}

template <typename T, bool SWIGLU, bool EDGE>
__global__ __launch_bounds__(256) void w8a8_one_kernel(T* y, const uint8_t* x, const uint8_t* w, int N, int K,
                                                       int64_t swn, int64_t syn, W8Epi e) {
  typedef u32x4 u32x4_any __attribute__((aligned(1)));
  constexpr int G = kOneGroup, R = 2, O = SWIGLU ? 1 : 2;  // chunks, rows, outputs of a wave
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const int half = N / 2, cols = SWIGLU ? half : N;
  const int o0 = ((int)blockIdx.x * 4 + wave) * O;
  if (o0 >= cols) return;

  // the output of this lane, and what it needs
  const int o = o0 + lane;
  const bool mine = lane < O && o < cols;
  float xs = 0.f, ws1 = 0.f, ws2 = 0.f;
  uint32_t bias1 = 0, bias2 = 0, add = 0;
  if (mine) {
    xs = e.xs[0];
    ws1 = e.ws[o];
    if (e.bias) bias1 = load_raw(e.bias, e.bias_dtype, o * e.sb);
    if constexpr (SWIGLU) {
      ws2 = e.ws[o + half];
      if (e.bias) bias2 = load_raw(e.bias, e.bias_dtype, (o + (int64_t)half) * e.sb);
    }
    if (e.row) add = load_raw(e.row, e.row_dtype, o * e.srn);
  }

  const uint8_t* wr[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int n = o0 + (SWIGLU ? i / 2 : i);
    wr[i] = w + ((n < cols ? n : cols - 1) + (int64_t)(SWIGLU && i % 2 ? half : 0)) * swn;
  }
  float acc[R] = {0.f, 0.f};

  struct Group {
    u32x4 w[G][R], x[G];
  };
  const int chunks = (K + kOneChunk - 1) / kOneChunk;
  auto load = [&](Group& b, int c) {  // chunks c .. c + G - 1
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const int k = (c + j) * kOneChunk + lane * 16;
      if constexpr (EDGE) {
        b.x[j] = load16_end(x, k, K);
#pragma unroll
        for (int i = 0; i < R; ++i) b.w[j][i] = load16_end(wr[i], k, K);
      } else {
        const unsigned at = k < K ? (unsigned)k : 0u;
        b.x[j] = *reinterpret_cast<const u32x4_any*>(x + at);
#pragma unroll
        for (int i = 0; i < R; ++i)
          b.w[j][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(wr[i] + at));
      }
    }
  };
  auto multiply = [&](const Group& b, int c) {
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const uint32_t keep = EDGE || (c + j) * kOneChunk + lane * 16 < K ? ~0u : 0u;  // zeros past K
      f16x2 xh[8];
      codes_to_f16(b.x[j] & keep, xh);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        f16x2 wh[8];
        codes_to_f16(b.w[j][i], wh);
#pragma unroll
        for (int p = 0; p < 8; ++p) acc[i] = __builtin_amdgcn_fdot2(wh[p], xh[p], acc[i], false);
      }
    }
  };
  Group b0, b1;
  if (chunks <= G) {
    load(b0, 0);
    multiply(b0, 0);
  } else {
    load(b0, 0);
    for (int c = 0; c < chunks; c += 2 * G) {
      load(b1, c + G);
      __builtin_amdgcn_sched_barrier(0);
      multiply(b0, c);
      __builtin_amdgcn_sched_barrier(0);
      load(b0, c + 2 * G);
      __builtin_amdgcn_sched_barrier(0);
      multiply(b1, c + G);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  const float s0 = wave_sum(acc[0]), s1 = wave_sum(acc[1]);
  if (!mine) return;
  float v = (SWIGLU || lane == 0 ? s0 : s1) * xs * ws1 + raw_f32(bias1, e.bias_dtype);
  if constexpr (SWIGLU) {
    v = times_sigmoid(v, v) * (s1 * xs * ws2 + raw_f32(bias2, e.bias_dtype));
  } else {
    float one[1] = {v};
    activate(one, e.act);
    v = one[0];
  }
  y[o * syn] = from_f32<T>(e.row ? v + raw_f32(add, e.row_dtype) : v);
}

namespace {

template <typename T, bool SWIGLU>
int one_go(const W8Args& a) {
  const int64_t cols = SWIGLU ? a.N / 2 : a.N, per = 4 * (SWIGLU ? 1 : 2);  // outputs of a workgroup
  const int64_t blocks = (cols + per - 1) / per;
  if (blocks * 256 > 0xffffffffLL) return set_error(FD_EUNSUPPORTED, "too many outputs");
  auto kernel = a.K % 16 ? w8a8_one_kernel<T, SWIGLU, true> : w8a8_one_kernel<T, SWIGLU, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, a.st, static_cast<T*>(a.y), a.x, a.w, a.N, a.K,
                     a.swn, a.syn, a.e);
  return FD_OK;
}

}  // namespace

int w8_one_launch(const W8Args& a) {
  if (a.act_dtype == FD_F16) return a.swiglu ? one_go<f16, true>(a) : one_go<f16, false>(a);
  return a.swiglu ? one_go<bf16, true>(a) : one_go<bf16, false>(a);
}

}  // namespace fd
