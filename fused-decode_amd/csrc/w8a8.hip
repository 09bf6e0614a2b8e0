// Products of E4M3 activations and weights in tiles of the output, for any number of
// activation rows (fd_w8a8.h has the mathematics).
//
// A workgroup of WN x WM waves owns BN weight rows x BM activation rows and walks K in stages
// of 128. Both tiles of a stage go to LDS, D - 1 stages ahead of the one being multiplied, one
// barrier a stage: by DMA (global_load_lds_dwordx4) where rows are 16-byte aligned and K % 16
// == 0, else through registers with 16-byte loads at any address (bytes for the piece that
// crosses K). The DMAs are inline assembly, so the compiler sees plain LDS reads and schedules
// and waits for those itself; the vmcnt waits are explicit.
//
// LDS layout: a tile row is 8 chunks of 16 bytes, chunk c at slot c ^ (row mod 8), so the 8
// lanes of a read (8 rows, one chunk) hit distinct bank groups and a DMA instruction still fills
// 1 KiB in lane order. The weight rows of a wave lie in LDS in the order that gives a lane
// consecutive outputs: lane group g's sums are outputs 4 NT g .. 4 NT g + 4 NT - 1 of the wave
// (SWIGLU: gate and up rows in turn, so that a lane holds both of an output), and leave in
// 16-byte pieces along a row without another pass through LDS.
//
// Where the output has fewer tiles than the GPU has CUs, K is split over workgroups whose
// float32 sums go through scratch and are added in split order by a second launch.
#include <type_traits>

#include "fd_w8a8.h"

namespace fd {

template <int BN, int BM> constexpr int kStageBytes = (BN + BM) * kStep;

enum W8Form { W8_OUT = 0, W8_PART = 1 };

// 16 bytes of a row of K at k, any alignment; zeros past K.
__device__ __forceinline__ u32x4 load16_any(const uint8_t* row, int k, int K) {
  typedef u32x4 u32x4_b __attribute__((aligned(1)));
  if (k + 16 <= K) return *reinterpret_cast<const u32x4_b*>(row + k);
  u32x4 v = {0u, 0u, 0u, 0u};
  for (int i = 0; i < 16; ++i)
    if (k + i < K) v[i / 4] |= (uint32_t)row[k + i] << (i % 4 * 8);
  return v;
}

template <typename T, int WN, int WM, int NT, int MT, int D, bool SWIGLU, int FORM, bool DMA>
__global__ __launch_bounds__(WN * WM * kWave) void w8a8_tile_kernel(T* y, float* part, const uint8_t* x,
                                                                    const uint8_t* w, int M, int N, int K, int64_t sxm,
                                                                    int64_t swn, int64_t sym, int64_t syn, W8Epi e,
                                                                    int mtiles, int splits) {
  typedef typename Vec8<T>::type V8;
  constexpr int NW = WN * WM, BN = WN * NT * 16, BM = WM * MT * 16;
  constexpr int AOPS = BN / 8 / NW, BOPS = BM / 8 / NW, OPS = AOPS + BOPS;
  static_assert(AOPS * 8 * NW == BN && BOPS * 8 * NW == BM, "the waves share a stage evenly");
  static_assert(!SWIGLU || NT % 2 == 0, "gate and up tiles in turn");
  extern __shared__ __align__(16) u32x4 w8_smem[];
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int wm = wave % WM, wn = wave / WM;
  const int r = lane & 15, g = lane >> 4;

  // Block -> (tile, K split). Consecutive blocks go to the eight XCDs in turn: each XCD takes
  // a contiguous run of tiles, the row blocks of one weight tile next to each other.
  int tile, split = 0;
  {
    int b = (int)blockIdx.x;
    const int total = (int)gridDim.x;
    if (splits > 1) {
      split = b % splits;
      tile = b / splits;
    } else {
      const int xcd = b & 7, q = total >> 3, rem = total & 7;
      tile = xcd * q + (xcd < rem ? xcd : rem) + (b >> 3);
    }
  }
  const int ntile = tile / mtiles, m0 = (tile - ntile * mtiles) * BM;
  const int half = N / 2, cols = SWIGLU ? half : N;
  constexpr int OUT = SWIGLU ? BN / 2 : BN, LANE = SWIGLU ? NT * 2 : NT * 4;  // outputs of a tile, of a lane
  const int stages_all = (K + kStep - 1) / kStep;
  const int s0 = (int)((int64_t)stages_all * split / splits);
  const int ns = (int)((int64_t)stages_all * (split + 1) / splits) - s0;

  // weight row at LDS row t of the tile (past the last: one that exists, never stored)
  auto wrow = [&](int t) -> int64_t {
    const int wv = t / (NT * 16), f = t / 16 % NT, i = t & 15;
    if constexpr (SWIGLU) {
      const int n = ntile * OUT + wv * (NT * 8) + (i >> 2) * LANE + (f >> 1) * 4 + (i & 3);
      return (n < half ? n : half - 1) + (int64_t)((f & 1) ? half : 0);
    } else {
      const int n = ntile * OUT + wv * (NT * 16) + (i >> 2) * LANE + f * 4 + (i & 3);
      return n < N ? n : N - 1;
    }
  };

  const unsigned lds0 = lds_addr(w8_smem);
  constexpr unsigned kStage = (unsigned)kStageBytes<BN, BM>;
  const uint8_t* src[OPS];
  int off[OPS];
#pragma unroll
  for (int i = 0; i < OPS; ++i) {
    const bool wt = i < AOPS;
    const int t = (wt ? wave * AOPS + i : wave * BOPS + i - AOPS) * 8 + lane / 8;
    const int m = m0 + t;
    src[i] = wt ? w + wrow(t) * swn : x + (int64_t)(m < M ? m : M - 1) * sxm;
    off[i] = ((lane & 7) ^ (t & 7)) * 16;
  }
  auto place = [&](int i) {  // byte address in a stage of this wave's i-th KiB
    return (unsigned)(i < AOPS ? wave * AOPS + i : BN / 8 + wave * BOPS + i - AOPS) * 1024u;
  };
  auto issue = [&](int s) {
    const unsigned base = lds0 + (unsigned)(s % D) * kStage;
#pragma unroll
    for (int i = 0; i < OPS; ++i) {
      const int k = (s0 + s) * kStep + off[i];
      dma16<false>(src[i] + (k < K ? k : 0), base + place(i));
    }
  };
  u32x4 held[DMA ? 1 : OPS];
  auto fetch = [&](int s) {
#pragma unroll
    for (int i = 0; i < OPS; ++i) held[DMA ? 0 : i] = load16_any(src[i], (s0 + s) * kStep + off[i], K);
  };
  auto put = [&](int s) {
#pragma unroll
    for (int i = 0; i < OPS; ++i) w8_smem[((s % D) * kStage + place(i)) / 16 + lane] = held[DMA ? 0 : i];
  };

  f32x4 acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};

  // this lane's two chunks of a tile row (u32x4 entries): row r of a 16-row tile, r mod 8 is
  // every tile's swizzle
  const int c0 = g ^ (r & 7), c1 = (4 + g) ^ (r & 7);
  auto multiply = [&](int s) {
    const u32x4* st = w8_smem + (size_t)(s % D) * (kStage / 16);
    u32x4 b0[MT], b1[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const u32x4* p = st + BN * 8 + ((wm * MT + m) * 16 + r) * 8;
      b0[m] = p[c0];
      b1[m] = p[c1];
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const u32x4* p = st + ((wn * NT + n) * 16 + r) * 8;
      const u32x4 a0 = p[c0], a1 = p[c1];
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[n][m] = mfma_e4m3(a0, a1, b0[m], b1[m], acc[n][m]);
    }
  };

  if constexpr (DMA) {
    const int pre = ns < D - 1 ? ns : D - 1;
    for (int s = 0; s < pre; ++s) issue(s);
    for (int s = 0; s < ns; ++s) {
      // stages issued so far end at s + D - 2: D - 2 of them may stay in flight
      if (s + D - 2 < ns)
        wait_vm<OPS*(D - 2)>();
      else
        wait_vm<0>();
      if ((s0 + s + 1) * kStep > K) {  // K tail: activations past K are zero
#pragma unroll
        for (int i = AOPS; i < OPS; ++i)
          if ((s0 + s) * kStep + off[i] >= K)
            ds_zero16(lds0 + (unsigned)(s % D) * kStage + place(i) + (unsigned)lane * 16u);
      }
      lds_barrier();  // stage s has landed everywhere; every wave is done with stage s - 1
      if (s + D - 1 < ns) issue(s + D - 1);
      multiply(s);
    }
  } else {
    if (ns > 0) fetch(0);
    for (int s = 0; s < ns; ++s) {
      put(s);  // D = 2: the other half may still be read
      lds_barrier();
      if (s + 1 < ns) fetch(s + 1);
      multiply(s);
    }
  }

  const int n0 = ntile * OUT + wn * (OUT / WN) + g * LANE;  // this lane's first output column
  if (n0 >= cols) return;
  if constexpr (FORM == W8_PART) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = m0 + (wm * MT + m) * 16 + r;
      if (row >= M) continue;
      float* to = part + ((int64_t)split * M + row) * N;
#pragma unroll
      for (int f = 0; f < NT; ++f) {
        const int n = n0 + (SWIGLU ? f >> 1 : f) * 4, at = n + (SWIGLU && (f & 1) ? half : 0);
        if (n + 4 <= cols && N % 4 == 0 && (!SWIGLU || half % 4 == 0)) {
          *reinterpret_cast<f32x4*>(to + at) = acc[f][m];
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (n + i < cols) to[at + i] = acc[f][m][i];
        }
      }
    }
  } else {
    const bool wide = syn == 1 && sym % 8 == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
    // eight outputs at a time: their scales and bias once for all of this lane's rows
#pragma unroll
    for (int q = 0; q < LANE / 8; ++q) {
      const int n = n0 + q * 8;
      if (n >= cols) break;
      float s1[8], b1[8], s2[SWIGLU ? 8 : 1], b2[SWIGLU ? 8 : 1];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = n + i < cols ? n + i : cols - 1;
        s1[i] = e.ws[c];
        b1[i] = w8_bias(e, c);
        if constexpr (SWIGLU) {
          s2[i] = e.ws[half + c];
          b2[i] = w8_bias(e, (int64_t)half + c);
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const int row = m0 + (wm * MT + m) * 16 + r;
        if (row >= M) continue;
        const float xs = e.xs[row];
        V8 o;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float v;
          if constexpr (SWIGLU) {
            const int f = (q * 2 + i / 4) * 2;
            v = silu_stable(acc[f][m][i % 4] * xs * s1[i] + b1[i]) * (acc[f + 1][m][i % 4] * xs * s2[i] + b2[i]);
          } else {
            v = activate(acc[q * 2 + i / 4][m][i % 4] * xs * s1[i] + b1[i], e.act);
          }
          if (e.row && n + i < cols) v += load_any(e.row, e.row_dtype, row * e.srm + (n + i) * e.srn);
          o[i] = from_f32<T>(v);
        }
        T* to = y + (int64_t)row * sym + n * syn;
        if (wide && n + 8 <= cols) {
          store8<T>(to, o);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (n + i < cols) to[i * syn] = o[i];
        }
      }
    }
  }
}

// The K splits' sums, added in split order, then the epilogue: a thread per output.
template <typename T, bool SWIGLU>
__global__ __launch_bounds__(256) void w8a8_sum_kernel(T* y, const float* part, int M, int N, int splits, int64_t sym,
                                                       int64_t syn, W8Epi e, FastDiv cols, uint32_t total) {
  const uint32_t v = blockIdx.x * 256 + threadIdx.x;
  if (v >= total) return;
  uint32_t c;
  const uint32_t m = cols.divmod(v, c);
  const int half = N / 2;
  const float* p = part + (int64_t)m * N + c;
  const int64_t step = (int64_t)M * N;
  float a = 0.f, u = 0.f;
  for (int i = 0; i < splits; ++i) {
    a += p[i * step];
    if constexpr (SWIGLU) u += p[i * step + half];
  }
  y[(int64_t)m * sym + c * syn] = from_f32<T>(w8_out<SWIGLU>(e, a, u, m, c, half));
}

namespace {

template <typename T, int WN, int WM, int NT, int MT, int D, bool SWIGLU, int FORM, bool DMA>
int tile_launch(const W8Args& a, int splits) {
  constexpr int BN = WN * NT * 16, BM = WM * MT * 16;
  constexpr size_t lds = (size_t)kStageBytes<BN, BM> * D;
  static_assert(lds <= kMaxLds, "a launch fits the LDS of a CU");
  const int64_t nt = (a.N + BN - 1) / BN, mt = (a.M + BM - 1) / BM;
  if (nt * mt * splits > 0x7fffffffLL) return set_error(FD_EUNSUPPORTED, "too many tiles");
  auto kernel = w8a8_tile_kernel<T, WN, WM, NT, MT, D, SWIGLU, FORM, DMA>;
  if (!allow_lds(kernel, lds)) return set_error(FD_ELAUNCH, "cannot raise the LDS limit to %zu bytes", lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(nt * mt * splits)), dim3(WN * WM * kWave), lds, a.st,
                     static_cast<T*>(a.y), a.scratch, a.x, a.w, a.M, a.N, a.K, a.sxm, a.swn, a.sym, a.syn, a.e, (int)mt,
                     splits);
  return FD_OK;
}

template <typename T, bool SWIGLU, int FORM>
int pick_tile(const W8Args& a, int splits, bool dma) {
  if (!dma) return tile_launch<T, 2, 2, 4, 4, 2, SWIGLU, FORM, false>(a, splits);
  return tile_launch<T, 2, 2, 4, 4, 3, SWIGLU, FORM, true>(a, splits);
}

template <typename T, bool SWIGLU>
int tiles(const W8Args& a, int splits, bool dma) {
  if (splits == 1) return pick_tile<T, SWIGLU, W8_OUT>(a, 1, dma);
  const int rc = pick_tile<T, SWIGLU, W8_PART>(a, splits, dma);
  if (rc != FD_OK) return rc;
  const int cols = SWIGLU ? a.N / 2 : a.N;
  const uint32_t total = (uint32_t)a.M * (uint32_t)cols;  // splits > 1: few tiles, so M * N is small
  hipLaunchKernelGGL((w8a8_sum_kernel<T, SWIGLU>), dim3((total + 255) / 256), dim3(256), 0, a.st, static_cast<T*>(a.y),
                     a.scratch, a.M, a.N, splits, a.sym, a.syn, a.e, FastDiv((uint32_t)cols), total);
  return FD_OK;
}

// K splits of a product: enough for one workgroup on every CU, each with at least four stages.
int w8_splits(int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = ((N + 127) / 128) * ((M + 127) / 128), stages = (K + kStep - 1) / kStep;
  int64_t s = device_cus() / tiles;
  if (s > stages / 4) s = stages / 4;
  return s < 1 ? 1 : (int)s;
}

constexpr int64_t kMostIndex = 0x7fffffffLL - 512;  // indexes run to the end of the last tile and stage

}  // namespace
}  // namespace fd

using namespace fd;

extern "C" int fd_linear_w8a8_scratch(int64_t M, int64_t N, int64_t K, int64_t* bytes) {
  if (M < 0 || N < 0 || K < 0) return set_error(FD_EINVAL, "negative size");
  if (!bytes) return set_error(FD_EINVAL, "null pointer argument");
  *bytes = 0;
  if (M == 0 || N == 0 || M > kMostIndex || N > kMostIndex || K > kMostIndex) return FD_OK;
  const int s = w8_splits(M, N, K);
  if (s > 1) *bytes = (int64_t)s * M * N * 4;
  return FD_OK;
}

extern "C" int fd_linear_w8a8(void* y, const void* x8, const float* x_scale, const void* w8, const float* w_scale,
                              const void* bias, int bias_dtype, int activation, const void* row_add, int row_dtype,
                              int64_t M, int64_t N, int64_t K, int64_t sxm, int64_t swn, int64_t sb, int64_t srm,
                              int64_t srn, int64_t sym, int64_t syn, float* scratch, int64_t scratch_bytes,
                              int act_dtype, void* stream) {
  if (!check_act_dtype(act_dtype)) return FD_EINVAL;
  if (M < 0 || N < 0 || K < 0) return set_error(FD_EINVAL, "negative size");
  if (sxm < 0 || swn < 0 || sb < 0 || srm < 0 || srn < 0 || sym < 0 || syn < 0)
    return set_error(FD_EINVAL, "negative stride");
  if (activation < FD_ACT_NONE || activation > FD_ACT_SWIGLU)
    return set_error(FD_EINVAL, "activation must be one of FD_ACT_*, got %d", activation);
  const bool swiglu = activation == FD_ACT_SWIGLU;
  if (swiglu && N % 2 != 0) return set_error(FD_EINVAL, "FD_ACT_SWIGLU needs gate and up rows: N must be even");
  if (bias && !check_any_dtype(bias_dtype, "bias_dtype")) return FD_EINVAL;
  if (row_add && !check_any_dtype(row_dtype, "row_dtype")) return FD_EINVAL;
  if (M == 0 || N == 0) return FD_OK;
  if (!y || !x_scale || !w_scale || (K > 0 && (!x8 || !w8))) return set_error(FD_EINVAL, "null pointer argument");
  if (M > kMostIndex || N > kMostIndex || K > kMostIndex) return set_error(FD_EUNSUPPORTED, "too large");
  // tiles are stored while other workgroups still read their operands
  const int64_t cols = swiglu ? N / 2 : N, ny = span_bytes(M, cols, sym, syn, 2);
  if (overlaps(y, ny, x8, span_bytes(M, K, sxm, 1, 1)) || overlaps(y, ny, w8, span_bytes(N, K, swn, 1, 1)) ||
      overlaps(y, ny, x_scale, M * 4) || overlaps(y, ny, w_scale, N * 4) ||
      (bias && overlaps(y, ny, bias, span_bytes(1, N, 0, sb, dtype_bytes(bias_dtype)))) ||
      row_add_meets(row_add, row_dtype, srm, srn, y, act_dtype, sym, syn, M, cols))
    return set_error(FD_EUNSUPPORTED, "y must not overlap an operand, other than as row_add itself");
  if (scratch && !aligned16(scratch)) return set_error(FD_EUNSUPPORTED, "scratch must be 16-byte aligned");
  W8Args a{};
  a.y = y;
  a.x = static_cast<const uint8_t*>(x8);
  a.w = static_cast<const uint8_t*>(w8);
  a.M = (int)M;
  a.N = (int)N;
  a.K = (int)K;
  a.sxm = sxm;
  a.swn = swn;
  a.sym = sym;
  a.syn = syn;
  a.swiglu = swiglu;
  a.e = W8Epi{x_scale, w_scale, bias, bias_dtype, sb, activation, row_add, row_dtype, srm, srn};
  a.scratch = scratch;
  a.scratch_bytes = scratch ? scratch_bytes : 0;
  a.act_dtype = act_dtype;
  a.st = static_cast<hipStream_t>(stream);
  const bool dma = K % 16 == 0 && aligned16(x8) && aligned16(w8) && (M == 1 || sxm % 16 == 0) &&
                   (N == 1 || swn % 16 == 0);
  int splits = w8_splits(M, N, K);
  while (splits > 1 && a.scratch_bytes < (int64_t)splits * M * N * 4) --splits;
  const int rc = act_dtype == FD_F16 ? (swiglu ? tiles<f16, true>(a, splits, dma) : tiles<f16, false>(a, splits, dma))
                                     : (swiglu ? tiles<bf16, true>(a, splits, dma) : tiles<bf16, false>(a, splits, dma));
  if (rc != FD_OK) return rc;
  return check_launch();
}
