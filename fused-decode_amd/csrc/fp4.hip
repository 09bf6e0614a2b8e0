// Products with E2M1 weights in tiles of the output, for any number of activation rows from 2 on (fd_fp4.h has the
// mathematics), and the entry points.
//
// A workgroup of four waves owns BN weight rows x BM activation rows; each wave has its own weight rows and all of the
// activations. K goes in stages of 128, double-buffered: while a stage is multiplied, the next one's codes and
// activations come to LDS by DMA and its scales, a byte a lane, to registers. A wave turns its codes into matrix operands
// once and multiplies them by all of the tile's activation rows.
//
// Activations are rows of bfloat16, whole stages of them: float16 rows, and rows off alignment or of no whole stages, are
// first copied into scratch (fp4_x_kernel), float16 as its two parts, one behind the other.
//
// Where the output has fewer tiles than the GPU has room for, K is split over workgroups whose float32 sums go through
// scratch and are added in split order by a second launch.
//
// Traced medians: 384 x 4096 x 14336 bfloat16 79 to 86 us in separate runs (525 to 570 TFLOP/s) and 6.6 for the splits' sums,
// float16 132, 5.4 and 7.9 for the copy; 29 x 5003 x 2051 float16 12.2, 4.0 and 3.1. Each stage waits for all of its loads:
// the matrix cores are busy a quarter of the first one's cycles.
//
// LDS layout: activation rows of 16 chunks of 16 bytes, chunk c at c ^ (row mod 16), so that the lanes of a read (16
// rows, one chunk) hit distinct banks; codes 64 bytes a row, read in order.
#include "fd_fp4.h"

namespace fd {

constexpr int kF4Stage = 128;

enum Fp4Form { F4_OUT = 0, F4_PART = 1 };

template <int H, int NT, int MT>
constexpr int f4_stage_bytes() {
  return 4 * NT * 16 * 64 + MT * 16 * 256 * H;
}

// TAIL: whether K ends inside a piece. (Asked in the loop it costs 384 x 4096 x 14336 bfloat16 2 us of 89.)
template <typename T, int H, int NT, int MT, bool SWIGLU, int FORM, bool TAIL>
__global__ __launch_bounds__(256) void fp4_tile_kernel(T* y, float* part, const bf16* x, int64_t lo_off,
                                                       const uint8_t* w, const uint8_t* ws, int M, int N, int K,
                                                       int64_t sxm, int64_t swn, int64_t ssn, int64_t sym, int64_t syn,
                                                       Fp4Epi e, int mtiles, int splits) {
  static_assert(!SWIGLU || NT % 2 == 0, "gate and up tiles in turn");
  constexpr int BM = MT * 16, OUT = (SWIGLU ? 2 : 4) * NT * 16, WOUT = OUT / 4;  // output columns of a tile, of a wave
  constexpr int STAGE = f4_stage_bytes<H, NT, MT>(), WBYTES = 4 * NT * 1024;
  extern __shared__ __align__(16) u32x4 f4_smem[];
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane & 15, g = lane >> 4;
  const int half = N / 2, cols = SWIGLU ? half : N;

  // Consecutive blocks go to the eight XCDs in turn: each takes a contiguous run of tiles, the row blocks of one weight
  // tile next to each other.
  int tile;
  {
    const int b = (int)blockIdx.x, total = (int)gridDim.x, xcd = b & 7, q = total >> 3, rem = total & 7;
    tile = xcd * q + (xcd < rem ? xcd : rem) + (b >> 3);
  }
  const int mtile = tile % mtiles, rest = tile / mtiles, ntiles = (int)gridDim.x / (mtiles * splits);
  const int ntile = rest % ntiles, split = rest / ntiles;
  const int m0 = mtile * BM, n0 = ntile * OUT + wave * WOUT;  // this wave's first output column
  const int groups = (K + kGroupK - 1) / kGroupK, stages = (groups + 3) / 4;
  const int s0 = (int)((int64_t)stages * split / splits), s1 = (int)((int64_t)stages * (split + 1) / splits);

  // weight row at row t of this wave's tiles (past the last: one that exists, never stored)
  auto wrow = [&](int t) -> int64_t {
    if constexpr (SWIGLU) {
      const int n = n0 + (t >> 5) * 16 + (t & 15);
      return (n < half ? n : half - 1) + (int64_t)((t >> 4) & 1 ? half : 0);
    } else {
      const int n = n0 + t;
      return n < N ? n : N - 1;
    }
  };
  const unsigned lds0 = lds_addr(f4_smem);
  const uint8_t *wp[NT], *sp[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    wp[i] = w + wrow(i * 16 + lane / 4) * swn;
    sp[i] = ws + wrow(i * 16 + r) * ssn;
  }
  const bf16* xp[MT * H];  // this wave's quarter of the tile's activations: 4 rows to a KiB
#pragma unroll
  for (int i = 0; i < MT * H; ++i) {
    const int t = (i % MT) * 16 + wave * 4 + g, m = m0 + t;
    xp[i] = x + (i >= MT ? lo_off : 0) + (m < M ? m : M - 1) * sxm + ((lane & 15) ^ (t & 15)) * 8;
  }
  auto issue = [&](int s) {
    const unsigned to = lds0 + (unsigned)((s & 1) * STAGE);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int c = s * 4 + (lane & 3);  // past the last piece: the row's first, times activations that are zero
      dma16_at(wp[i] + (int64_t)(c < groups ? c : 0) * 16, to + (unsigned)((wave * NT + i) * 1024));
    }
#pragma unroll
    for (int i = 0; i < MT * H; ++i)
      dma16_at(xp[i] + (int64_t)s * kF4Stage, to + (unsigned)(WBYTES + i * 4096 + wave * 1024));
  };
  auto scales = [&](int s, uint32_t (&b)[NT]) {
    const int c = s * 4 + g;
#pragma unroll
    for (int i = 0; i < NT; ++i) b[i] = sp[i][c < groups ? c : 0];
#pragma unroll
    for (int i = 0; i < NT; ++i) b[i] = c < groups ? b[i] : 127u;
  };

  f32x4 acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  uint32_t sc[NT], next[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) next[n] = 127u;
  if (s0 < s1) {
    issue(s0);
    scales(s0, sc);
    wait_vm<0>();
    lds_barrier();
  }
  for (int s = s0; s < s1; ++s) {
    if (s + 1 < s1) {
      issue(s + 1);
      scales(s + 1, next);
    }
    __builtin_amdgcn_sched_barrier(0);
    const u32x4* wl = f4_smem + ((s & 1) * STAGE + wave * NT * 1024) / 16 + lane / 16 + (lane & 15) * 4;
    const u32x4* xl = f4_smem + ((s & 1) * STAGE + WBYTES) / 16 + r * 16;
    bf16x8 a[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      u32x4 c = wl[n * 64];
      if constexpr (TAIL) {
        if (s * 4 + g == groups - 1) c = fp4_tail(c, K % kGroupK);
      }
      const float f = e8m0_operand(sc[n]);
#pragma unroll
      for (int j = 0; j < 4; ++j) a[n][j] = fp4_to_bf16(c[j], f);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bf16x8 b = __builtin_bit_cast(bf16x8, xl[(h * MT + m) * 256 + ((4 * g + j) ^ r)]);
#pragma unroll
          for (int n = 0; n < NT; ++n) acc[n][m] = mfma16(a[n][j], b, acc[n][m]);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    wait_vm<0>();
    lds_barrier();  // stage s has been read by every wave, stage s + 1 is in LDS
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      asm volatile("" : "+v"(next[n]));  // waited for here, not behind the next stage's DMAs
      sc[n] = next[n];
    }
  }

#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int row = m0 + m * 16 + r;
    if (row >= M) continue;
#pragma unroll
    for (int n = 0; n < NT; n += SWIGLU ? 2 : 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = n0 + (SWIGLU ? n / 2 : n) * 16 + g * 4 + i;
        if (c >= cols) continue;
        const float v = acc[n][m][i], up = SWIGLU ? acc[n + (SWIGLU ? 1 : 0)][m][i] : 0.f;
        if constexpr (FORM == F4_PART) {
          float* to = part + ((int64_t)split * M + row) * N + c;
          to[0] = v;
          if constexpr (SWIGLU) to[half] = up;
        } else {
          y[row * sym + c * syn] = from_f32<T>(fp4_out<SWIGLU>(e, v, up, row, c, half));
        }
      }
    }
  }
}

// The K splits' sums, added in split order, then the epilogue: a thread per output.
template <typename T, bool SWIGLU>
__global__ __launch_bounds__(256) void fp4_sum_kernel(T* y, const float* part, int M, int N, int splits, int64_t sym,
                                                      int64_t syn, Fp4Epi e, FastDiv width, uint32_t total) {
  const uint32_t v = blockIdx.x * 256 + threadIdx.x;
  if (v >= total) return;
  uint32_t c;
  const uint32_t m = width.divmod(v, c);
  const int half = N / 2;
  const float* p = part + (int64_t)m * N + c;
  const int64_t step = (int64_t)M * N;
  float a = 0.f, u = 0.f;
  for (int i = 0; i < splits; ++i) {
    a += p[i * step];
    if constexpr (SWIGLU) u += p[i * step + half];
  }
  y[(int64_t)m * sym + (int64_t)c * syn] = from_f32<T>(fp4_out<SWIGLU>(e, a, u, m, c, half));
}

// Activation rows as bfloat16 rows of Kq, zeros past K: a thread per 8 elements, float16's second parts `lo_off` further.
template <typename T>
__global__ __launch_bounds__(256) void fp4_x_kernel(bf16* to, int64_t lo_off, const T* x, int K, int64_t sxm,
                                                    FastDiv pieces, uint32_t total) {
  const uint32_t v = blockIdx.x * 256 + threadIdx.x;
  if (v >= total) return;
  uint32_t piece;
  const uint32_t row = pieces.divmod(v, piece);
  const int k = (int)piece * 8;
  const T* p = x + row * sxm;
  typename Vec8<T>::type in;
  if (k + 8 <= K) {
    in = load8_any<T>(p + k);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) in[i] = k + i < K ? p[k + i] : (T)0.f;
  }
  if constexpr (std::is_same<T, f16>::value) {
    bf16x8 hi, lo;
    split_f16(in, hi, lo);
    store8<bf16>(to + (int64_t)v * 8, hi);
    store8<bf16>(to + lo_off + (int64_t)v * 8, lo);
  } else {
    store8<bf16>(to + (int64_t)v * 8, in);
  }
}

namespace {

constexpr int64_t kF4Most = 0x7fffffffLL - 8192;  // indexes run to the end of the last tile, stage and chunk

struct Fp4Plan {
  int splits;
  int64_t kq;  // elements of a copied activation row, 0 where the rows are taken as they are
};

constexpr int kF4BN = 128;

int f4_mt(int64_t M) { return M <= 16 ? 1 : M <= 32 ? 2 : 4; }

// K splits: as many as give every CU two workgroups, each with at least four stages.
int f4_splits(int64_t M, int64_t N, int64_t K) {
  const int64_t stages = (K + kF4Stage - 1) / kF4Stage, bm = f4_mt(M) * 16;
  const int64_t tiles = (N + kF4BN - 1) / kF4BN * ((M + bm - 1) / bm);
  int64_t s = 2 * device_cus() / (tiles > 0 ? tiles : 1);
  if (s > stages / 4) s = stages / 4;
  return s < 1 ? 1 : s > 32 ? 32 : (int)s;
}

// Scratch bytes of the copied activations.
int64_t f4_copy_bytes(int64_t M, int64_t K, int act_dtype) {
  return M * ((K + kF4Stage - 1) / kF4Stage * kF4Stage) * (act_dtype == FD_F16 ? 4 : 2);
}

// Scratch bytes of a product in tiles: the copies, and the sums of K splits.
int64_t f4_scratch_bytes(int64_t M, int64_t N, int64_t K, int act_dtype) {
  const int64_t s = f4_splits(M, N, K);
  return f4_copy_bytes(M, K, act_dtype) + (s > 1 ? s * M * N * 4 : 0);
}

template <typename T, int H, int NT, int MT, bool SWIGLU, int FORM, bool TAIL>
int f4_tile_tail(const Fp4Args& a, const bf16* x, int64_t lo_off, int64_t sxm, int splits) {
  constexpr size_t lds = 2 * (size_t)f4_stage_bytes<H, NT, MT>();
  static_assert(lds <= kMaxLds, "a launch fits the LDS of a CU");
  const int out = (SWIGLU ? 2 : 4) * NT * 16, cols = SWIGLU ? a.N / 2 : a.N;
  const int64_t nt = ((int64_t)cols + out - 1) / out, mt = ((int64_t)a.M + MT * 16 - 1) / (MT * 16);
  if (nt * mt * splits * 256 > 0xffffffffLL) return set_error(FD_EUNSUPPORTED, "too many tiles");
  auto kernel = fp4_tile_kernel<T, H, NT, MT, SWIGLU, FORM, TAIL>;
  if (!allow_lds(kernel, lds)) return set_error(FD_ELAUNCH, "cannot raise the LDS limit to %zu bytes", lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(nt * mt * splits)), dim3(256), lds, a.st, static_cast<T*>(a.y), a.scratch,
                     x, lo_off, a.w, a.ws, a.M, a.N, a.K, sxm, a.swn, a.ssn, a.sym, a.syn,
                     a.e, (int)mt, splits);
  return FD_OK;
}

template <typename T, int H, int NT, int MT, bool SWIGLU, int FORM>
int f4_tile_launch(const Fp4Args& a, const bf16* x, int64_t lo_off, int64_t sxm, int splits) {
  return a.K % kGroupK ? f4_tile_tail<T, H, NT, MT, SWIGLU, FORM, true>(a, x, lo_off, sxm, splits)
                       : f4_tile_tail<T, H, NT, MT, SWIGLU, FORM, false>(a, x, lo_off, sxm, splits);
}

template <typename T, bool SWIGLU, int FORM>
int f4_pick(const Fp4Args& a, const bf16* x, int64_t lo_off, int64_t sxm, int splits) {
  constexpr int H = std::is_same<T, f16>::value ? 2 : 1, NT = kF4BN / 64;
  switch (f4_mt(a.M)) {
    case 1: return f4_tile_launch<T, H, NT, 1, SWIGLU, FORM>(a, x, lo_off, sxm, splits);
    case 2: return f4_tile_launch<T, H, NT, 2, SWIGLU, FORM>(a, x, lo_off, sxm, splits);
    default: return f4_tile_launch<T, H, NT, 4, SWIGLU, FORM>(a, x, lo_off, sxm, splits);
  }
}

template <typename T, bool SWIGLU>
int f4_product(Fp4Args a) {
  if (a.M == 1) return fp4_one_launch(a);
  if (fp4_few_fits(a.M, a.K, SWIGLU) && (fp4_few_wins(a.M, a.K, a.act_dtype) ||
                                         a.scratch_bytes < f4_scratch_bytes(a.M, a.N, a.K, a.act_dtype)))
    return fp4_few_launch(a);  // (it needs none)
  constexpr bool F16 = std::is_same<T, f16>::value;
  const bf16* x = static_cast<const bf16*>(a.x);
  int64_t sxm = a.sxm, lo_off = 0;
  const bool direct = !F16 && a.K % kF4Stage == 0 && aligned16(a.x) && (a.M == 1 || a.sxm % 8 == 0);
  if (!direct && a.K > 0) {
    const int64_t bytes = f4_copy_bytes(a.M, a.K, a.act_dtype);
    if (a.scratch_bytes < bytes) return set_error(FD_EUNSUPPORTED, "the activations' copy needs scratch");
    const int64_t pieces = ((int64_t)a.K + kF4Stage - 1) / kF4Stage * (kF4Stage / 8), total = a.M * pieces;
    if (total > 0xffffff00LL) return set_error(FD_EUNSUPPORTED, "too large");
    bf16* to = reinterpret_cast<bf16*>(a.scratch);
    sxm = pieces * 8;
    lo_off = a.M * sxm;
    hipLaunchKernelGGL((fp4_x_kernel<T>), dim3((unsigned)((total + 255) / 256)), dim3(256), 0, a.st, to, lo_off,
                       static_cast<const T*>(a.x), a.K, a.sxm, FastDiv((uint32_t)pieces), (uint32_t)total);
    x = to;
    a.scratch += bytes / 4;
    a.scratch_bytes -= bytes;
  }
  int splits = f4_splits(a.M, a.N, a.K);
  while (splits > 1 && a.scratch_bytes < (int64_t)splits * a.M * a.N * 4) --splits;
  if (splits == 1) return f4_pick<T, SWIGLU, F4_OUT>(a, x, lo_off, sxm, 1);
  const int rc = f4_pick<T, SWIGLU, F4_PART>(a, x, lo_off, sxm, splits);
  if (rc != FD_OK) return rc;
  const int cols = SWIGLU ? a.N / 2 : a.N;
  const uint32_t total = (uint32_t)a.M * (uint32_t)cols;  // splits > 1: few tiles, so M * N is small
  hipLaunchKernelGGL((fp4_sum_kernel<T, SWIGLU>), dim3((total + 255) / 256), dim3(256), 0, a.st, static_cast<T*>(a.y),
                     a.scratch, a.M, a.N, splits, a.sym, a.syn, a.e, FastDiv((uint32_t)cols), total);
  return FD_OK;
}

}  // namespace
}  // namespace fd

using namespace fd;

extern "C" int fd_linear_fp4_scratch(int64_t M, int64_t N, int64_t K, int act_dtype, int64_t* bytes) {
  if (!check_act_dtype(act_dtype)) return FD_EINVAL;
  if (M < 0 || N < 0 || K < 0) return set_error(FD_EINVAL, "negative size");
  if (!bytes) return set_error(FD_EINVAL, "null pointer argument");
  *bytes = 0;
  if (M == 0 || N == 0 || K == 0 || M > kF4Most || N > kF4Most || K > kF4Most) return FD_OK;
  if (M == 1 || (fp4_few_wins(M, K, act_dtype) && fp4_few_fits(M, K, false) && fp4_few_fits(M, K, true))) return FD_OK;
  *bytes = f4_scratch_bytes(M, N, K, act_dtype);
  return FD_OK;
}

extern "C" int fd_linear_fp4(void* y, const void* x, const void* w4, const void* w_scale, const void* bias,
                             int bias_dtype, int activation, const void* row_add, int row_dtype, int64_t M, int64_t N,
                             int64_t K, int64_t sxm, int64_t swn, int64_t ssn, int64_t sb, int64_t srm, int64_t srn,
                             int64_t sym, int64_t syn, float* scratch, int64_t scratch_bytes, int act_dtype,
                             void* stream) {
  if (!check_act_dtype(act_dtype)) return FD_EINVAL;
  if (M < 0 || N < 0 || K < 0) return set_error(FD_EINVAL, "negative size");
  if (sxm < 0 || swn < 0 || ssn < 0 || sb < 0 || srm < 0 || srn < 0 || sym < 0 || syn < 0)
    return set_error(FD_EINVAL, "negative stride");
  if (activation < FD_ACT_NONE || activation > FD_ACT_SWIGLU)
    return set_error(FD_EINVAL, "activation must be one of FD_ACT_*, got %d", activation);
  const bool swiglu = activation == FD_ACT_SWIGLU;
  if (swiglu && N % 2 != 0) return set_error(FD_EINVAL, "FD_ACT_SWIGLU needs gate and up rows: N must be even");
  if (bias && !check_any_dtype(bias_dtype, "bias_dtype")) return FD_EINVAL;
  if (row_add && !check_any_dtype(row_dtype, "row_dtype")) return FD_EINVAL;
  if (M == 0 || N == 0) return FD_OK;
  if (!y || (K > 0 && (!x || !w4 || !w_scale))) return set_error(FD_EINVAL, "null pointer argument");
  if (M > kF4Most || N > kF4Most || K > kF4Most) return set_error(FD_EUNSUPPORTED, "too large");
  if (K > 0 && (!aligned16(w4) || (N > 1 && swn % 16 != 0)))
    return set_error(FD_EUNSUPPORTED, "rows of codes must be 16-byte aligned");
  const int64_t cols = swiglu ? N / 2 : N, groups = (K + kGroupK - 1) / kGroupK;
  if (rows_meet(fd_rows{1, 1, M, 0, 0, sym, syn, cols}))
    return set_error(FD_EINVAL, "y's elements must not share memory");
  // tiles are stored while other workgroups still read their operands
  const int64_t ny = span_bytes(M, cols, sym, syn, 2);
  if (overlaps(y, ny, x, span_bytes(M, K, sxm, 1, 2)) || overlaps(y, ny, w4, span_bytes(N, groups * 16, swn, 1, 1)) ||
      overlaps(y, ny, w_scale, span_bytes(N, groups, ssn, 1, 1)) ||
      (bias && overlaps(y, ny, bias, span_bytes(1, N, 0, sb, dtype_bytes(bias_dtype)))) ||
      row_add_meets(row_add, row_dtype, srm, srn, y, act_dtype, sym, syn, M, cols))
    return set_error(FD_EUNSUPPORTED, "y must not overlap an operand, other than as row_add itself");
  if (scratch && !aligned16(scratch)) return set_error(FD_EUNSUPPORTED, "scratch must be 16-byte aligned");
  Fp4Args a{};
  a.y = y;
  a.x = x;
  a.w = static_cast<const uint8_t*>(w4);
  a.ws = static_cast<const uint8_t*>(w_scale);
  a.M = (int)M;
  a.N = (int)N;
  a.K = (int)K;
  a.sxm = sxm;
  a.swn = swn;
  a.ssn = ssn;
  a.sym = sym;
  a.syn = syn;
  a.swiglu = swiglu;
  a.e = Fp4Epi{bias, bias_dtype, sb, activation, row_add, row_dtype, srm, srn};
  a.scratch = scratch;
  a.scratch_bytes = scratch ? scratch_bytes : 0;
  a.act_dtype = act_dtype;
  a.st = static_cast<hipStream_t>(stream);
  const int rc = act_dtype == FD_F16 ? (swiglu ? f4_product<f16, true>(a) : f4_product<f16, false>(a))
                                     : (swiglu ? f4_product<bf16, true>(a) : f4_product<bf16, false>(a));
  if (rc != FD_OK) return rc;
  return check_launch();
}
