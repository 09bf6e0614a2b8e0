// Products of E4M3 activations and weights in tiles of the output, for any number of
// activation rows (fd_w8a8.h has the mathematics).
//
// A workgroup of WN x WM waves owns BN weight rows x BM activation rows and walks K in stages
// of 128. Both tiles of a stage go to LDS in a ring of D stages by DMA (global_load_lds_dwordx4), so
// rows have to be 16-byte aligned: others are copied into scratch first (w8a8_align_kernel). The
// DMAs are inline assembly, so the compiler sees plain LDS reads and schedules and waits for those
// itself; the vmcnt waits are explicit.
//
// The matrix cores are fed from registers that hold the whole stage: weight tile n's registers
// are refilled with the next stage's once row n of the wave's tiles is multiplied, the
// activations' during the last row. So no MFMA waits for the LDS read in front of it, the LDS
// reads lie evenly between the MFMAs, a buffer is free for the DMAs of stage s + D as soon as
// stage s begins, and one barrier a stage is enough. It stands behind the first row's MFMAs,
// which run on while the waves meet.
//
// LDS layout: a tile row is 8 chunks of 16 bytes, chunk c at slot c ^ (row mod 8), so the 8
// lanes of a read (8 rows, one chunk) hit distinct bank groups and a DMA instruction still fills
// 1 KiB in lane order. At the end each wave's sums go through LDS and leave along the rows in
// 16-byte nontemporal stores. SWIGLU: gate and up tiles of 16 rows in turn, so that a lane finds
// both of an output.
//
// Large products run at the clock that their power leaves, with the matrix cores busy 55% of the
// cycles (8192 x 28672 x 4096 SWIGLU 755 us captured alone, 790 to 830 on a busy card, 2550 to 2320
// TFLOP/s at 1.98 GHz; MFMA alone on random codes reaches 3500), ordinary ones at the rate at which the
// L2s feed a CU, 46 KB a microsecond over the whole kernel, 55 to 60 between its start and end (2048 x
// 4096 x 4096 35 us, 1950 TFLOP/s), which smaller tiles load more of. Nontemporal stores leave the L2s to the operands
// (825 -> 745 us).
//
// Where the output has fewer tiles than the GPU has room for, K is split over workgroups whose
// float32 sums go through scratch and are added in split order by a second launch.
#include <type_traits>
#include <utility>

#include "fd_w8a8.h"

namespace fd {

template <int BN, int BM> constexpr int kStageBytes = (BN + BM) * kStep;

// 16-row tiles of a wave's sums that its workgroup's LDS holds at once, without a workgroup less on a CU.
template <int NW, int NT, int MT, int RING>
constexpr int epi_tiles() {
  const int limit = (int)kMaxLds / ((int)kMaxLds / RING);
  int em = MT;
  while (em > 1 && (MT % em != 0 || NW * em * 16 * (NT * 16 + 4) * 4 + NW * MT * 64 > limit)) --em;
  return em;
}
template <int NW, int NT, int MT, int RING>
constexpr size_t epi_bytes() {
  return (size_t)NW * epi_tiles<NW, NT, MT, RING>() * 16 * (NT * 16 + 4) * 4 + NW * MT * 64;
}

template <typename F, int... I>
__device__ __forceinline__ void each_part(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}

// Elements n .. n + 7 of p (at n * stride + shift * stride) in float32: one or two loads where they lie together,
// the last element again past cols; zeros of no p.
__device__ __forceinline__ void load8_vec(const void* p, int dtype, int n, int64_t stride, int cols, float (&f)[8],
                                          int shift = 0) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.f;
  } else if (stride == 1 && n + 8 <= cols) {
    const char* q = static_cast<const char*>(p) + (int64_t)(n + shift) * (dtype == FD_F32 ? 4 : 2);
    const u32x4 lo = *reinterpret_cast<const u32x4_any*>(q);
    if (dtype == FD_F32) {
      const u32x4 hi = *reinterpret_cast<const u32x4_any*>(q + 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[i] = __builtin_bit_cast(float, (uint32_t)lo[i]);
        f[i + 4] = __builtin_bit_cast(float, (uint32_t)hi[i]);
      }
    } else if (dtype == FD_F16) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = to_f32(__builtin_bit_cast(f16x8, lo)[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = to_f32(__builtin_bit_cast(bf16x8, lo)[i]);
    }
  } else {
    for (int i = 0; i < 8; ++i) {
      const int c = n + i < cols ? n + i : cols - 1;
      f[i] = load_any(p, dtype, (int64_t)(c + shift) * stride);
    }
  }
}

// A K split's sums of columns n .. n + 7 of a row.
__device__ __forceinline__ void store8_part(float* to, const float (&v)[8], int n, int cols) {
  if (n + 8 <= cols) {
    typedef f32x4 f32x4_any __attribute__((aligned(4)));
    *reinterpret_cast<f32x4_any*>(to) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4_any*>(to + 4) = f32x4{v[4], v[5], v[6], v[7]};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < cols) to[i] = v[i];
  }
}

enum W8Form { W8_OUT = 0, W8_PART = 1 };

// Tiles of a group of row blocks: an XCD's workgroups share the activations of kGroup row blocks
// and walk the weights (8192 x 28672 x 4096: 4, 8, 16 row blocks 750, 746, 781 us).
constexpr int kGroup = 8;

template <typename T, int PW, int WN, int WM, int NT, int MT, int D, bool SWIGLU, int FORM>
__global__ __launch_bounds__((WN * WM + PW) * kWave) void w8a8_tile_kernel(T* y, float* part, const uint8_t* x,
                                                                    const uint8_t* w, int M, int N, int K, int64_t sxm,
                                                                    int64_t swn, int64_t sym, int64_t syn, W8Epi e,
                                                                    int mtiles, int splits) {
  typedef typename Vec8<T>::type V8;
  constexpr int NW = WN * WM, LW = PW ? PW : NW, BN = WN * NT * 16, BM = WM * MT * 16;
  constexpr int AOPS = BN / 8 / LW, BOPS = BM / 8 / LW, OPS = AOPS + BOPS;  // of a wave that loads
  static_assert(AOPS * 8 * LW == BN && BOPS * 8 * LW == BM, "the loading waves share a stage evenly");
  static_assert(NT > 1 && (!SWIGLU || NT % 2 == 0), "gate and up tiles in turn");
  extern __shared__ __align__(16) u32x4 w8_smem[];
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int wm = wave % WM, wn = wave / WM;
  const int lw = PW ? wave - NW : wave;  // which of the loading waves
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
  int ntile, mtile;
  {
    const int ntiles = (int)gridDim.x / splits / mtiles;
    const int G = kGroup, per = G * ntiles, gi = tile / per, rem = tile - gi * per;
    const int gs = mtiles - gi * G < G ? mtiles - gi * G : G;
    ntile = rem / gs;
    mtile = gi * G + rem - ntile * gs;
  }
  const int m0 = mtile * BM;
  const int half = N / 2, cols = SWIGLU ? half : N;
  constexpr int OUT = SWIGLU ? BN / 2 : BN, WOUT = OUT / WN;  // output columns of a tile, of a wave
  const int stages_all = (K + kStep - 1) / kStep;
  const int s0 = (int)((int64_t)stages_all * split / splits);
  const int ns = (int)((int64_t)stages_all * (split + 1) / splits) - s0;
  // With one row block no two workgroups share weights: each starts its K sweep at a stage of its
  // own, so that they do not all read one line of every weight row at once (120 x 28672 x 4096:
  // 33.1 -> 28.2 us). With more, workgroups that read the same lines together are faster.
  const int rot = mtiles == 1 ? (int)((int64_t)(ntile & 31) * ns >> 5) : 0;
  auto stage_k = [&](int s) {  // first k of this block's s-th stage
    const int u = s + rot;
    return (s0 + (u >= ns ? u - ns : u)) * kStep;
  };

  // weight row at LDS row t of the tile (past the last: one that exists, never stored); SWIGLU:
  // a wave's 16-row tiles are gate and up rows in turn
  auto wrow = [&](int t) -> int64_t {
    if constexpr (SWIGLU) {
      const int f = t / 16, n = ntile * OUT + (f >> 1) * 16 + (t & 15);
      return (n < half ? n : half - 1) + (int64_t)((f & 1) ? half : 0);
    } else {
      const int n = ntile * OUT + t;
      return n < N ? n : N - 1;
    }
  };

  const unsigned lds0 = lds_addr(w8_smem);
  constexpr unsigned kStage = (unsigned)kStageBytes<BN, BM>;
  // a scalar base for the tile's weight rows (SWIGLU: and its up rows) and activation rows, and a 32-bit
  // offset a lane
  const int64_t n_first = (int64_t)ntile * OUT < cols ? (int64_t)ntile * OUT : cols - 1;
  const uint8_t* const wbase = w + n_first * swn;
  const uint8_t* const ubase = SWIGLU ? wbase + (int64_t)half * swn : wbase;
  const uint8_t* const xbase = x + (int64_t)m0 * sxm;
  unsigned voff[OPS];
  int off[OPS];
#pragma unroll
  for (int i = 0; i < OPS; ++i) {
    const bool wt = i < AOPS;
    const int t = (wt ? lw * AOPS + i : lw * BOPS + i - AOPS) * 8 + lane / 8;  // its row of the tile
    const int m = m0 + t;
    const int64_t row = wt ? wrow(t) : (m < M ? m : M - 1);
    off[i] = ((lane & 7) ^ (t & 7)) * 16;
    const int64_t first = n_first + (SWIGLU && ((t >> 4) & 1) ? half : 0);
    voff[i] = (unsigned)(wt ? (row - first) * swn : (row - m0) * sxm) + off[i];
  }
  auto place = [&](int i) {  // byte address in a stage of this wave's i-th KiB: weights, then activations
    return (unsigned)(i < AOPS ? lw * AOPS + i : BN / 8 + lw * BOPS + i - AOPS) * 1024u;
  };
  auto issue_one = [&](int s, int i) {
    const int k0 = stage_k(s);
    const bool up = SWIGLU && (((lw * AOPS + i) >> 1) & 1);  // 8 rows of an up tile
    const uint8_t* base = i < AOPS ? (up ? ubase : wbase) : xbase;
    const unsigned to = lds0 + (unsigned)(s % D) * kStage + place(i), o = voff[i];
    if (k0 + kStep <= K)
      dma16(base + k0, o, to);
    else  // pieces past K: the row's start
      dma16(base, k0 + off[i] < K ? o + (unsigned)k0 : o - (unsigned)off[i], to);
  };
  auto zero_tail = [&](int s) {  // DMA past K brought the row's start: the activations there become zero
    const int k0 = stage_k(s);
    if (k0 + kStep > K) {
#pragma unroll
      for (int i = AOPS; i < OPS; ++i)
        if (k0 + off[i] >= K) ds_zero16(lds0 + (unsigned)(s % D) * kStage + place(i) + (unsigned)lane * 16u);
    }
  };

  f32x4 acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};

  // this lane's two chunks of a tile row (u32x4 entries): row r of a 16-row tile, r mod 8 is
  // every tile's swizzle
  const int c0 = g ^ (r & 7), c1 = (4 + g) ^ (r & 7);
  // The loads of a stage and its waits, by the waves that load: all of them, or PW of their own
  // whose DMAs, each of which holds its wave for over a hundred cycles, then hold no MFMA.
  auto load_first = [&]() {
    const int pre = ns < D ? ns : D;
    for (int s = 0; s < pre; ++s)
#pragma unroll
      for (int i = 0; i < OPS; ++i) issue_one(s, i);
    if (ns >= D)
      wait_vm<OPS*(D - 1)>();
    else
      wait_vm<0>();
    zero_tail(0);
  };
  auto wait_next = [&](int s) {  // stage s + 1 has landed
    if (s + D <= ns)             // issued so far: to stage s + D - 1
      wait_vm<OPS*(D - 2)>();
    else
      wait_vm<0>();
    if (s + 1 < ns) zero_tail(s + 1);
  };
  if constexpr (PW > 0) {
    if (wave >= NW) {
      if (ns > 0) {
        load_first();
        lds_barrier();
      }
      for (int s = 0; s < ns; ++s) {
        wait_next(s);
        lds_barrier();
        if (s + D < ns) {
#pragma unroll
          for (int i = 0; i < OPS; ++i) issue_one(s + D, i);
        }
      }
      return;  // a wave that has ended is not waited for at a barrier
    }
  }

  u32x4 a0[NT], a1[NT], b0[MT], b1[MT];
  auto load_a = [&](int s, int n) {
    const u32x4* p = w8_smem + (s % D) * (kStage / 16) + ((wn * NT + n) * 16 + r) * 8;
    a0[n] = p[c0];
    a1[n] = p[c1];
  };
  auto load_b = [&](int s, int m) {
    const u32x4* p = w8_smem + (s % D) * (kStage / 16) + (BN + (wm * MT + m) * 16 + r) * 8;
    b0[m] = p[c0];
    b1[m] = p[c1];
  };
  if (ns > 0) {
    if constexpr (PW == 0) load_first();
    lds_barrier();
#pragma unroll
    for (int n = 0; n < NT; ++n) load_a(0, n);
#pragma unroll
    for (int m = 0; m < MT; ++m) load_b(0, m);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0), so that the loop's waits count its own reads alone
  }
  for (int s = 0; s < ns; ++s) {
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[0][m] = mfma_e4m3(a0[0], a1[0], b0[m], b1[m], acc[0][m]);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (PW == 0) wait_next(s);
    lds_barrier();  // stage s is in every wave's registers, stage s + 1 in LDS
    const bool more = PW == 0 && s + D < ns;
    // (past the last stage the registers are refilled with what the ring holds, and not used)
#pragma unroll
    for (int n = 1; n < NT; ++n) {
      load_a(s + 1, n - 1);
      if constexpr (PW == 0) {
        if (more) {
#pragma unroll
          for (int i = OPS * (n - 1) / (NT - 1); i < OPS * n / (NT - 1); ++i) issue_one(s + D, i);
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        acc[n][m] = mfma_e4m3(a0[n], a1[n], b0[m], b1[m], acc[n][m]);
        if (n == NT - 1) {
          __builtin_amdgcn_sched_barrier(0);
          load_b(s + 1, m);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    load_a(s + 1, NT - 1);
    __builtin_amdgcn_sched_barrier(0);
  }

  // The sums go through LDS, EM tiles of 16 activation rows of a wave at a time, and leave along the
  // rows: a lane has the same eight output columns of every row it writes.
  constexpr int EM = epi_tiles<NW, NT, MT, (int)(kStageBytes<BN, BM> * D)>(), PITCH = NT * 16 + 4, TPR = WOUT / 8,
                RPP = kWave / TPR, U = EM * 16 >= RPP * 2 ? 2 : 1;
  static_assert(EM * 16 % (RPP * U) == 0, "whole passes");
  const int n0 = ntile * OUT + wn * WOUT;  // this wave's first output column
  float* const all = reinterpret_cast<float*>(w8_smem);
  float* const sums = all + wave * (EM * 16 * PITCH);
  float* const xsl = all + NW * (EM * 16 * PITCH) + wave * (MT * 16);
  const int oc = lane % TPR * 8, n = n0 + oc, rr = lane / TPR;
  const int sc = SWIGLU ? (oc >> 4) * 32 + (oc & 15) : oc;  // its column of the sums; SWIGLU: up 16 further
  const int mrow = m0 + wm * MT * 16;
  const bool whole = n + 8 <= cols, wide = whole && syn == 1;
  const int add_dtype = e.row_dtype, add = !e.row ? 0 : e.srn != 1 ? 3 : add_dtype == FD_F32 ? 2 : 1;
  float scale1[8], bias1[8], scale2[SWIGLU ? 8 : 1], bias2[SWIGLU ? 8 : 1], xv[(MT * 16 + kWave - 1) / kWave];
  if constexpr (FORM == W8_OUT) {
    load8_vec(e.ws, FD_F32, n, 1, cols, scale1);
    load8_vec(e.bias, e.bias_dtype, n, e.sb, cols, bias1);
    if constexpr (SWIGLU) {
      load8_vec(e.ws + half, FD_F32, n, 1, cols, scale2);
      load8_vec(e.bias, e.bias_dtype, n, e.sb, cols, bias2, half);
    }
#pragma unroll
    for (int i = 0; i < MT * 16; i += kWave) {
      const int row = mrow + i + lane;
      xv[i / kWave] = e.xs[row < M ? row : M - 1];
    }
  }
  auto part_of = [&](auto which) {
    constexpr int h = decltype(which)::value;
    if constexpr (h == 0) lds_barrier();  // the last stage has been read everywhere
    if constexpr (FORM == W8_OUT && h == 0) {
#pragma unroll
      for (int i = 0; i < MT * 16; i += kWave)
        if (i + lane < MT * 16) xsl[i + lane] = xv[i / kWave];
    }
#pragma unroll
    for (int m = 0; m < EM; ++m)
#pragma unroll
      for (int f = 0; f < NT; ++f)
        *reinterpret_cast<f32x4*>(sums + (m * 16 + r) * PITCH + f * 16 + g * 4) = acc[f][h * EM + m];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 1
    for (int t0 = rr; t0 < EM * 16; t0 += RPP * U) {
      u32x4 lo[U], hi[U];
      if (FORM == W8_OUT && whole && (add == 1 || add == 2)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int row = mrow + h * EM * 16 + t0 + u * RPP;
          const int64_t at = (row < M ? row : M - 1) * e.srm + n;
          const char* p = static_cast<const char*>(e.row) + at * (add == 2 ? 4 : 2);
          lo[u] = *reinterpret_cast<const u32x4_any*>(p);
          if (add == 2) hi[u] = *reinterpret_cast<const u32x4_any*>(p + 16);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = t0 + u * RPP, row = mrow + h * EM * 16 + t;
        const float* p = sums + t * PITCH + sc;
        float v[8], up[SWIGLU ? 8 : 1];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[i] = p[i];
          if constexpr (SWIGLU) up[i] = p[16 + i];
        }
        if constexpr (FORM == W8_PART) {
          if (row < M) {
            float* const to = part + ((int64_t)split * M + row) * N + n;
            store8_part(to, v, n, cols);
            if constexpr (SWIGLU) store8_part(to + half, up, n, cols);
          }
        } else {
          const float xs = xsl[h * EM * 16 + t];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            v[i] = v[i] * xs * scale1[i] + bias1[i];
            if constexpr (SWIGLU) v[i] = times_sigmoid(v[i], v[i]) * (up[i] * xs * scale2[i] + bias2[i]);
          }
          if constexpr (!SWIGLU) activate(v, e.act);
          if (row >= M || n >= cols) continue;
          if (add) {
            if (!whole || add == 3) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (n + i < cols) v[i] += load_any(e.row, add_dtype, row * e.srm + (n + i) * e.srn);
            } else if (add == 2) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                v[i] += __builtin_bit_cast(float, (uint32_t)lo[u][i]);
                v[i + 4] += __builtin_bit_cast(float, (uint32_t)hi[u][i]);
              }
            } else if (add_dtype == FD_F16) {
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] += to_f32(__builtin_bit_cast(f16x8, lo[u])[i]);
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] += to_f32(__builtin_bit_cast(bf16x8, lo[u])[i]);
            }
          }
          V8 o;
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = from_f32<T>(v[i]);
          T* to = y + (int64_t)row * sym + n * syn;
          if (wide) {
            store8_any<T>(to, o);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (n + i < cols) to[i * syn] = o[i];
          }
        }
      }
    }
  };
  each_part(part_of, std::make_integer_sequence<int, MT / EM>{});
}

// The K splits' sums, added in split order, then the epilogue: a thread per four columns of a
// row, with four splits' sums on the way at once.
template <typename T, bool SWIGLU>
__global__ __launch_bounds__(256) void w8a8_sum_kernel(T* y, const float* part, int M, int N, int splits, int64_t sym,
                                                       int64_t syn, W8Epi e, FastDiv quads, uint32_t total) {
  const uint32_t v = blockIdx.x * 256 + threadIdx.x;
  if (v >= total) return;
  uint32_t q;
  const uint32_t m = quads.divmod(v, q);
  const int c = (int)q * 4, half = N / 2, cols = SWIGLU ? half : N;
  const float* p = part + (int64_t)m * N + c;
  const int64_t step = (int64_t)M * N;
  f32x4 a = {0.f, 0.f, 0.f, 0.f}, u = a;
  if (N % 4 == 0 && (!SWIGLU || half % 4 == 0)) {
    for (int i = 0; i < splits; i += 4) {
      f32x4 t[4], w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float* at = p + (i + j < splits ? i + j : splits - 1) * step;
        t[j] = *reinterpret_cast<const f32x4*>(at);
        if constexpr (SWIGLU) w[j] = *reinterpret_cast<const f32x4*>(at + half);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j < splits) {
          a += t[j];
          if constexpr (SWIGLU) u += w[j];
        }
    }
  } else {
    for (int i = 0; i < splits; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < cols) {
          a[j] += p[i * step + j];
          if constexpr (SWIGLU) u[j] += p[i * step + half + j];
        }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (c + j < cols)
      y[(int64_t)m * sym + (c + j) * syn] = from_f32<T>(w8_out<SWIGLU>(e, a[j], u[j], m, c + j, half));
}

namespace {

constexpr int64_t kMostIndex = 0x7fffffffLL - 512;  // indexes run to the end of the last tile and stage
constexpr int64_t kMostStride = 1 << 23;            // 256 rows of it, and a row, are below 2^32 bytes

template <typename T, int PW, int WN, int WM, int NT, int MT, int D, bool SWIGLU, int FORM>
int tile_launch(const W8Args& a, int splits) {
  constexpr int BN = WN * NT * 16, BM = WM * MT * 16;
  constexpr size_t ring = (size_t)kStageBytes<BN, BM> * D;
  constexpr size_t sums = epi_bytes<WN * WM, NT, MT, (int)ring>();
  constexpr size_t lds = ring > sums ? ring : sums;
  static_assert(lds <= kMaxLds, "a launch fits the LDS of a CU");
  const int64_t nt = (a.N + BN - 1) / BN, mt = (a.M + BM - 1) / BM;
  if (nt * mt * splits * ((WN * WM + PW) * kWave) > 0xffffffffLL) return set_error(FD_EUNSUPPORTED, "too many tiles");
  auto kernel = w8a8_tile_kernel<T, PW, WN, WM, NT, MT, D, SWIGLU, FORM>;
  if (!allow_lds(kernel, lds)) return set_error(FD_ELAUNCH, "cannot raise the LDS limit to %zu bytes", lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(nt * mt * splits)), dim3((WN * WM + PW) * kWave), lds, a.st,
                     static_cast<T*>(a.y), a.scratch, a.x, a.w, a.M, a.N, a.K, a.sxm, a.swn, a.sym, a.syn, a.e, (int)mt,
                     splits);
  return FD_OK;
}

// The forms of a tile launch: output columns (weight rows) and activation rows of a tile, and the microseconds that
// a stage takes with a workgroup on every CU and a round of them besides (its start, its output). Fitted to products
// of 64 to 8192 rows, 1024 to 28672 columns and K of 512 to 14336 whose time was measured in every form.
struct TileForm {
  int bn, bm;
  float stage, round;
};
enum { T_256 = 0, T_256x128, T_128, T_64x128, T_64, T_128x32, T_FORMS };
constexpr TileForm kTiles[T_FORMS] = {{256, 256, 1.40f, 9.f}, {256, 128, 0.80f, 6.f}, {128, 128, 0.58f, 5.f},
                                      {64, 128, 0.37f, 5.f},  {64, 64, 0.29f, 4.5f},  {128, 32, 0.33f, 4.f}};

struct TilePlan {
  int form, splits;
};

// The form and the K splits (as many as give every CU one workgroup, each with at least six stages) that take the
// least time by that table. Adding the splits' sums is a launch, and their floats go to memory and back.
TilePlan tile_plan(int64_t M, int64_t N, int64_t K) {
  const int64_t stages = (K + kStep - 1) / kStep, cus = device_cus();
  TilePlan best{T_128, 1};
  float least = INFINITY;
  for (int f = 0; f < T_FORMS; ++f) {
    const TileForm& t = kTiles[f];
    const int64_t tiles = ((N + t.bn - 1) / t.bn) * ((M + t.bm - 1) / t.bm);
    int64_t most = cus / (tiles < cus ? tiles : cus);
    if (most > stages / 6) most = stages / 6;
    for (int64_t s = 1; s == 1 || s <= most; ++s) {
      const int64_t rounds = (tiles * s + cus - 1) / cus;
      const float sum = s > 1 ? 4.f + (float)(s * M * N) * 8e-6f / 4.f : 0.f;  // 4 TB/s there and back
      const float us = (float)rounds * ((float)((stages + s - 1) / s) * t.stage + t.round) + sum;
      if (us < least) {
        least = us;
        best = TilePlan{f, (int)s};
      }
    }
  }
  return best;
}

template <typename T, bool SWIGLU, int FORM>
int pick_tile(const W8Args& a, TilePlan p) {
  switch (p.form) {
    case T_256: return tile_launch<T, 0, 4, 2, 4, 8, 2, SWIGLU, FORM>(a, p.splits);
    case T_256x128: return tile_launch<T, 4, 4, 2, 4, 4, 3, SWIGLU, FORM>(a, p.splits);
    case T_128: return tile_launch<T, 0, 2, 4, 4, 2, 4, SWIGLU, FORM>(a, p.splits);
    case T_64x128: return tile_launch<T, 0, 2, 4, 2, 2, 4, SWIGLU, FORM>(a, p.splits);
    case T_64: return tile_launch<T, 4, 2, 2, 2, 2, 4, SWIGLU, FORM>(a, p.splits);
    default: return tile_launch<T, 0, 4, 1, 2, 2, 4, SWIGLU, FORM>(a, p.splits);
  }
}

template <typename T, bool SWIGLU>
int tiles(const W8Args& a, TilePlan p) {
  if (p.splits == 1) return pick_tile<T, SWIGLU, W8_OUT>(a, p);
  const int rc = pick_tile<T, SWIGLU, W8_PART>(a, p);
  if (rc != FD_OK) return rc;
  const int quads = ((SWIGLU ? a.N / 2 : a.N) + 3) / 4;
  const uint32_t total = (uint32_t)a.M * (uint32_t)quads;  // splits > 1: few tiles, so M * N is small
  hipLaunchKernelGGL((w8a8_sum_kernel<T, SWIGLU>), dim3((total + 255) / 256), dim3(256), 0, a.st, static_cast<T*>(a.y),
                     a.scratch, a.M, a.N, p.splits, a.sym, a.syn, a.e, FastDiv((uint32_t)quads), total);
  return FD_OK;
}

// K below one 16-byte piece, none included: a thread per output, and as many more as the grid leaves it.
template <typename T, bool SWIGLU>
__global__ __launch_bounds__(256) void w8a8_short_kernel(T* y, const uint8_t* x, const uint8_t* w, int M, int N, int K,
                                                         int64_t sxm, int64_t swn, int64_t sym, int64_t syn, W8Epi e,
                                                         int64_t total) {
  const int cols = SWIGLU ? N / 2 : N;
  for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < total; v += (int64_t)gridDim.x * 256) {
    const int m = (int)(v / cols), c = (int)(v - (int64_t)m * cols);
    float a = 0.f, u = 0.f;
    for (int k = 0; k < K; ++k) {
      const float xv = __builtin_amdgcn_cvt_f32_fp8(x[m * sxm + k], 0);
      a += xv * __builtin_amdgcn_cvt_f32_fp8(w[c * swn + k], 0);
      if constexpr (SWIGLU) u += xv * __builtin_amdgcn_cvt_f32_fp8(w[(c + (int64_t)cols) * swn + k], 0);
    }
    y[m * sym + c * syn] = from_f32<T>(w8_out<SWIGLU>(e, a, u, m, c, cols));
  }
}

template <typename T, bool SWIGLU>
int short_launch(const W8Args& a) {
  const int64_t total = (int64_t)a.M * (SWIGLU ? a.N / 2 : a.N), most = 1 << 20;
  const int64_t blocks = (total + 255) / 256 < most ? (total + 255) / 256 : most;
  hipLaunchKernelGGL((w8a8_short_kernel<T, SWIGLU>), dim3((unsigned)blocks), dim3(256), 0, a.st, static_cast<T*>(a.y),
                     a.x, a.w, a.M, a.N, a.K, a.sxm, a.swn, a.sym, a.syn, a.e, total);
  return FD_OK;
}

// The rows of both operands, at any address, to rows of K rounded up to 16 bytes, dense and padded with zeros, the
// activations' first: a thread per 16 bytes (777 x 2051 and 5003 x 2051: 6 us, where tiles loaded through registers
// from rows off alignment took 14 more than aligned ones).
__global__ __launch_bounds__(256) void w8a8_align_kernel(u32x4* to, const uint8_t* x, const uint8_t* w, uint32_t M,
                                                         int64_t sxm, int64_t swn, int K, FastDiv pieces,
                                                         uint32_t total) {
  const uint32_t v = blockIdx.x * 256 + threadIdx.x;
  if (v >= total) return;
  uint32_t piece;
  const uint32_t row = pieces.divmod(v, piece);
  to[v] = load16_end(row < M ? x + row * sxm : w + (row - M) * swn, (int)piece * 16, K);
}

// Copies the operands' rows into the scratch of `a`, which then starts behind them.
int align_rows(W8Args& a) {
  const int64_t pieces = ((int64_t)a.K + 15) / 16, total = ((int64_t)a.M + a.N) * pieces;
  if (pieces * 16 >= kMostStride || total > 0xffffff00LL) return set_error(FD_EUNSUPPORTED, "too large to align");
  if (a.scratch_bytes < total * 16) return set_error(FD_EUNSUPPORTED, "rows off 16-byte alignment need scratch");
  uint8_t* const to = reinterpret_cast<uint8_t*>(a.scratch);
  hipLaunchKernelGGL(w8a8_align_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, a.st,
                     reinterpret_cast<u32x4*>(to), a.x, a.w, (uint32_t)a.M, a.sxm, a.swn, a.K,
                     FastDiv((uint32_t)pieces), (uint32_t)total);
  a.K = (int)(pieces * 16);
  a.sxm = a.swn = a.K;
  a.x = to;
  a.w = to + (int64_t)a.M * a.K;
  a.scratch += total * 4;
  a.scratch_bytes -= total * 16;
  return FD_OK;
}

template <typename T, bool SWIGLU>
int product(const W8Args& a) {
  if (a.K < 16) return short_launch<T, SWIGLU>(a);
  if (a.M == 1) {
    if (a.K > kMostIndex - (1 << 14)) return set_error(FD_EUNSUPPORTED, "too large");
    return w8_one_launch(a);
  }
  if (w8_few_fits(a.M, a.K)) return w8_few_launch(a);
  TilePlan p = tile_plan(a.M, a.N, a.K);
  while (p.splits > 1 && a.scratch_bytes < (int64_t)p.splits * a.M * a.N * 4) --p.splits;
  return tiles<T, SWIGLU>(a, p);
}

}  // namespace
}  // namespace fd

using namespace fd;

extern "C" int fd_linear_w8a8_scratch(int64_t M, int64_t N, int64_t K, int aligned, int64_t* bytes) {
  if (M < 0 || N < 0 || K < 0) return set_error(FD_EINVAL, "negative size");
  if (!bytes) return set_error(FD_EINVAL, "null pointer argument");
  *bytes = 0;
  if (M <= 1 || N == 0 || K < 16 || M > kMostIndex || N > kMostIndex || K > kMostIndex) return FD_OK;
  const int64_t Kp = (K + 15) / 16 * 16;
  if (!aligned || K != Kp) *bytes = (M + N) * Kp;
  if (w8_few_fits(M, Kp)) return FD_OK;
  const int s = tile_plan(M, N, Kp).splits;
  if (s > 1) *bytes += (int64_t)s * M * N * 4;
  return FD_OK;
}

extern "C" int fd_linear_w8a8_form(int64_t M, int64_t N, int64_t K, int* form) {
  if (M < 0 || N < 0 || K < 0) return set_error(FD_EINVAL, "negative size");
  if (!form) return set_error(FD_EINVAL, "null pointer argument");
  for (int i = 0; i < 4; ++i) form[i] = 0;
  if (M == 0 || N == 0 || M > kMostIndex || N > kMostIndex || K > kMostIndex) return FD_OK;
  if (K < 16) {
    form[0] = FD_W8A8_SHORT;
  } else if (M == 1) {
    form[0] = FD_W8A8_ONE;
  } else {
    const int64_t Kp = (K + 15) / 16 * 16;
    if (w8_few_fits(M, Kp)) {
      form[0] = FD_W8A8_FEW;
      w8_few_form(M, Kp, &form[1], &form[2]);
    } else {
      const TilePlan p = tile_plan(M, N, Kp);
      form[0] = FD_W8A8_TILES;
      form[1] = kTiles[p.form].bn;
      form[2] = kTiles[p.form].bm;
      form[3] = p.splits;
    }
  }
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
  const int64_t cols = swiglu ? N / 2 : N;
  if (rows_meet(fd_rows{1, 1, M, 0, 0, sym, syn, cols}))
    return set_error(FD_EINVAL, "y's elements must not share memory");
  // tiles are stored while other workgroups still read their operands
  const int64_t ny = span_bytes(M, cols, sym, syn, 2);
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
  // The DMAs take 16-byte pieces, and their 32-bit offsets reach over a tile's rows: other rows are copied first.
  auto fits = [&](const void* p, int64_t rows, int64_t stride) {
    return K % 16 == 0 && aligned16(p) && (rows == 1 || (stride % 16 == 0 && stride < kMostStride));
  };
  if (K >= 16 && M > 1 && !(fits(x8, M, sxm) && fits(w8, N, swn)) && align_rows(a) != FD_OK) return FD_EUNSUPPORTED;
  const int rc = act_dtype == FD_F16 ? (swiglu ? product<f16, true>(a) : product<f16, false>(a))
                                     : (swiglu ? product<bf16, true>(a) : product<bf16, false>(a));
  if (rc != FD_OK) return rc;
  return check_launch();
}
