// Products with E2M1 weights for few activation rows (2 to 32, where fp4_few_wins says so): the weights stream through LDS once, the activations
// stay in registers (fd_fp4.h has the mathematics).
//
// A workgroup of eight waves, one to a CU, owns a run of outputs and walks them in tiles of 16 weight rows (SWIGLU: 8 gate
// rows and their 8 up rows). K is split over the waves: wave w takes the steps w, w + 8, ... of 256 k, so that the workgroup
// reads 1 KiB of a weight row at a time, and keeps S steps' activations, the B operands, in registers for all tiles; a
// longer K takes several such phases. Each wave streams its codes by DMA (global_load_lds_dwordx4, nontemporal) into a ring
// of D slots of its own, D - 1 units (one step of one tile, 2 KiB) ahead, across tiles and phases and without a barrier.
// The scales of all of the workgroup's rows are in LDS before. After a tile the waves' sums meet in LDS: one barrier a
// tile, behind which one wave adds them, in wave order, while the others go on. The outputs leave after the last tile, so
// that no load or store of the epilogue stands in a wave's queue of DMAs.
//
// The run of a workgroup is N / workgroups rows, to the row; a last tile shorter than 16 rows reads its last row again in
// the lanes past it.
//
// Bound by a launch's start and end, the activations' and the scales' way into registers and LDS in front of the stream,
// and then by the stream. Traced medians: 13 x 28672 x 4096 SWIGLU float16 20.6 us (3.0 TB/s of weights), bfloat16 18.3;
// 13 x 6144 x 4096 11.7 and 10.0; 32 x 4096 x 4096 15.6 and 13.2. With five slots in the ring and parts of the work left
// out, the first took 22.3, without activations 21.4, without scales 19.2, without either 18.7, the units alone, nothing
// multiplied, 19.6. A long K leaves more before the stream (13 x 4096 x 14336 bfloat16 23.8: without activations 18.4, scales
// 20.5, either 16.1, units alone 12.1) and goes to the tiles. Activations loaded 64 bytes of a row at a time and exchanged
// between lane groups took as long, and loading them and the scales before the first units longer (22.4 us of the first):
// the stream then starts later.
//
// Slot layout: 16 rows of 8 pieces of 16 bytes, piece c at c ^ (row mod 8).
#include "fd_fp4.h"

namespace fd {

constexpr int kF4Waves = 8;
constexpr int kF4Step = 256;   // k of a unit
constexpr int kF4Tiles = 16;   // tiles of a workgroup at most
constexpr int kF4Ring = 4;     // slots of a wave (4, 5, 6: 13 x 28672 x 4096 SwiGLU float16 20.2, 20.7, 21.2 us captured)

// Bytes of a scale row in LDS: whole words, and an odd number of them, so that 16 rows' bytes lie in different banks.
__host__ __device__ __forceinline__ int f4_scale_pitch(int pieces) { return (((pieces + 7) / 8 * 8) / 4 | 1) * 4; }

template <int MF>
constexpr size_t f4_fixed_lds() {
  return (size_t)kF4Waves * kF4Ring * 2048 + (size_t)2 * kF4Waves * MF * 1024;
}

// TAIL: whether K ends inside a piece. (Asked in the loop it costs 13 x 4096 x 4096 bfloat16 0.4 us of 8.4.)
template <typename T, int MF, int S, bool SWIGLU, bool TAIL>
__global__ __launch_bounds__(kF4Waves * kWave) void fp4_few_kernel(T* y, const T* x, const uint8_t* w, const uint8_t* ws,
                                                                   int M, int N, int K, int64_t sxm, int64_t swn,
                                                                   int64_t ssn, int64_t sym, int64_t syn, Fp4Epi e,
                                                                   int per, int longer, int max_tiles) {
  constexpr int NW = kF4Waves, D = kF4Ring, Q = SWIGLU ? 8 : 16;  // outputs of a tile
  constexpr int H = std::is_same<T, f16>::value ? 2 : 1;          // parts of an activation
  extern __shared__ __align__(16) u32x4 f4_smem[];
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane & 15, g = lane >> 4;
  const int half = N / 2;
  // `per` outputs a workgroup, one more in the first `longer`
  const int b = (int)blockIdx.x, o0 = b * per + (b < longer ? b : longer), o1 = o0 + per + (b < longer ? 1 : 0);
  const int tiles = (o1 - o0 + Q - 1) / Q;
  const int pieces = (K + kGroupK - 1) / kGroupK, steps = (pieces + 7) / 8;
  const int sn = (steps - wave + NW - 1) / NW;            // this wave's steps of a tile
  const int phases = ((steps + NW - 1) / NW + S - 1) / S;  // the same in every wave
  const int units = tiles * sn;

  u32x4* const ring = f4_smem + wave * (D * 128);
  const unsigned ring0 = lds_addr(ring);
  f32x4* const parts = reinterpret_cast<f32x4*>(f4_smem + NW * D * 128);  // [2][NW][MF][64]
  f32x4* const done = parts + 2 * NW * MF * kWave;                        // [tiles][MF][64]
  uint8_t* const scales = reinterpret_cast<uint8_t*>(done + max_tiles * MF * kWave);
  const int pitch = f4_scale_pitch(pieces);

  // weight row at row t of tile `it` (past the last: the last again)
  auto wrow = [&](int it, int t) -> int64_t {
    const int q = it * Q + (SWIGLU ? t & 7 : t);
    const int o = o0 + q < o1 ? o0 + q : o1 - 1;
    return o + (int64_t)(SWIGLU && t >= 8 ? half : 0);
  };
  // a unit's DMA: two instructions of 8 rows x 128 bytes
  int it = 0, is = 0, ip = 0;  // the next unit to issue: tile, step of the phase, phase
  auto issue = [&](int slot) {
    const int first = ((ip * S + is) * NW + wave) * 8;  // its first piece
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = i * 8 + lane / 8, c = first + ((lane & 7) ^ (t & 7));
      dma16_ptr(w + wrow(it, t) * swn + (int64_t)(c < pieces ? c : 0) * 16, ring0 + (unsigned)(slot * 2048 + i * 1024));
    }
    const int left = sn - ip * S, here = left < S ? left : S;
    if (++is == here) {
      is = 0;
      if (++it == tiles) {
        it = 0;
        ++ip;
      }
    }
  };
  for (int u = 0; u < (units < D - 1 ? units : D - 1); ++u) issue(u);

  // all rows' scales; past the last piece 2^0, times activations that are zero
  {
    typedef uint32_t u1 __attribute__((aligned(1)));
    const int words = pitch / 4;
    for (int c = lane; c < pieces / 4; c += kWave) {  // a wave takes every eighth row, eight of them on the way at once
      for (int row0 = wave; row0 < tiles * 16; row0 += 8 * NW) {
        uint32_t v[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const int row = row0 + n * NW < tiles * 16 ? row0 + n * NW : row0;
          const uint8_t* p = ws + wrow(row >> 4, row & 15) * ssn;
          v[n] = *reinterpret_cast<const u1*>(p + c * 4);
        }
#pragma unroll
        for (int n = 0; n < 8; ++n)
          if (row0 + n * NW < tiles * 16) reinterpret_cast<uint32_t*>(scales)[(row0 + n * NW) * words + c] = v[n];
      }
    }
    // the words that the pieces end in, or that lie behind them, byte by byte
    const int whole = pieces / 4;
    for (int i = tid; i < tiles * 16 * (words - whole); i += NW * kWave) {
      const int row = i / (words - whole), c = whole + i - row * (words - whole);
      const uint8_t* p = ws + wrow(row >> 4, row & 15) * ssn;
      uint32_t v = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) v |= (c * 4 + j < pieces ? (uint32_t)p[c * 4 + j] : 127u) << (8 * j);
      reinterpret_cast<uint32_t*>(scales)[row * words + c] = v;
    }
  }

  const int c0 = r * 8 + (g ^ (r & 7)), c1 = r * 8 + ((4 + g) ^ (r & 7));
  int u = 0, slot = 0;
  for (int ph = 0; ph < phases; ++ph) {
    // this wave's activations of the phase: step s, half of it, four operands of 8 k; float16's two parts
    bf16x8 xb[MF][H][S][2][4];
#pragma unroll
    for (int f = 0; f < MF; ++f) {
      const int m = f * 16 + r;
      const T* p = x + (int64_t)(m < M ? m : M - 1) * sxm;
#pragma unroll
      for (int s = 0; s < S; ++s) {
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const int k0 = ((((ph * S + s) * NW + wave) * 8) + a * 4 + g) * kGroupK;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int k = k0 + j * 8;
            typename Vec8<T>::type v;
            if (k + 8 <= K) {
              typedef typename Vec8<T>::type any __attribute__((aligned(2)));
              v = *reinterpret_cast<const any*>(p + k);
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = k + i < K ? p[k + i] : (T)0.f;
            }
            if constexpr (H == 2) {
              split_f16(v, xb[f][0][s][a][j], xb[f][H - 1][s][a][j]);
            } else {
              xb[f][0][s][a][j] = v;
            }
          }
        }
      }
    }
    // all of it has landed here (the first units' codes with it), so that no wait of the compiler's for an activation
    // stands in the loop
    __builtin_amdgcn_s_waitcnt(0x0f70);
    if (ph == 0) lds_barrier();  // the scales are there

    const int here = sn - ph * S;  // this wave's steps of the phase, S at most
    for (int t = 0; t < tiles; ++t) {
      f32x4 acc[MF][2][H];  // chains of sums: a step's halves, an activation's parts
#pragma unroll
      for (int f = 0; f < MF; ++f)
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int h = 0; h < H; ++h) acc[f][a][h] = f32x4{0.f, 0.f, 0.f, 0.f};
      const uint8_t* const sp = scales + (t * 16 + r) * pitch + (ph * S * NW + wave) * 8 + g;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (s < here) {
          const float f0 = e8m0_operand(sp[s * NW * 8]), f1 = e8m0_operand(sp[s * NW * 8 + 4]);
          if (u + D - 1 <= units)
            wait_vm<2 * (D - 2)>();
          else
            wait_vm<0>();
          const u32x4* p = ring + slot * 128;
          u32x4 a0 = p[c0], a1 = p[c1];
          if constexpr (TAIL) {
            const int first = ((ph * S + s) * NW + wave) * 8 + g;  // the lane's pieces: this one and the fourth behind it
            if (first == pieces - 1) a0 = fp4_tail(a0, K % kGroupK);
            if (first + 4 == pieces - 1) a1 = fp4_tail(a1, K % kGroupK);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int a = 0; a < 2; ++a) {
              const bf16x8 wv = fp4_to_bf16(a ? a1[j] : a0[j], a ? f1 : f0);
#pragma unroll
              for (int f = 0; f < MF; ++f)
#pragma unroll
                for (int h = 0; h < H; ++h) acc[f][a][h] = mfma16(wv, xb[f][h][s][a][j], acc[f][a][h]);
            }
          }
          // the unit before this one has been read: its slot takes the next
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          if (u + D - 1 < units) issue(slot == 0 ? D - 1 : slot - 1);
          ++u;
          slot = slot == D - 1 ? 0 : slot + 1;
        }
      }
      const int at = (ph * tiles + t) & 1;
      f32x4* pp = parts + (at * NW + wave) * MF * kWave + lane;
#pragma unroll
      for (int f = 0; f < MF; ++f) {
        f32x4 v = acc[f][0][0] + acc[f][1][0];
        if constexpr (H == 2) v += acc[f][0][H - 1] + acc[f][1][H - 1];
        pp[f * kWave] = v;
      }
      lds_barrier();
      if (wave == (t & (NW - 1))) {
        const f32x4* q = parts + at * NW * MF * kWave + lane;
#pragma unroll
        for (int f = 0; f < MF; ++f) {
          f32x4 v = q[f * kWave];
#pragma unroll
          for (int i = 1; i < NW; ++i) v += q[(i * MF + f) * kWave];
          f32x4* const to = done + (t * MF + f) * kWave + lane;  // (one wave's in every phase)
          *to = ph ? *to + v : v;
        }
      }
    }
  }
  lds_barrier();
  // sum of weight row `row` of tile t and activation row m
  auto sum = [&](int t, int row, int m) {
    const int lane_of = (t * MF + m / 16) * kWave + (row >> 2) * 16 + (m & 15);
    return reinterpret_cast<const float*>(done)[lane_of * 4 + (row & 3)];
  };
  const int run = o1 - o0;
  for (int i = tid; i < run * M; i += NW * kWave) {
    const int m = i / run, q = i - m * run, t = q / Q, o = o0 + q;
    const float a = sum(t, q % Q, m), up = SWIGLU ? sum(t, 8 + q % Q, m) : 0.f;
    y[(int64_t)m * sym + (int64_t)o * syn] = from_f32<T>(fp4_out<SWIGLU>(e, a, up, m, o, half));
  }
}

namespace {

// Outputs of a workgroup whose sums and scales its LDS holds; 0: none.
template <int MF>
int f4_most_outputs(int64_t K, bool swiglu) {
  const int64_t pieces = (K + kGroupK - 1) / kGroupK;
  if (pieces > 1 << 16) return 0;
  const int64_t tile = (int64_t)MF * 1024 + 16 * f4_scale_pitch((int)pieces);
  int64_t tiles = ((int64_t)kMaxLds - (int64_t)f4_fixed_lds<MF>()) / tile;
  if (tiles > kF4Tiles) tiles = kF4Tiles;
  return (int)tiles * (swiglu ? 8 : 16);
}

template <typename T, int MF, int S, bool SWIGLU, bool TAIL>
int f4_few_tail(const Fp4Args& a) {
  const int cols = SWIGLU ? a.N / 2 : a.N, most = f4_most_outputs<MF>(a.K, SWIGLU), Q = SWIGLU ? 8 : 16;
  int grid = device_cus();
  if (grid > (cols + 3) / 4) grid = (cols + 3) / 4;
  if ((int64_t)grid * most < cols) grid = (cols + most - 1) / most;
  const int tiles = (cols / grid + (cols % grid ? 1 : 0) + Q - 1) / Q, pieces = (a.K + kGroupK - 1) / kGroupK;
  const size_t lds = f4_fixed_lds<MF>() + (size_t)tiles * (MF * 1024 + 16 * f4_scale_pitch(pieces));
  auto kernel = fp4_few_kernel<T, MF, S, SWIGLU, TAIL>;
  if (!allow_lds(kernel, lds)) return set_error(FD_ELAUNCH, "cannot raise the LDS limit to %zu bytes", lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(kF4Waves * kWave), lds, a.st, static_cast<T*>(a.y),
                     static_cast<const T*>(a.x), a.w, a.ws, a.M, a.N, a.K, a.sxm, a.swn, a.ssn, a.sym, a.syn, a.e,
                     cols / grid, cols % grid, tiles);
  return FD_OK;
}

template <typename T, int MF, int S, bool SWIGLU>
int f4_few_go(const Fp4Args& a) {
  return a.K % kGroupK ? f4_few_tail<T, MF, S, SWIGLU, true>(a) : f4_few_tail<T, MF, S, SWIGLU, false>(a);
}

// Steps of K that a wave keeps the activations of: 32 registers each, twice that for float16 and for a second 16 rows.
template <typename T, bool SWIGLU>
int f4_few_pick(const Fp4Args& a) {
  constexpr bool F16 = std::is_same<T, f16>::value;
  const int steps = (a.K + kF4Step * kF4Waves - 1) / (kF4Step * kF4Waves);  // of a wave
  if (a.M <= 16) {
    if (steps <= 1) return f4_few_go<T, 1, 1, SWIGLU>(a);
    if (steps <= 2 || F16) return f4_few_go<T, 1, 2, SWIGLU>(a);
    return f4_few_go<T, 1, F16 ? 2 : 4, SWIGLU>(a);
  }
  if (steps <= 1 || F16) return f4_few_go<T, 2, 1, SWIGLU>(a);
  return f4_few_go<T, 2, F16 ? 1 : 2, SWIGLU>(a);
}

}  // namespace

bool fp4_few_fits(int64_t M, int64_t K, bool swiglu) {
  return K > 0 && ((M <= 16 && f4_most_outputs<1>(K, swiglu) > 0) || (M <= 32 && f4_most_outputs<2>(K, swiglu) > 0));
}

// Every workgroup brings all of the activations to its registers, in phases where K is long, in 2-byte loads where rows lie
// at odd elements; tiles bring them once a tile. Captured, weights from HBM, here and in tiles (us):
//
//   rows x N x K                      here    tiles        rows x N x K                      here    tiles
//   32 x 4096 x 4096     bfloat16     13.2    14.5         32 x 4096 x 4096     float16      15.5    18.5
//   32 x 4096 x 5120     bfloat16     21.8    18.7         32 x 2048 x 8192     float16      25.2    21.2
//   16 x 2048 x 8192     bfloat16     13.3    14.8         16 x 8192 x 8192     float16      20.4    23.4
//   4 x 4096 x 14336     bfloat16     17.7    20.0         4 x 4096 x 11008     float16      22.5    20.8
//   13 x 4096 x 14336    bfloat16     22.2    20.6         2 x 4096 x 14336     float16      27.6    22.6
//   16 x 28672 x 2051    bfloat16     19.8    22.6         12 x 16384 x 3001    float16      17.6    19.4
//   29 x 5003 x 2051     bfloat16     18      14.5         29 x 5003 x 2051     float16      23.5    16.7
//
// Over 526 products (30 shapes, 2 to 32 rows, both types) the rule's choice takes 0.2 in 100 more than the better of the
// two, 13 in the worst; this kernel always, 10, and twice as long in the worst.
bool fp4_few_wins(int64_t M, int64_t K, int act_dtype) {
  if (K % 2) return K <= 4096 && (M > 16 ? 32 : M) * K <= 49152;
  if (K > (M > 16 ? 4096 : act_dtype == FD_F16 ? 8192 : 16384)) return false;
  return K <= 8192 || M * K <= 65536;
}

int fp4_few_launch(const Fp4Args& a) {
  if (a.act_dtype == FD_F16) return a.swiglu ? f4_few_pick<f16, true>(a) : f4_few_pick<f16, false>(a);
  return a.swiglu ? f4_few_pick<bf16, true>(a) : f4_few_pick<bf16, false>(a);
}

}  // namespace fd
