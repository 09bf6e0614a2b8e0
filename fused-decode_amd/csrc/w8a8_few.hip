// Products of E4M3 activations and weights for few activation rows (2 to 32): the weights
// stream through LDS once, the activations stay in registers (fd_w8a8.h has the mathematics).
//
// A workgroup of eight waves, one to a CU, owns a run of outputs and walks them in tiles of 16
// weight rows (SWIGLU: 8 gate rows and their 8 up rows). K is split over the waves: wave w takes
// the steps w, w + 8, ... of 128 k, so that the workgroup reads 1 KiB of a weight row at a time,
// and keeps its steps' activations, the B operands, in registers for all tiles. Each wave
// streams its weights by DMA (global_load_lds_dwordx4, nontemporal) into a ring of D slots of
// its own, D - 1 units (one step of one tile, 2 KiB) ahead, across tile boundaries and without
// a barrier. After a tile the waves' sums meet in LDS: one barrier a tile, behind which one
// wave adds them, in wave order, while the others go on. The outputs leave after the last
// tile, so that no load or store of the epilogue stands in a wave's queue of DMAs.
//
// The run of a workgroup is N / CUs rows, to the row; a last tile shorter than 16 rows reads
// its last row again in the lanes past it.
//
// Bound by what a CU takes in a clock, weights and activations, and by a launch's start and end:
// 13 x 28672 x 4096 SWIGLU 21.5 us (5.5 TB/s of weights), 16 x 4096 x 14336 17.3, 16 x 6144 x 4096
// 8.8; 17 to 32 rows, two groups of 16: 24 x 6144 x 4096 9.6, 32 x 28672 x 4096 SWIGLU 24.1.
// Activations as the stream's first units, so that nothing waits for all of it, 15.0 against 12.9
// (2 x 4096 x 14336: they take the weights' slots); weights straight into registers, in the operand's
// layout, 20.5 (loads of 64 bytes a row).
//
// Slot layout: 16 rows of 8 chunks of 16 bytes, chunk c at c ^ (row mod 8).
#include "fd_w8a8.h"

namespace fd {

constexpr int kFewWaves = 8;
constexpr int kFewTiles = 16;  // tiles of a workgroup whose sums its LDS holds

template <int MF, int D>
constexpr size_t few_lds() {
  return (size_t)kFewWaves * D * 2048 + (size_t)2 * kFewWaves * MF * 1024 + (size_t)kFewTiles * MF * 1024;
}

template <typename T, int MF, int S, int D, bool SWIGLU>
__global__ __launch_bounds__(kFewWaves * kWave) void w8a8_few_kernel(T* y, const uint8_t* x, const uint8_t* w, int M,
                                                                     int N, int K, int64_t sxm, int64_t swn,
                                                                     int64_t sym, int64_t syn, W8Epi e, int per,
                                                                     int longer) {
  constexpr int NW = kFewWaves, Q = SWIGLU ? 8 : 16;  // outputs of a tile
  extern __shared__ __align__(16) u32x4 w8_smem[];
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane & 15, g = lane >> 4;
  const int half = N / 2;
  // `per` outputs a workgroup, one more in the first `longer`
  const int b = (int)blockIdx.x, o0 = b * per + (b < longer ? b : longer), o1 = o0 + per + (b < longer ? 1 : 0);
  const int tiles = (o1 - o0 + Q - 1) / Q;
  const int steps = (K + kStep - 1) / kStep;
  const int sn = (steps - wave + NW - 1) / NW;  // this wave's steps of a tile
  const int units = tiles * sn;

  u32x4* const ring = w8_smem + wave * (D * 128);
  const unsigned ring0 = lds_addr(ring);
  f32x4* const parts = reinterpret_cast<f32x4*>(w8_smem + NW * D * 128);  // [2][NW][MF][64]
  f32x4* const done = parts + 2 * NW * MF * kWave;                        // [tiles][MF][64]

  // a unit's DMA: two instructions of 8 rows x 128 bytes
  int it = 0, is = 0;  // the next unit to issue
  auto issue = [&](int slot) {
    const int k0 = (is * NW + wave) * kStep;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = i * 8 + lane / 8;
      const int q = it * Q + (SWIGLU ? t & 7 : t);
      const int o = o0 + q < o1 ? o0 + q : o1 - 1;
      const int64_t row = o + (int64_t)(SWIGLU && t >= 8 ? half : 0);
      const int k = k0 + ((lane & 7) ^ (t & 7)) * 16;
      const uint8_t* p = w + row * swn + (k < K ? k : 0);  // past K: the row's start, times zero
      dma16_ptr(p, ring0 + (unsigned)(slot * 2048 + i * 1024));
    }
    if (++is == sn) {
      is = 0;
      ++it;
    }
  };
  for (int u = 0; u < (units < D - 1 ? units : D - 1); ++u) issue(u);

  // this wave's activations: step s, rows r of each 16, the two 16-byte pieces of group g
  u32x4 b0[MF][S], b1[MF][S];
#pragma unroll
  for (int f = 0; f < MF; ++f) {
    const int m = f * 16 + r;
    const uint8_t* p = x + (int64_t)(m < M ? m : M - 1) * sxm;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int k = (s * NW + wave) * kStep + g * 16;
      const u32x4 z = {0u, 0u, 0u, 0u};
      b0[f][s] = k < K ? *reinterpret_cast<const u32x4*>(p + k) : z;
      b1[f][s] = k + 64 < K ? *reinterpret_cast<const u32x4*>(p + k + 64) : z;
    }
  }
  // all of it has landed here (the first units' weights with it), so that no wait of the compiler's
  // for an activation stands in the loop
  __builtin_amdgcn_s_waitcnt(0x0f70);

  const int c0 = r * 8 + (g ^ (r & 7)), c1 = r * 8 + ((4 + g) ^ (r & 7));
  int u = 0, slot = 0;
  for (int t = 0; t < tiles; ++t) {
    f32x4 acc[MF];
#pragma unroll
    for (int f = 0; f < MF; ++f) acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < sn) {
        if (u + D - 1 <= units)
          wait_vm<2 * (D - 2)>();
        else
          wait_vm<0>();
        const u32x4* p = ring + slot * 128;
        const u32x4 a0 = p[c0], a1 = p[c1];
#pragma unroll
        for (int f = 0; f < MF; ++f) acc[f] = mfma_e4m3(a0, a1, b0[f][s], b1[f][s], acc[f]);
        // the unit before this one has been read: its slot takes the next
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (u + D - 1 < units) issue(slot == 0 ? D - 1 : slot - 1);
        ++u;
        slot = slot == D - 1 ? 0 : slot + 1;
      }
    }
    f32x4* pp = parts + ((t & 1) * NW + wave) * MF * kWave + lane;
#pragma unroll
    for (int f = 0; f < MF; ++f) pp[f * kWave] = acc[f];
    lds_barrier();
    if (wave == (t & (NW - 1))) {
      const f32x4* q = parts + (t & 1) * NW * MF * kWave + lane;
#pragma unroll
      for (int f = 0; f < MF; ++f) {
        f32x4 v = q[f * kWave];
#pragma unroll
        for (int i = 1; i < NW; ++i) v += q[(i * MF + f) * kWave];
        done[(t * MF + f) * kWave + lane] = v;
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
    y[(int64_t)m * sym + (int64_t)o * syn] = from_f32<T>(w8_out<SWIGLU>(e, a, up, m, o, half));
  }
}

namespace {

template <typename T, int MF, int S, int D, bool SWIGLU>
int few_go(const W8Args& a) {
  constexpr size_t lds = few_lds<MF, D>();
  static_assert(lds <= kMaxLds, "a launch fits the LDS of a CU");
  const int cols = a.swiglu ? a.N / 2 : a.N, per = kFewTiles * (SWIGLU ? 8 : 16);
  int grid = device_cus();
  if (grid > (cols + 3) / 4) grid = (cols + 3) / 4;
  if ((int64_t)grid * per < cols) grid = (cols + per - 1) / per;
  auto kernel = w8a8_few_kernel<T, MF, S, D, SWIGLU>;
  if (!allow_lds(kernel, lds)) return set_error(FD_ELAUNCH, "cannot raise the LDS limit to %zu bytes", lds);
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(kFewWaves * kWave), lds, a.st, static_cast<T*>(a.y), a.x, a.w,
                     a.M, a.N, a.K, a.sxm, a.swn, a.sym, a.syn, a.e, cols / grid, cols % grid);
  return FD_OK;
}

int few_steps(int64_t K) { return (int)(((K + kStep - 1) / kStep + kFewWaves - 1) / kFewWaves); }  // of a wave

template <typename T, bool SWIGLU>
int few_pick(const W8Args& a) {
  int groups, steps;
  w8_few_form(a.M, a.K, &groups, &steps);
  if (groups == 1) {
    if (steps == 4) return few_go<T, 1, 4, 7, SWIGLU>(a);
    if (steps == 8) return few_go<T, 1, 8, 7, SWIGLU>(a);
    return few_go<T, 1, 16, 7, SWIGLU>(a);
  }
  if (steps == 4) return few_go<T, 2, 4, 6, SWIGLU>(a);
  return few_go<T, 2, 8, 6, SWIGLU>(a);
}

}  // namespace

void w8_few_form(int64_t M, int64_t K, int* groups, int* steps) {
  const int s = few_steps(K);
  *groups = M <= 16 ? 1 : 2;
  *steps = s <= 4 ? 4 : s <= 8 || *groups == 2 ? 8 : 16;
}

// Whether the activations fit the registers.
bool w8_few_fits(int64_t M, int64_t K) { return M <= 16 ? few_steps(K) <= 16 : M <= 32 && few_steps(K) <= 8; }

int w8_few_launch(const W8Args& a) {
  if (a.act_dtype == FD_F16) return a.swiglu ? few_pick<f16, true>(a) : few_pick<f16, false>(a);
  return a.swiglu ? few_pick<bf16, true>(a) : few_pick<bf16, false>(a);
}

}  // namespace fd
