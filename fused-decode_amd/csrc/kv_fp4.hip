// A key/value cache held as OCP E2M1 codes, two a byte, with an E8M0 scale for each group of 32 along the head: the store
// of new tokens, the read of cached ones, and the attention of one or a few new tokens over it.
//
//   store: a group's scale is 2^e, the smallest with max|v| < 7 2^e (e >= -126; 2^0 for zeros, NaN beside an infinity or
//          a NaN); code = nearest E2M1 of v / 2^e, ties to even, 6 at most
//   attention, query row i of a sequence of `length` tokens that its L last are queries of:
//          y = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q . k_t - max),  t <= length - L + i / G
//
// A cache is pages of `page` slots: codes [pages, heads, page, dim / 2], scales [pages, heads, page, dim / 32], keys and
// values alike. A slot's codes start at a multiple of 16 bytes and are 16 bytes for one of scales, so one number, its
// place in units of 16 bytes of codes and of 1 byte of scales, finds all four. Which pages a sequence has says a table,
// or, without one, page b is sequence b's. A page number outside the cache is not followed: its tokens are neither
// stored nor seen.
#include <type_traits>

#include "fd_fp4.h"

namespace fd {

struct KvCache {
  uint8_t *k, *ks, *v, *vs;
  uint32_t pages, heads, page;
  int64_t page_step, head_step;  // between pages and heads, in units of 16 bytes of codes
};
struct KvTable {
  const int32_t* lengths;
  const int32_t* pages;  // null: page b is sequence b's
  int64_t step;          // between sequences
  uint32_t capacity;     // tokens that a sequence's pages hold
};

constexpr uint32_t kNoPlace = 0xffffffffu;

// Place of head 0 of token t < capacity of sequence b, or kNoPlace.
__device__ __forceinline__ uint32_t kv_place(const KvCache& c, const KvTable& tb, const FastDiv& page, uint32_t row16,
                                             uint32_t b, uint32_t t) {
  uint32_t slot;
  const uint32_t at = page.divmod(t, slot);
  const uint32_t id = tb.pages ? (uint32_t)tb.pages[b * tb.step + at] : b;
  return id < c.pages ? (uint32_t)(id * c.page_step) + slot * row16 : kNoPlace;
}

// ------------------------------------------------------------------ store and read

// Eight values a lane, four lanes a group; bound by a launch's start and end (one token: 2.7 us) and by its stores of 4 and 1
// bytes (4 x 2048 tokens of 8 heads of 128: 12.6 us, 3.4 TB/s, keys and values in two halves of the grid).
template <typename T>
__global__ __launch_bounds__(256) void kv_append_kernel(KvCache c, KvTable tb, const T* k, const T* v, int64_t skb,
                                                        int64_t skl, int64_t skh, int64_t svb, int64_t svl, int64_t svh,
                                                        uint32_t L, uint32_t row16, FastDiv lanes, FastDiv heads,
                                                        FastDiv len, FastDiv page, uint32_t half, uint32_t total) {
  const uint32_t idx = blockIdx.x * 256 + threadIdx.x;
  const bool live = idx < total;  // groups are whole: four lanes stay or go together
  const bool value = idx >= half;
  uint32_t e, h, l;
  uint32_t q = lanes.divmod(live ? (value ? idx - half : idx) : 0, e);
  q = heads.divmod(q, h);
  const uint32_t b = len.divmod(q, l);
  const T* p = value ? v + b * svb + l * svl + h * svh : k + b * skb + l * skl + h * skh;
  const typename Vec8<T>::type in = load8_any<T>(p + e * 8);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t m = __builtin_bit_cast(uint32_t, to_f32(in[i])) & 0x7fffffffu;
    top = m > top ? m : top;
  }
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, XlaneDpp<1>::ctrl, 0xf, 0xf, false));
  top = max(top, (uint32_t)__builtin_amdgcn_mov_dpp((int)top, XlaneDpp<2>::ctrl, 0xf, 0xf, false));
  const bool bad = top >= 0x7f800000u;
  // the exponent of max / 4, one more from 1.75 times a power of two on
  int byte = (int)((top + 0x200000u) >> 23) - 2;
  byte = bad ? 255 : top == 0 ? 127 : byte < 1 ? 1 : byte;
  const float scale = __builtin_bit_cast(float, (uint32_t)byte << 23);
  uint32_t code = 0;
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, to_f32(in[0]), to_f32(in[1]), scale, 0);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, to_f32(in[2]), to_f32(in[3]), scale, 1);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, to_f32(in[4]), to_f32(in[5]), scale, 2);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, to_f32(in[6]), to_f32(in[7]), scale, 3);
  const int64_t t = (int64_t)tb.lengths[b] - L + l;
  if (!live || t < 0 || t >= tb.capacity) return;
  const uint32_t at = kv_place(c, tb, page, row16, b, (uint32_t)t);
  if (at == kNoPlace) return;
  const uint64_t place = (uint64_t)at + h * c.head_step;
  *reinterpret_cast<uint32_t*>((value ? c.v : c.k) + place * 16 + e * 4) = bad ? 0u : code;
  if (e % 4 == 0) (value ? c.vs : c.ks)[place + e / 4] = (uint8_t)byte;
}

// Eight values a lane; rows in the order of four tokens, heads, tokens, so that what is read and what is written both
// lie together: 4 x 8192 tokens of 8 heads of 128 in 26.8 us, 6.3 TB/s, four fifths of it writes.
template <typename T>
__global__ __launch_bounds__(256) void kv_read_kernel(T* ko, T* vo, KvCache c, KvTable tb, uint32_t count, uint32_t dim,
                                                      uint32_t row16, FastDiv lanes, FastDiv heads, FastDiv quads,
                                                      FastDiv page, uint32_t first, uint32_t total) {
  const uint32_t idx = blockIdx.x * 256 + threadIdx.x;
  if (idx >= total) return;
  uint32_t e, h, t4;
  uint32_t q = lanes.divmod(idx, e);
  const uint32_t sub = q & 3;
  q = heads.divmod((q >> 2) + first, h);
  const uint32_t b = quads.divmod(q, t4);
  const uint32_t t = t4 * 4 + sub;
  if (t >= count) return;
  const int32_t length = tb.lengths[b];
  uint32_t at = kNoPlace;
  if ((int64_t)t < length && t < tb.capacity) at = kv_place(c, tb, page, row16, b, t);
  uint32_t codes[2] = {0u, 0u}, bytes[2] = {127u, 127u};
  if (at != kNoPlace) {
    const uint64_t place = (uint64_t)at + h * c.head_step;
    codes[0] = *reinterpret_cast<const uint32_t*>(c.k + place * 16 + e * 4);
    codes[1] = *reinterpret_cast<const uint32_t*>(c.v + place * 16 + e * 4);
    bytes[0] = c.ks[place + e / 4];
    bytes[1] = c.vs[place + e / 4];
  }
  const uint64_t to = (((uint64_t)b * count + t) * c.heads + h) * dim + e * 8;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bf16x8 x = fp4_to_bf16(codes[i], e8m0_operand(bytes[i]));
    T* o = (i ? vo : ko) + to;
    if constexpr (std::is_same<T, bf16>::value) {
      store8_nt<T>(o, x);
    } else {
      f16x8 y;
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = (f16)(float)x[j];
      store8_nt<T>(o, y);
    }
  }
}

// ------------------------------------------------------------------ attention

constexpr int kKvTile = 32;     // tokens of a step
constexpr int kKvChunk = 4096;  // tokens whose places a workgroup's LDS holds

// The larger one, NaN beside a NaN.
__device__ __forceinline__ float kv_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

template <int MASK>
__device__ __forceinline__ float xlane_fmax(float v) {
  static_assert(MASK >= 16, "between lane groups");
  const unsigned a = __builtin_bit_cast(unsigned, v);
  const auto r = MASK == 32 ? __builtin_amdgcn_permlane32_swap(a, a, false, false)
                            : __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const unsigned r0 = r[0], r1 = r[1];
  return kv_max(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
}

// N 32-bit words (2, 3, 4, 6 or 8).
template <int N>
struct KvWords {
  uint32_t w[N];
  template <int I>
  __device__ __forceinline__ void four(const uint8_t* p) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(4)));
    const u4 v = *reinterpret_cast<const u4*>(p + I * 4);
    w[I] = v[0], w[I + 1] = v[1], w[I + 2] = v[2], w[I + 3] = v[3];
  }
  template <int I>
  __device__ __forceinline__ void two(const uint8_t* p) {
    typedef uint32_t u2 __attribute__((ext_vector_type(2), aligned(4)));
    const u2 v = *reinterpret_cast<const u2*>(p + I * 4);
    w[I] = v[0], w[I + 1] = v[1];
  }
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (N == 2 || N == 3) two<0>(p);
    if constexpr (N >= 4) four<0>(p);
    if constexpr (N == 3) w[2] = *reinterpret_cast<const uint32_t*>(p + 8);
    if constexpr (N == 6) two<4>(p);
    if constexpr (N == 8) four<4>(p);
  }
};

// B bytes (2, 3, 4, 6 or 8) at a multiple of B as words.
template <int B>
__device__ __forceinline__ void kv_bytes(const uint8_t* p, uint32_t (&w)[(B + 3) / 4]) {
  if constexpr (B == 2) {
    w[0] = *reinterpret_cast<const uint16_t*>(p);
  } else if constexpr (B == 3) {
    w[0] = p[0] | (uint32_t)p[1] << 8 | (uint32_t)p[2] << 16;
  } else if constexpr (B == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (B == 6) {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
    w[0] = q[0] | (uint32_t)q[1] << 16;
    w[1] = q[2];
  } else {
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    const u2 v = *reinterpret_cast<const u2*>(p);
    w[0] = v[0];
    w[1] = v[1];
  }
}

// Byte B of words.
template <int B>
__device__ __forceinline__ uint32_t kv_pair(const uint32_t* w, float scale) {
  return fp4_pair<B % 4>(w[B / 4], scale);
}

struct KvQuery {
  int64_t sb, sl, sh;  // strides of q
  uint32_t L, Hq, G, rows;  // rows: L * G
  float scale;              // its magnitude times log2 e
  bool flip;                // whether it is negative: q's sign takes it
};

// Tokens of a step in one run of slots, or each at a place of its own (pages that end inside a step).
enum KvMode { KV_RUN = 0, KV_PLACES = 1 };

// One step's keys and values of a lane, as they lie in memory.
//
// Keys are the A operand of q . k: lane (r, g) has quarter g of tokens r and 16 + r. Values, the other way round, are the A
// operand of the sum over tokens: lane (r, g) has the sixteenth r of tokens 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3,
// the tokens whose scores it gets.
template <int D, int MODE>
struct KvStep {
  static constexpr int KW = D / 32;                                                     // words of a quarter
  static constexpr int KS = D == 64 || D == 128 ? 1 : D == 256 ? 2 : D / 32;            // scales of it
  static constexpr int VB = D / 32, VW = (VB + 3) / 4;                                  // bytes of a sixteenth
  static constexpr int VS = D == 96 || D == 192 ? 2 : 1;                                // scales of it
  // a run's four tokens' scales come together where they are whole words (2 or 4 bytes a token)
  static constexpr bool PACKED = MODE == KV_RUN && (D == 64 || D == 128);
  KvWords<KW> k[2];
  uint32_t ks[2][KS];
  uint32_t v[8][VW];
  uint32_t vs[PACKED ? 2 : 8][PACKED ? D / 32 : VS];
  uint32_t at[MODE == KV_PLACES ? 8 : 1];  // places of the value's tokens
  uint32_t some;                           // a word of the run's values' scales: the lanes have all of them

  static __device__ __forceinline__ int key_first(int j, int g) {
    return KS == 1 ? g * (D / 4) / 32 : KS == 2 ? 2 * g + j : (g * (D / 4) + 8 * j) / 32;
  }
  __device__ __forceinline__ void key(int s, const uint8_t* codes, const uint8_t* scales, int g) {
    k[s].load(codes);
#pragma unroll
    for (int j = 0; j < KS; ++j) ks[s][j] = scales[key_first(j, g)];
  }
  __device__ __forceinline__ void value(int n, const uint8_t* codes) { kv_bytes<VB>(codes, v[n]); }
  __device__ __forceinline__ void value_scale(int n, const uint8_t* scales, int r) {
    if constexpr (!PACKED) {
      vs[n][0] = scales[r * (D / 16) / 32];
      if constexpr (VS == 2) vs[n][1] = scales[(r * (D / 16) + D / 16 - 1) / 32];
    }
  }
  // from place `at` on, a run
  __device__ __forceinline__ void load_run(const KvCache& c, uint64_t at, int r, int g) {
    const uint8_t *kp = c.k + at * 16, *ksp = c.ks + at, *vp = c.v + at * 16, *vsp = c.vs + at;
    const unsigned ko = r * (D / 2) + g * (D / 8), so = r * (D / 32), vo = 4 * g * (D / 2) + r * VB,
                   wo = 4 * g * (D / 32);
    typedef uint32_t u1 __attribute__((aligned(1)));
    some = *reinterpret_cast<const u1*>(vsp + (r + 16 * g) % (D / 4) * 4);
#pragma unroll
    for (int s = 0; s < 2; ++s) key(s, kp + (ko + s * 8 * D), ksp + (so + s * (D / 2)), g);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if constexpr (PACKED) {
        typedef uint32_t uw __attribute__((ext_vector_type(D / 32), aligned(1)));
        const uw w = *reinterpret_cast<const uw*>(vsp + (wo + s * (D / 2)));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) vs[s][i] = w[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        value(s * 4 + i, vp + (vo + s * 8 * D + i * (D / 2)));
        value_scale(s * 4 + i, vsp + (wo + s * (D / 2) + i * (D / 32)), r);
      }
    }
  }
  // 32 places, kNoPlace where there is no token
  __device__ __forceinline__ void load_places(const KvCache& c, uint64_t head, const uint32_t* places, int r, int g) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint32_t a = places[s * 16 + r];
      const uint64_t b = head + (a == kNoPlace ? 0u : a);
      key(s, c.k + b * 16 + g * (D / 8), c.ks + b, g);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const u32x4 a = *reinterpret_cast<const u32x4*>(places + s * 16 + g * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = s * 4 + i;
        if constexpr (MODE == KV_PLACES) at[n] = a[i];
        const uint64_t b = head + (a[i] == kNoPlace ? 0u : a[i]);
        value(n, c.v + b * 16 + r * VB);
        value_scale(n, c.vs + b, r);
      }
    }
  }
  // the scale of the key words' j-th
  __device__ __forceinline__ float key_scale(int s, int j) const {
    return e8m0_operand(ks[s][KS == 1 ? 0 : KS == 2 ? j / 4 : j]);
  }
  // Of byte B of a token's values, as the conversion takes it: it reads the exponent alone, so a word that is turned
  // until the byte stands there will do. `turn`: by how much, for this lane's byte of an even word.
  template <int B>
  __device__ __forceinline__ float value_scale_of(int n, int r, uint32_t turn) const {
    if constexpr (PACKED) {
      const uint32_t w = vs[n / 4][D == 128 ? n % 4 : n % 4 / 2];
      return __builtin_bit_cast(float, __builtin_amdgcn_alignbit(w, w, D == 64 && n % 2 ? turn + 16 : turn));
    } else {
      const uint32_t e = VS == 1 || (r * (D / 16) + 2 * B) / 32 == r * (D / 16) / 32 ? vs[n][0] : vs[n][VS - 1];
      return e8m0_operand(e);
    }
  }
  // Scales of 1 for tokens that nobody sees (from `seen` on, or without a place): what lies there may be no number.
  __device__ __forceinline__ void drop_unseen(int t0, int seen, int g) {
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      bool none = t0 + (n / 4) * 16 + g * 4 + n % 4 >= seen;
      if constexpr (MODE == KV_PLACES) none = at[n] == kNoPlace;
      if constexpr (PACKED) {
        uint32_t& w = vs[n / 4][D == 128 ? n % 4 : n % 4 / 2];
        const uint32_t keep = D == 128 ? 0u : n % 2 ? 0x0000ffffu : 0xffff0000u;
        w = none ? (w & keep) | (0x7f7f7f7fu & ~keep) : w;
      } else {
#pragma unroll
        for (int j = 0; j < VS; ++j) vs[n][j] = none ? 127u : vs[n][j];
      }
    }
  }
  // Whether a scale of 2^65 or more is among the step's (from 2^126 on codes leave bfloat16's range), of which the lanes
  // have all; MASK: behind drop_unseen.
  template <bool MASK>
  __device__ __forceinline__ bool any_big() const {
    if constexpr (MODE == KV_RUN && !MASK) return (some & some << 1 & 0x80808080u) != 0;
    uint32_t big = 0;
    if constexpr (PACKED) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) big |= vs[s][i] & vs[s][i] << 1 & 0x80808080u;
    } else {
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int j = 0; j < VS; ++j) big |= vs[n][j] & vs[n][j] << 1 & 0x80u;
    }
    return big != 0;
  }
};

template <int D, int B, typename F>
__device__ __forceinline__ void kv_each_byte(F&& f) {
  if constexpr (B < D / 32) {
    f(std::integral_constant<int, B>{});
    kv_each_byte<D, B + 1>(f);
  }
}

// A workgroup of four waves has 16 query rows of one sequence and key/value head (G query heads times L queries), and a
// share of the tokens; its waves take steps of 32 of them in turn, each with a softmax of its own (running maximum and
// sum, float32), joined in LDS at the end. Shares of the tokens are joined by kv_join_kernel.
//
// The scores of a step, S = K Q^T, come out of the matrix cores with a query row a lane column and 4 tokens a lane group
// and half: exactly as the second product, Y^T += V^T P^T, takes P. Nothing is transposed but the codes' pairs of
// neighbouring channels into pairs of neighbouring tokens, one permute each. q is bfloat16, float16 as two bfloat16
// parts. P is two bfloat16 parts, each to the nearest: within 2^-17 of p, where a single one (2^-8) would cost as much
// again as the output's own rounding, and a third two more matrix instructions to every four.
//
// Bound by the instructions between the loads and the matrix cores (two codes a conversion, two a permute), so addresses
// are a wave's: a step whose tokens lie in one run of slots (KV_RUN: pages of whole steps, or a sequence in one page,
// whose last step starts early enough to end with it) needs one place. Masks are for the steps that need them.
//
// Traced medians: one sequence of 131072 tokens, 32 query and 8 key/value heads of 128, float16: 31 us (4.6 TB/s); 32
// sequences of 2048 to 8192, bfloat16: 44 (4.2 TB/s); the joins 5.2 and 5.0. Counted, 257 and 232 vector instructions a step,
// which keep the vector units busy 0.6 of the cycles and the matrix cores 0.29 and 0.24. With a place a token and masks in
// every step they took 66 and 68 us. The next step's loads stand under no condition: with three workgroups a CU 41 and 47 us
// under one, 32 and 44 without.
//
// Scores that are no numbers are a row's maximum, and so in all of its sums. Scores of -infinity weigh 0 beside larger ones;
// a row that has nothing else is NaN, one that sees no token 0, and the sum beside a maximum of -infinity says which.
//
// An infinity or NaN among the values of one token must not reach query rows that do not see it (0 times it is NaN): a
// step that holds a scale from which codes leave bfloat16's range is left out, and summed token by token behind the
// others.
template <typename T, int D, int MODE>
__global__ __launch_bounds__(256, D <= 128 && MODE == KV_RUN ? 3 : 2) void kv_attend_kernel(T* y, float* part, const T* q, KvCache c, KvTable tb,
                                                           KvQuery qa, FastDiv page, FastDiv group, uint32_t tiles16) {
  constexpr int H = std::is_same<T, f16>::value ? 2 : 1, VD = D / 16, PITCH = D + 4;
  constexpr uint32_t row16 = D / 32;
  constexpr int kJoin = 4 * 16 * PITCH, kWords = MODE == KV_PLACES && kKvChunk > kJoin ? kKvChunk : kJoin;
  __shared__ __align__(16) uint32_t smem[kWords];
  __shared__ float stat[4][16][2];
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t split = blockIdx.x, splits = gridDim.x, b = blockIdx.z;
  const uint32_t h = blockIdx.y / tiles16, tile16 = blockIdx.y - h * tiles16;

  const int64_t length = __builtin_amdgcn_readfirstlane(tb.lengths[b]);
  const uint32_t seen = (uint32_t)(length < 0 ? 0 : length > tb.capacity ? tb.capacity : length);
  // this lane's query row, and the last token that it sees
  const uint32_t i0 = tile16 * 16 + r;
  uint32_t gi;
  const uint32_t l = group.divmod(i0 < qa.rows ? i0 : qa.rows - 1, gi);
  const int64_t last64 = length - qa.L + l;
  const int last = (int)(last64 < 0 ? -1 : last64 > 0x7ffffffe ? 0x7ffffffe : last64);
  const int whole = (int)(length - qa.L < -1 ? -1 : length - qa.L);  // tokens up to here every query sees

  bf16x8 qf[H][D / 32];
  {
    const T* p = q + b * qa.sb + l * qa.sl + (h * qa.G + gi) * qa.sh + g * (D / 4);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      u32x4 bits = __builtin_bit_cast(u32x4, load8_any<T>(p + j * 8));
      if (qa.flip) bits ^= 0x80008000u;
      const typename Vec8<T>::type in = __builtin_bit_cast(typename Vec8<T>::type, bits);
      if constexpr (H == 2)
        split_f16(in, qf[0][j], qf[H - 1][j]);
      else
        qf[0][j] = in;
    }
  }

  f32x4 acc[VD];
#pragma unroll
  for (int n = 0; n < VD; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = 0.f;  // top: of q . k, before its scale; sum: of this lane's tokens
  const float scale = qa.scale;
  const uint64_t head = (uint64_t)h * c.head_step;
  // this lane's byte of four tokens' scales, turned to where an exponent stands
  const uint32_t turn = ((D == 128 ? r / 4 : r / 8) * 8 + 9) & 31;

  bool left_out = false;  // whether a step was

  // One step: tokens t0 .. t0 + 31; MASK: those before `low` and after a row's last are left out; SLOW: its values token
  // by token. KV_RUN: at `place` of head 0.
  auto one = [&](auto mask, auto slow, KvStep<D, MODE>& s, int t0, int low, uint32_t place) {
    constexpr bool MASK = decltype(mask)::value, SLOW = decltype(slow)::value;
    if constexpr (MASK) s.drop_unseen(t0, (int)seen, g);
    const bool big = __builtin_amdgcn_ballot_w64(s.template any_big<MASK>()) != 0;
    if (big != SLOW) {
      left_out = left_out || big;
      return;
    }
    f32x4 sc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      sc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const bf16x8 a = fp4_to_bf16(s.k[u].w[j], s.key_scale(u, j));
#pragma unroll
        for (int f = 0; f < H; ++f) sc[u] = mfma16(a, qf[f][j], sc[u]);
      }
    }
    auto here = [&](int n) {
      const int t = t0 + (n / 4) * 16 + g * 4 + n % 4;
      return t <= last && t >= low && (MODE == KV_RUN || s.at[MODE == KV_PLACES ? n : 0] != kNoPlace);
    };
    float p[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      p[n] = sc[n / 4][n % 4];
      if constexpr (MASK) p[n] = here(n) ? p[n] : -INFINITY;
    }
    float most = kv_max(kv_max(kv_max(p[0], p[1]), kv_max(p[2], p[3])), kv_max(kv_max(p[4], p[5]), kv_max(p[6], p[7])));
    most = xlane_fmax<32>(xlane_fmax<16>(most));
    if (__builtin_amdgcn_ballot_w64(!(most <= top))) {  // (a NaN is the maximum too: the row's sums are NaN from here on)
      const float now = kv_max(top, most);
      const bool first = top == -INFINITY;
      const float f = first ? 0.f : __builtin_amdgcn_exp2f((top - now) * scale);
      // Scores of -infinity below a maximum of -infinity have made the sums NaN, as a softmax of nothing else is. Below a
      // larger one they weigh 0. (A lane's sum is of its own tokens, its row's channels are of all: the row's lanes drop both.)
      if (__builtin_amdgcn_ballot_w64(first && sum != 0.f)) {
        if (first && now != -INFINITY) {
          sum = 0.f;
#pragma unroll
          for (int n = 0; n < VD; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
      }
      top = now;
      sum *= f;
#pragma unroll
      for (int n = 0; n < VD; ++n) acc[n] *= f;
    }
    const float from = -top * scale;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      p[n] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[n], scale, from));
      // (a row that has seen nothing yet has no maximum, and a scale of 0 no -infinity)
      if constexpr (MASK) p[n] = here(n) ? p[n] : 0.f;
    }
    sum += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    if constexpr (!SLOW) {
      // P rounded, and what that leaves out (2^-8 of p at most, so a step of it is 2^-16) rounded: within 2^-17
      u32x4 hi, lo;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        hi[n] = __builtin_bit_cast(uint32_t, bf16x2{(bf16)p[2 * n], (bf16)p[2 * n + 1]});
        const float x = p[2 * n] - __builtin_bit_cast(float, hi[n] << 16);
        const float z = p[2 * n + 1] - __builtin_bit_cast(float, hi[n] & 0xffff0000u);
        lo[n] = __builtin_bit_cast(uint32_t, bf16x2{(bf16)x, (bf16)z});
      }
      const bf16x8 ph = __builtin_bit_cast(bf16x8, hi), pl = __builtin_bit_cast(bf16x8, lo);
      kv_each_byte<D, 0>([&](auto byte) {
        constexpr int B = decltype(byte)::value;
        uint32_t w[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) w[n] = kv_pair<B>(s.v[n], s.template value_scale_of<B>(n, r, turn));
        u32x4 even, odd;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          even[n] = __builtin_amdgcn_perm(w[2 * n + 1], w[2 * n], 0x05040100);
          odd[n] = __builtin_amdgcn_perm(w[2 * n + 1], w[2 * n], 0x07060302);
        }
        const bf16x8 a0 = __builtin_bit_cast(bf16x8, even), a1 = __builtin_bit_cast(bf16x8, odd);
        acc[2 * B] = mfma16(a0, ph, acc[2 * B]);
        acc[2 * B + 1] = mfma16(a1, ph, acc[2 * B + 1]);
        acc[2 * B] = mfma16(a0, pl, acc[2 * B]);
        acc[2 * B + 1] = mfma16(a1, pl, acc[2 * B + 1]);
      });
    } else {
      // this lane's outputs are channels VD (4 g + i) + n of its query row
#pragma unroll 1
      for (int t = 0; t < kKvTile; ++t) {
        const int from = ((t % 16) / 4) * 16 + r, n = (t / 16) * 4 + t % 4;
        float mine = 0.f;
        uint32_t at = place + t * row16;
#pragma unroll
        for (int m = 0; m < 8; ++m) {
          if (m == n) {
            mine = p[m];
            if constexpr (MODE == KV_PLACES) at = s.at[m];
          }
        }
        const float pt = __shfl(mine, from);
        if constexpr (MODE == KV_PLACES) at = (uint32_t)__shfl((int)at, from);
        const bool sees = t0 + t <= last && t0 + t >= low && at != kNoPlace;
        const uint64_t to = head + (sees ? at : 0u);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int m = 0; m < VD; ++m) {
            const int d = VD * (4 * g + i) + m;
            const uint32_t pair = fp4_pair<0>(c.v[to * 16 + d / 2], e8m0_operand(c.vs[to + d / 32]));
            const float v = pt * __builtin_bit_cast(float, d & 1 ? pair & 0xffff0000u : pair << 16);
            acc[m][i] += sees ? v : 0.f;
          }
      }
    }
  };
  constexpr std::true_type yes{};
  constexpr std::false_type no{};

  // This workgroup's steps are a share of whole rounds of its four waves, this wave's each fourth. The next one's loads
  // are on the way while a step is computed, where the registers hold both.
  constexpr bool TWO = D <= 128;
  const uint32_t steps = (seen + kKvTile - 1) / kKvTile, rounds = (steps + 3) / 4, per = (rounds + splits - 1) / splits;
  if constexpr (MODE == KV_RUN) {
    const uint32_t first = min(split * per * 4, steps) + wave, end = min((split + 1) * per * 4, steps);
    // where step i's tokens begin: a page that ends inside a step is the last one, and the step ends with it
    auto start = [&](uint32_t i) { return min(i * kKvTile, tb.capacity - kKvTile); };
    // its page's number, by a scalar load that nothing waits for until it is a place; kNoPlace past `to`
    auto page_of = [&](uint32_t i, uint32_t to) -> uint32_t {
      if (i >= to) return kNoPlace;
      if (!tb.pages) return b;
      typedef const __attribute__((address_space(4))) uint32_t* Scalar;
      return ((Scalar)(uintptr_t)tb.pages)[b * tb.step + page.div(start(i))];
    };
    auto place_of = [&](uint32_t i, uint32_t id) -> uint32_t {
      uint32_t slot;
      page.divmod(start(i), slot);
      return id < c.pages ? (uint32_t)(id * c.page_step) + slot * row16 : kNoPlace;
    };
    // steps up to here need no mask: every query sees all of their tokens, and they end by themselves where the tokens do
    // (a length may be past the tokens; a step moved back to end with them has tokens of the one before it)
    const uint32_t plain = min(end, whole < 0 ? 0u : min((uint32_t)whole + 1, seen) / kKvTile);
    KvStep<D, MODE> s0, s1;
    uint32_t i = first, id0 = page_of(i, plain), id1 = page_of(i + 4, plain), id2 = page_of(i + 8, plain);
    const uint32_t mark = first + (plain > first ? (plain - first + 3) / 4 * 4 : 0), marked = page_of(mark, end);
    uint32_t p0 = place_of(i, id0), p1 = place_of(i + 4, id1);
    // Loads stand under no condition (page 0's for a step that has none): behind one the compiler would wait for all.
    auto load = [&](KvStep<D, MODE>& s, uint32_t at) { s.load_run(c, head + (at == kNoPlace ? 0u : at), r, g); };
    if constexpr (TWO) load(s0, p0);
    // those that do, first: their loads wait beside the others'
    for (uint32_t j = mark; j < end; j += 4) {
      const uint32_t at = place_of(j, j == mark ? marked : page_of(j, end));
      if (at == kNoPlace) continue;
      s1.load_run(c, head + at, r, g);
      one(yes, no, s1, (int)start(j), (int)(j * kKvTile), at);
    }
    while (i < plain) {
      const uint32_t p2 = place_of(i + 8, id2);
      id2 = page_of(i + 12, plain);
      if constexpr (TWO) {
        load(s1, p1);
        if (p0 != kNoPlace) one(no, no, s0, (int)(i * kKvTile), 0, p0);
        i += 4;
        if (i >= plain) break;
        const uint32_t p3 = place_of(i + 8, id2);
        id2 = page_of(i + 12, plain);
        load(s0, p2);
        if (p1 != kNoPlace) one(no, no, s1, (int)(i * kKvTile), 0, p1);
        i += 4;
        p0 = p2;
        p1 = p3;
      } else {
        if (p0 != kNoPlace) {
          s0.load_run(c, head + p0, r, g);
          one(no, no, s0, (int)(i * kKvTile), 0, p0);
        }
        i += 4;
        p0 = p1;
        p1 = p2;
      }
    }
    if (left_out) {
#pragma unroll 1
      for (uint32_t j = first; j < end; j += 4) {
        const uint32_t at = place_of(j, page_of(j, end));
        if (at == kNoPlace) continue;
        s0.load_run(c, head + at, r, g);
        one(yes, yes, s0, (int)start(j), (int)(j * kKvTile), at);
      }
    }
  } else {
    const uint32_t from = min(split * per * 4 * kKvTile, seen), to = min((split + 1) * per * 4 * kKvTile, seen);
    for (uint32_t c0 = from; c0 < to; c0 += kKvChunk) {
      const uint32_t n = min(to - c0, (uint32_t)kKvChunk), padded = (n + kKvTile - 1) / kKvTile * kKvTile;
      __syncthreads();  // the places before these have been read
      for (uint32_t t = tid; t < padded; t += 256)
        smem[t] = t < n ? kv_place(c, tb, page, row16, b, c0 + t) : kNoPlace;
      __syncthreads();
      const uint32_t here = padded / kKvTile;
      KvStep<D, MODE> s0, s1;
      left_out = false;
      if constexpr (TWO) {
        if ((uint32_t)wave < here) s0.load_places(c, head, smem + wave * kKvTile, r, g);
        for (uint32_t i = wave; i < here; i += 8) {
          s1.load_places(c, head, smem + min(i + 4, here - 1) * kKvTile, r, g);
          one(yes, no, s0, (int)(c0 + i * kKvTile), 0, 0u);
          if (i + 4 >= here) break;
          s0.load_places(c, head, smem + min(i + 8, here - 1) * kKvTile, r, g);
          one(yes, no, s1, (int)(c0 + (i + 4) * kKvTile), 0, 0u);
        }
      } else {
        for (uint32_t i = wave; i < here; i += 4) {
          s0.load_places(c, head, smem + i * kKvTile, r, g);
          one(yes, no, s0, (int)(c0 + i * kKvTile), 0, 0u);
        }
      }
      if (left_out) {
#pragma unroll 1
        for (uint32_t i = wave; i < here; i += 4) {
          s0.load_places(c, head, smem + i * kKvTile, r, g);
          one(yes, yes, s0, (int)(c0 + i * kKvTile), 0, 0u);
        }
      }
    }
  }

  // the waves' sums meet
  sum = xlane_sum<32>(xlane_sum<16>(sum));
  __syncthreads();
  if (g == 0) {
    stat[wave][r][0] = top;
    stat[wave][r][1] = sum;
  }
  __syncthreads();
  float all = stat[0][r][0];
#pragma unroll
  for (int w = 1; w < 4; ++w) all = kv_max(all, stat[w][r][0]);
  const float f = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((top - all) * scale);
  float* const rows = reinterpret_cast<float*>(smem);
  float* const out = rows + (wave * 16 + r) * PITCH + g * (D / 4);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < VD; ++n) out[i * VD + n] = acc[n][i] * f;
  __syncthreads();
  for (int e = tid; e < 16 * (D / 8); e += 256) {
    const int row = e / (D / 8), d = e % (D / 8) * 8;
    const uint32_t i = tile16 * 16 + row;
    if (i >= qa.rows) continue;
    float m = stat[0][row][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) m = kv_max(m, stat[w][row][0]);
    float total = 0.f, v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float t = stat[w][row][0];
      if (t == -INFINITY) {  // its sum is 0, or NaN where the row sees tokens, which counts if no wave has more
        if (m == -INFINITY) total += stat[w][row][1];
        continue;
      }
      total += stat[w][row][1] * __builtin_amdgcn_exp2f((t - m) * scale);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += rows[(w * 16 + row) * PITCH + d + j];
    }
    if (splits == 1) {
      uint32_t gi;
      const uint32_t l = group.divmod(i, gi);
      const float inv = m == -INFINITY && total == 0.f ? 0.f : 1.f / total;  // (zeros where no token is seen)
      typename Vec8<T>::type o;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = from_f32<T>(v[j] * inv);
      store8<T>(y + (((uint64_t)b * qa.L + l) * qa.Hq + h * qa.G + gi) * D + d, o);
    } else {
      const uint64_t unit = ((uint64_t)b * gridDim.y + blockIdx.y) * splits + split;
      float* ps = part + (unit * 16 + row) * (D + 4);
      if (m != -INFINITY) {  // what was never summed is not read
        *reinterpret_cast<f32x4*>(ps + d) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(ps + d + 4) = f32x4{v[4], v[5], v[6], v[7]};
      }
      if (d == 0) {
        ps[D] = m;
        ps[D + 1] = total;
      }
    }
  }
}

// The shares' sums of one query row, added by a workgroup: a thread a share for their weights, then four channels a lane
// and several shares at a time.
constexpr int kKvShares = 256;

template <typename T, int D>
__global__ __launch_bounds__(256) void kv_join_kernel(T* y, const float* part, uint32_t splits, KvQuery qa,
                                                      FastDiv group, FastDiv rows, uint32_t tiles16) {
  constexpr int LANES = D / 4, PAR = 256 / LANES;
  __shared__ float weight[kKvShares];
  __shared__ float sums[PAR][D];
  __shared__ float tops[4], totals[4];
  uint32_t i, gi;
  const uint32_t bh = rows.divmod(blockIdx.x, i);  // (sequence, head) and query row
  const uint32_t unit = bh * tiles16 + i / 16;
  const float* p = part + ((uint64_t)unit * splits * 16 + i % 16) * (D + 4);
  const int64_t step = 16 * (D + 4);
  const int t = threadIdx.x, wave = t / kWave;
  const bool mine = (uint32_t)t < splits;
  const float own = mine ? p[t * step + D] : -INFINITY, count = mine ? p[t * step + D + 1] : 0.f;
  float m = kv_max(own, xlane_dpp<1>(own));
  m = kv_max(m, xlane_dpp<2>(m));
  m = kv_max(m, xlane_dpp<4>(m));
  m = kv_max(m, xlane_dpp<8>(m));
  m = xlane_fmax<32>(xlane_fmax<16>(m));
  if (t % kWave == 0) tops[wave] = m;
  __syncthreads();
  m = kv_max(kv_max(tops[0], tops[1]), kv_max(tops[2], tops[3]));
  const float w = own == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((own - m) * qa.scale);
  weight[t] = w;
  const float all = wave_sum(own != -INFINITY ? count * w : m == -INFINITY ? count : 0.f);  // (as between waves)
  if (t % kWave == 0) totals[wave] = all;
  __syncthreads();
  const int lane = t % LANES, at = t / LANES;
  if (at < PAR) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (uint32_t s = at; s < splits; s += PAR) {
      const float f = weight[s];
      if (f != 0.f) v += *reinterpret_cast<const f32x4*>(p + s * step + lane * 4) * f;  // (NaN is not 0)
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[at][lane * 4 + j] = v[j];
  }
  __syncthreads();
  const uint32_t heads = qa.Hq / qa.G, b = bh / heads, h = bh - b * heads, l = group.divmod(i, gi);
  const float total = (totals[0] + totals[1]) + (totals[2] + totals[3]);
  const float inv = m == -INFINITY && total == 0.f ? 0.f : 1.f / total;
  T* to = y + (((uint64_t)b * qa.L + l) * qa.Hq + h * qa.G + gi) * D;
  for (int d = t; d < D; d += 256) {
    float v = 0.f;
#pragma unroll
    for (int s = 0; s < PAR; ++s) v += sums[s][d];
    to[d] = from_f32<T>(v * inv);
  }
}

namespace {

bool kv_dim(int64_t d) { return d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

// Bytes from the first to past the last code of a cache's tensor (below 2^36 where kv_check passes; strides may be any).
__int128 kv_span(const fd_kv_shape& s, int64_t row) {
  return (__int128)(s.pages - 1) * s.page_stride + (__int128)(s.heads - 1) * s.head_stride + s.page * row;
}

int kv_check(const fd_kv_shape* s, const void* k, const void* ks, const void* v, const void* vs, const int32_t* lengths,
             const int32_t* table, int64_t table_stride, int64_t table_pages, int64_t B, KvCache* c, KvTable* tb) {
  if (!s) return set_error(FD_EINVAL, "null pointer argument");
  if (s->pages < 0 || s->heads < 1 || s->page < 1) return set_error(FD_EINVAL, "a cache has pages, heads and slots");
  if (!kv_dim(s->dim)) return set_error(FD_EUNSUPPORTED, "dim must be 64, 96, 128, 192 or 256, got %lld", (long long)s->dim);
  const int64_t row = s->dim / 2;
  if (s->page_stride < 0 || s->head_stride < 0 || table_stride < 0 || table_pages < 0)
    return set_error(FD_EINVAL, "negative stride or size");
  if (s->page_stride % 16 || s->head_stride % 16)
    return set_error(FD_EUNSUPPORTED, "a cache's strides must be multiples of 16 bytes of codes");
  if (s->pages > 0x7fffffffLL || s->heads > 65535 || s->page > 0x7fffffffLL || B > 65535)
    return set_error(FD_EUNSUPPORTED, "too large");
  if (s->pages > 0 && kv_span(*s, row) / 16 >= 0xffffffffLL)
    return set_error(FD_EUNSUPPORTED, "a cache's tensor of 64 GiB of codes or more");
  if (rows_meet(fd_rows{1, s->pages, s->heads, 0, s->page_stride, s->head_stride, 1, s->page * row}))
    return set_error(FD_EINVAL, "a cache's slots must not share memory");
  if (B > 0 && !lengths) return set_error(FD_EINVAL, "null pointer argument");
  if (s->pages > 0 && (!k || !ks || !v || !vs)) return set_error(FD_EINVAL, "null pointer argument");
  if (!aligned16(k) || !aligned16(v)) return set_error(FD_EUNSUPPORTED, "codes must be 16-byte aligned");
  if (!table && B > s->pages) return set_error(FD_EINVAL, "without a table each sequence has a page: %lld, %lld pages",
                                               (long long)B, (long long)s->pages);
  const int64_t capacity = table ? table_pages * s->page : s->page;
  if (capacity > 0x7fffffffLL - 4096) return set_error(FD_EUNSUPPORTED, "a sequence of 2^31 tokens or more");
  *c = KvCache{(uint8_t*)k, (uint8_t*)ks, (uint8_t*)v, (uint8_t*)vs, (uint32_t)s->pages, (uint32_t)s->heads,
               (uint32_t)s->page, s->page_stride / 16, s->head_stride / 16};
  *tb = KvTable{lengths, table, table_stride, (uint32_t)capacity};
  return FD_OK;
}

// Whether [p, p + n) meets one of the cache's tensors.
bool kv_meets(const fd_kv_shape& s, const KvCache& c, const void* p, int64_t n) {
  const int64_t codes = s.pages > 0 ? (int64_t)kv_span(s, s.dim / 2) : 0, scales = codes / 16;
  return overlaps(p, n, c.k, codes) || overlaps(p, n, c.v, codes) || overlaps(p, n, c.ks, scales) ||
         overlaps(p, n, c.vs, scales);
}

// Query rows of a workgroup's tile, and the shares that a sequence's tokens are cut into: as many as give every CU two
// workgroups, each with 256 tokens at least of a cache that is full. (One, two, three, four workgroups a CU, with the
// join: one sequence of 131072 tokens, 8 heads of 128, 55, 45, 48, 51 us; 32 of 2048 to 8192, 85, 56, 57, 58; captured,
// while the step's loads were still under a condition.)
int64_t kv_tiles(int64_t L, int64_t G) { return (L * G + 15) / 16; }
// Whether a launch holds the query rows of L queries and G heads for each of the cache's `heads`.
bool kv_rows_fit(int64_t L, int64_t G, int64_t heads) {
  constexpr int64_t most = 0x7fffffffLL;
  return L <= most && G <= most && L * G <= most && kv_tiles(L, G) <= 65535 / heads;
}
int64_t kv_splits(int64_t B, int64_t L, int64_t Hq, int64_t heads, int64_t capacity) {
  const int64_t units = B * heads * kv_tiles(L, Hq / heads);
  int64_t s = units > 0 ? (2 * device_cus() + units - 1) / units : 1;
  const int64_t most = (capacity + 255) / 256;
  if (s > most) s = most;
  return s < 1 ? 1 : s > kKvShares ? kKvShares : s;
}

template <typename T, int D>
int kv_attend_launch(T* y, float* scratch, const T* q, const KvCache& c, const KvTable& tb, const KvQuery& qa, int64_t B,
                     int64_t splits, hipStream_t st) {
  const int64_t tiles = kv_tiles(qa.L, qa.G);
  const FastDiv group(qa.G);
  // steps in one run of slots: pages of whole steps, or a sequence in one page of a step at least
  const bool run = tb.pages ? c.page % kKvTile == 0 && tb.capacity > 0 : c.page >= kKvTile;
  auto kernel = run ? kv_attend_kernel<T, D, KV_RUN> : kv_attend_kernel<T, D, KV_PLACES>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)splits, (unsigned)(c.heads * tiles), (unsigned)B), dim3(256), 0, st, y,
                     scratch, q, c, tb, qa, FastDiv(c.page), group, (uint32_t)tiles);
  if (splits > 1)
    hipLaunchKernelGGL((kv_join_kernel<T, D>), dim3((unsigned)(B * c.heads * qa.rows)), dim3(256), 0, st, y, scratch,
                       (uint32_t)splits, qa, group, FastDiv(qa.rows), (uint32_t)tiles);
  return FD_OK;
}

template <typename T>
int kv_attend_pick(int64_t dim, T* y, float* scratch, const T* q, const KvCache& c, const KvTable& tb, const KvQuery& qa,
                   int64_t B, int64_t splits, hipStream_t st) {
  switch (dim) {
    case 64: return kv_attend_launch<T, 64>(y, scratch, q, c, tb, qa, B, splits, st);
    case 96: return kv_attend_launch<T, 96>(y, scratch, q, c, tb, qa, B, splits, st);
    case 128: return kv_attend_launch<T, 128>(y, scratch, q, c, tb, qa, B, splits, st);
    case 192: return kv_attend_launch<T, 192>(y, scratch, q, c, tb, qa, B, splits, st);
    default: return kv_attend_launch<T, 256>(y, scratch, q, c, tb, qa, B, splits, st);
  }
}

int64_t kv_q_span(int64_t B, int64_t L, int64_t H, int64_t dim, int64_t sb, int64_t sl, int64_t sh) {
  return ((B - 1) * sb + (L - 1) * sl + (H - 1) * sh + dim) * 2;
}

}  // namespace
}  // namespace fd

using namespace fd;

extern "C" int fd_append_kv_fp4(void* k, void* k_scale, void* v, void* v_scale, const fd_kv_shape* shape,
                                const void* new_k, const void* new_v, int64_t skb, int64_t skl, int64_t skh, int64_t svb,
                                int64_t svl, int64_t svh, const int32_t* lengths, const int32_t* table,
                                int64_t table_stride, int64_t table_pages, int64_t B, int64_t L, int act_dtype,
                                void* stream) {
  if (!check_act_dtype(act_dtype)) return FD_EINVAL;
  if (B < 0 || L < 0) return set_error(FD_EINVAL, "negative size");
  if (skb < 0 || skl < 0 || skh < 0 || svb < 0 || svl < 0 || svh < 0) return set_error(FD_EINVAL, "negative stride");
  KvCache c;
  KvTable tb;
  const int rc = kv_check(shape, k, k_scale, v, v_scale, lengths, table, table_stride, table_pages, B, &c, &tb);
  if (rc != FD_OK) return rc;
  if (B == 0 || L == 0 || tb.capacity == 0 || shape->pages == 0) return FD_OK;
  if (!new_k || !new_v) return set_error(FD_EINVAL, "null pointer argument");
  const int64_t codes = (int64_t)kv_span(*shape, shape->dim / 2), scales = codes / 16;
  const void* t[4] = {k, k_scale, v, v_scale};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < i; ++j)
      if (overlaps(t[i], i % 2 ? scales : codes, t[j], j % 2 ? scales : codes))
        return set_error(FD_EINVAL, "a cache's tensors must not overlap each other");
  const int64_t nk = kv_q_span(B, L, shape->heads, shape->dim, skb, skl, skh);
  const int64_t nv = kv_q_span(B, L, shape->heads, shape->dim, svb, svl, svh);
  if (kv_meets(*shape, c, new_k, nk) || kv_meets(*shape, c, new_v, nv) || kv_meets(*shape, c, lengths, B * 4) ||
      (table && kv_meets(*shape, c, table, ((B - 1) * table_stride + table_pages) * 4)))
    return set_error(FD_EINVAL, "a cache must not overlap what is stored into it");
  const int64_t lanes = shape->dim / 8, of_token = B * shape->heads * lanes;
  if (L > 0x7fffff00LL / of_token) return set_error(FD_EUNSUPPORTED, "too large");
  const int64_t half = of_token * L;
  const dim3 blocks((unsigned)((2 * half + 255) / 256));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  auto go = [&](auto one) {
    typedef decltype(one) T;
    hipLaunchKernelGGL((kv_append_kernel<T>), blocks, dim3(256), 0, st, c, tb, static_cast<const T*>(new_k),
                       static_cast<const T*>(new_v), skb, skl, skh, svb, svl, svh, (uint32_t)L,
                       (uint32_t)(shape->dim / 32), FastDiv((uint32_t)lanes), FastDiv(c.heads), FastDiv((uint32_t)L),
                       FastDiv(c.page), (uint32_t)half, (uint32_t)(2 * half));
  };
  if (act_dtype == FD_F16) go(f16{}); else go(bf16{});
  return check_launch();
}

extern "C" int fd_read_kv_fp4(void* out_k, void* out_v, const void* k, const void* k_scale, const void* v,
                              const void* v_scale, const fd_kv_shape* shape, const int32_t* lengths,
                              const int32_t* table, int64_t table_stride, int64_t table_pages, int64_t B, int64_t count,
                              int act_dtype, void* stream) {
  if (!check_act_dtype(act_dtype)) return FD_EINVAL;
  if (B < 0 || count < 0) return set_error(FD_EINVAL, "negative size");
  KvCache c;
  KvTable tb;
  const int rc = kv_check(shape, k, k_scale, v, v_scale, lengths, table, table_stride, table_pages, B, &c, &tb);
  if (rc != FD_OK) return rc;
  if (B == 0 || count == 0) return FD_OK;
  if (!out_k || !out_v) return set_error(FD_EINVAL, "null pointer argument");
  if (!aligned16(out_k) || !aligned16(out_v)) return set_error(FD_EUNSUPPORTED, "outputs must be 16-byte aligned");
  if (count > 0x7fffffffLL - 4096) return set_error(FD_EUNSUPPORTED, "too large");
  const int64_t n = B * count * shape->heads * shape->dim * 2;
  if (overlaps(out_k, n, out_v, n)) return set_error(FD_EINVAL, "the outputs must not overlap each other");
  for (const void* o : {out_k, out_v})
    if (kv_meets(*shape, c, o, n) || overlaps(o, n, lengths, B * 4) ||
        (table && overlaps(o, n, table, ((B - 1) * table_stride + table_pages) * 4)))
      return set_error(FD_EINVAL, "an output must not overlap what it is read from");
  const int64_t lanes = shape->dim / 8, quads = (count + 3) / 4, rows = B * quads * shape->heads;  // of four tokens
  if (rows > 0x7fffffffLL) return set_error(FD_EUNSUPPORTED, "too large");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t most = 0x40000000LL / (lanes * 4);  // rows of a launch
  auto go = [&](auto one) {
    typedef decltype(one) T;
    for (int64_t r = 0; r < rows; r += most) {
      const int64_t total = (rows - r < most ? rows - r : most) * 4 * lanes;
      hipLaunchKernelGGL((kv_read_kernel<T>), dim3((unsigned)((total + 255) / 256)), dim3(256), 0, st,
                         static_cast<T*>(out_k), static_cast<T*>(out_v), c, tb, (uint32_t)count, (uint32_t)shape->dim,
                         (uint32_t)(shape->dim / 32), FastDiv((uint32_t)lanes), FastDiv(c.heads), FastDiv((uint32_t)quads),
                         FastDiv(c.page), (uint32_t)r, (uint32_t)total);
    }
  };
  if (act_dtype == FD_F16) go(f16{}); else go(bf16{});
  return check_launch();
}

extern "C" int fd_attend_kv_fp4_scratch(int64_t B, int64_t L, int64_t Hq, int64_t heads, int64_t dim, int64_t capacity,
                                        int64_t* bytes) {
  if (B < 0 || L < 0 || Hq < 0 || heads < 1 || capacity < 0) return set_error(FD_EINVAL, "negative size");
  if (Hq % heads) return set_error(FD_EINVAL, "query heads must be a multiple of the cache's");
  if (!kv_dim(dim)) return set_error(FD_EUNSUPPORTED, "dim must be 64, 96, 128, 192 or 256, got %lld", (long long)dim);
  if (!bytes) return set_error(FD_EINVAL, "null pointer argument");
  *bytes = 0;
  if (B == 0 || L == 0 || Hq == 0 || B > 65535 || heads > 65535 || !kv_rows_fit(L, Hq / heads, heads)) return FD_OK;
  const int64_t s = kv_splits(B, L, Hq, heads, capacity);
  if (s > 1) *bytes = B * heads * kv_tiles(L, Hq / heads) * s * 16 * (dim + 4) * 4;
  return FD_OK;
}

extern "C" int fd_attend_kv_fp4(void* y, const void* q, const void* k, const void* k_scale, const void* v,
                                const void* v_scale, const fd_kv_shape* shape, int64_t sqb, int64_t sql, int64_t sqh,
                                const int32_t* lengths, const int32_t* table, int64_t table_stride, int64_t table_pages,
                                int64_t B, int64_t L, int64_t Hq, float scale, float* scratch, int64_t scratch_bytes,
                                int act_dtype, void* stream) {
  if (!check_act_dtype(act_dtype)) return FD_EINVAL;
  if (B < 0 || L < 0 || Hq < 0) return set_error(FD_EINVAL, "negative size");
  if (sqb < 0 || sql < 0 || sqh < 0) return set_error(FD_EINVAL, "negative stride");
  if (!(std::fabs(scale) <= 2e38f)) return set_error(FD_EINVAL, "scale must be a finite value, 2e38 at most");
  KvCache c;
  KvTable tb;
  const int rc = kv_check(shape, k, k_scale, v, v_scale, lengths, table, table_stride, table_pages, B, &c, &tb);
  if (rc != FD_OK) return rc;
  if (Hq % shape->heads) return set_error(FD_EINVAL, "query heads must be a multiple of the cache's: %lld, %lld",
                                          (long long)Hq, (long long)shape->heads);
  if (B == 0 || L == 0 || Hq == 0) return FD_OK;
  if (!y || !q) return set_error(FD_EINVAL, "null pointer argument");
  if (!aligned16(y)) return set_error(FD_EUNSUPPORTED, "y must be 16-byte aligned");
  if (shape->pages == 0) return set_error(FD_EUNSUPPORTED, "a cache without pages");
  const int64_t G = Hq / shape->heads;
  if (!kv_rows_fit(L, G, shape->heads)) return set_error(FD_EUNSUPPORTED, "too many query rows");
  const int64_t tiles = kv_tiles(L, G);
  const int64_t ny = B * L * Hq * shape->dim * 2;
  if (overlaps(y, ny, q, kv_q_span(B, L, Hq, shape->dim, sqb, sql, sqh)) || kv_meets(*shape, c, y, ny) ||
      overlaps(y, ny, lengths, B * 4) || (table && overlaps(y, ny, table, ((B - 1) * table_stride + table_pages) * 4)))
    return set_error(FD_EUNSUPPORTED, "y must not overlap what it is computed from");
  if (scratch && !aligned16(scratch)) return set_error(FD_EUNSUPPORTED, "scratch must be 16-byte aligned");
  int64_t splits = kv_splits(B, L, Hq, shape->heads, tb.capacity);
  while (splits > 1 && (!scratch || scratch_bytes < B * shape->heads * tiles * splits * 16 * (shape->dim + 4) * 4))
    --splits;
  const KvQuery qa{sqb, sql, sqh, (uint32_t)L, (uint32_t)Hq, (uint32_t)G, (uint32_t)(L * G),
                   std::fabs(scale) * 1.4426950408889634f, scale < 0.f};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (act_dtype == FD_F16)
    kv_attend_pick<f16>(shape->dim, static_cast<f16*>(y), scratch, static_cast<const f16*>(q), c, tb, qa, B, splits, st);
  else
    kv_attend_pick<bf16>(shape->dim, static_cast<bf16*>(y), scratch, static_cast<const bf16*>(q), c, tb, qa, B, splits, st);
  return check_launch();
}
