// A cache of keys and values in 4 bits for gfx950 (CDNA4): rows quantised as they are
// written, rows read back, and the newest tokens' attention over them.
//
// A value is step * code: code one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (2 exponent
// bits, 1 of mantissa: what the matrix cores and v_cvt_scalef32_* take as fp4), step the
// group's largest magnitude over 6 rounded to 6 significant bits, a group being 64
// elements of a row (the last 32 where D is an odd multiple of 32). A code has at most 2
// significant bits, so a value has at most 8 and is a bf16 number exactly; with the fp16
// steps' last bit at 2^-23 or above and their largest 10752 it is an fp16 number exactly.
// So rows are read back without rounding, products of values are the matrix cores' own,
// and attention over the cache is attention over the rows read back.
//
// Attention: rows, tiles and shares as in the cache of 16 and 32 bits (fbsa_cache.hip),
// whose join adds up the parts.
#include <algorithm>

#include "fbsa_cache.h"

namespace fbsa {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kGroup4 = 64;  // elements to a step

// ---- steps and codes --------------------------------------------------------
// T is the rows' type: fp16 rows have fp16 steps, the others bf16 ones.
template <typename T> __device__ __forceinline__ float step_f32(uint32_t bits) {  // of the low 16 bits
  if constexpr (__is_same(T, f16)) return (float)__builtin_bit_cast(f16, (uint16_t)bits);
  else return __uint_as_float(bits << 16);
}
// half e & 1 of words[e / 2]
template <typename T> __device__ __forceinline__ float step_half(uint32_t word, int e) {
  if constexpr (__is_same(T, f16)) return (float)__builtin_bit_cast(f16x2, word)[e & 1];
  else return __uint_as_float(e & 1 ? word & 0xffff0000u : word << 16);
}
// 8 codes (element 2i in byte i's low half) as bf16 or fp16 numbers, exact
template <typename K> __device__ __forceinline__ s16x8 codes8(uint32_t w) {
  u32x4 r;
  if constexpr (__is_same(K, f16)) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 3));
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 3));
  }
  return __builtin_bit_cast(s16x8, r);
}
__device__ __forceinline__ void values8_f32(uint32_t w, float step, float (&x)[8]) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3);
  x[0] = a[0] * step; x[1] = a[1] * step; x[2] = b[0] * step; x[3] = b[1] * step;
  x[4] = c[0] * step; x[5] = c[1] * step; x[6] = d[0] * step; x[7] = d[1] * step;
}
// 8 values as bf16 or fp16 numbers, exact
template <typename K> __device__ __forceinline__ s16x8 values8(uint32_t w, float step) {
  if constexpr (__is_same(K, f16)) {
    const f16 s = (f16)step;
    const f16x2 ss = f16x2{s, s};
    const s16x8 c = codes8<f16>(w);
    u32x4 r = __builtin_bit_cast(u32x4, c);
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, (uint32_t)r[j]) * ss);
    return __builtin_bit_cast(s16x8, r);
  } else {
    float x[8];
    values8_f32(w, step, x);
    u32x4 r;  // (nothing is lost: the lower halves are zero, NaN apart, whose upper half stays one)
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = __builtin_amdgcn_perm(__float_as_uint(x[2 * j + 1]), __float_as_uint(x[2 * j]), 0x07060302u);
    return __builtin_bit_cast(s16x8, r);
  }
}

struct Rows4Args {
  void *k4, *v4;
  uint16_t *step;
  void *k, *v;  // the new rows, or where rows are read to
  const int32_t *first, *count;
  int64_t sk4[3], sv4[3];  // bytes
  int64_t ss[2];           // steps
  int64_t sk[3], sv[3];    // elements
  int32_t B, H, T, S, D, ng;
};

// Eight lanes' group: the largest magnitude of its elements
__device__ __forceinline__ float group_max(float x) {
  x = fmaxf(x, shfl_xor_f(x, 1));
  x = fmaxf(x, shfl_xor_f(x, 2));
  return fmaxf(x, shfl_xor_f(x, 4));
}
// largest magnitude / 6 to 6 significant bits, ties to even. The division is correctly
// rounded and a quotient next to a tie never rounds onto one: x = 6 t (1 + d) with x and
// 6 t of 24 bits has a quotient at least 2/3 of a unit from t.
template <typename T> __device__ __forceinline__ float step_of(float most) {
  constexpr bool HALF = __is_same(T, f16);
  const float want = most / 6.f;
  const uint32_t b = __float_as_uint(want), up = b + 0x1ffffu + ((b >> 18) & 1u);
  float s = __uint_as_float(up & 0xfffc0000u);
  // below, the last bit stays at 2^-125 (fp16: 2^-23): values keep to normal numbers (fp16: to the type's own)
  constexpr float LEAST = HALF ? 0x1p-18f : 0x1p-120f, UNIT = HALF ? 0x1p-23f : 0x1p-125f;
  if (want < LEAST) s = __builtin_rintf(want * (1.f / UNIT)) * UNIT;
  return fminf(s, HALF ? 10752.f : 42.f * 0x1p120f);
}

// New rows: 8 elements a lane, LPR lanes a key or value row and both side by side, so the
// row's NaN or infinity is known to all of them. The quotient x / step goes to the
// converter, which rounds to the nearest code, ties to the even one, and saturates. As
// above a quotient is never rounded onto a tie that it is not.
// Bound by memory, long prompts; a step's rows by latency.
template <typename T, int LPR> __global__ __launch_bounds__(256) void cache4_append_kernel(Rows4Args a) {
  constexpr int RPB = 256 / (2 * LPR);
  const int tid = threadIdx.x, lane = tid & 63;
  const int which = (tid / LPR) & 1, e = tid % LPR;  // key or value; elements 8 e ...
  const uint32_t row = blockIdx.x * RPB + tid / (2 * LPR), rows = (uint32_t)a.B * a.H * a.T;
  const bool in = row < rows && 8 * e < a.D;
  const uint32_t x = row < rows ? row : 0;
  const int t = (int)(x % (uint32_t)a.T), h = (int)(x / (uint32_t)a.T % (uint32_t)a.H), b = (int)(x / (uint32_t)a.T / (uint32_t)a.H);
  const int count = a.count ? a.count[b] : a.T;
  const int64_t at = (int64_t)a.first[b] + t;
  const bool live = in && t < count && at >= 0 && at < a.S;
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = 0.f;
  if (live) {
    const int64_t *st = which ? a.sv : a.sk;
    const T *src = (const T *)(which ? a.v : a.k) + b * st[0] + h * st[1] + t * st[2] + 8 * e;
    if constexpr (sizeof(T) == 4) {
      const f32x4 p = ((const f32x4 *)src)[0], q = ((const f32x4 *)src)[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) { y[i] = p[i]; y[4 + i] = q[i]; }
    } else {
      const s16x8 p = *(const s16x8 *)src;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = to_f32<T>(__builtin_bit_cast(T, (short)p[i]));
    }
  }
  float most = 0.f;
  bool odd = false;  // (a maximum passes NaN over)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    most = fmaxf(most, fabsf(y[i]));
    odd = odd || !(fabsf(y[i]) < INFINITY);
  }
  const uint64_t vote = __ballot(odd);
  constexpr uint64_t ROW = LPR == 32 ? ~0ull : (1ull << (2 * LPR % 64)) - 1;
  const bool bad = (vote >> (lane / (2 * LPR) * (2 * LPR)) & ROW) != 0;
  most = LPR >= 8 ? group_max(most) : fmaxf(fmaxf(most, shfl_xor_f(most, 1)), shfl_xor_f(fmaxf(most, shfl_xor_f(most, 1)), 2));
  if (!live) return;
  const float step = bad ? __uint_as_float(0x7fc00000u) : step_of<T>(most);
  uint32_t w = 0;
  if (!bad && step > 0.f) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0] / step, y[1] / step, 1.f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2] / step, y[3] / step, 1.f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4] / step, y[5] / step, 1.f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6] / step, y[7] / step, 1.f, 3);
  }
  const int64_t *s4 = which ? a.sv4 : a.sk4;
  char *dst = (char *)(which ? a.v4 : a.k4) + b * s4[0] + h * s4[1] + at * s4[2] + 4 * e;
  *(uint32_t *)dst = w;
  if (e % 8 == 0) {
    uint16_t *sd = a.step + b * a.ss[0] + h * a.ss[1] + (at * 2 + which) * a.ng + e / 8;
    if constexpr (__is_same(T, f16)) *sd = __builtin_bit_cast(uint16_t, (f16)step);
    else *sd = (uint16_t)(__float_as_uint(step) >> 16);
  }
}

// Rows first[b] + t of each sequence as numbers of type T; rows outside the cache, and
// those from count[b] on, are zeros. 8 values a lane, written whole lines at a time.
template <typename T, int LPR> __global__ __launch_bounds__(256) void cache4_read_kernel(Rows4Args a) {
  constexpr int RPB = 256 / (2 * LPR);
  const int tid = threadIdx.x, which = (tid / LPR) & 1, e = tid % LPR;
  const uint32_t row = blockIdx.x * RPB + tid / (2 * LPR), rows = (uint32_t)a.B * a.H * a.T;
  if (row >= rows || 8 * e >= a.D) return;
  const int t = (int)(row % (uint32_t)a.T), h = (int)(row / (uint32_t)a.T % (uint32_t)a.H), b = (int)(row / (uint32_t)a.T / (uint32_t)a.H);
  const int count = a.count ? a.count[b] : a.T;
  const int64_t at = (int64_t)(a.first ? a.first[b] : 0) + t;
  uint32_t w = 0;
  float step = 0.f;
  if (t < count && at >= 0 && at < a.S) {
    const int64_t *s4 = which ? a.sv4 : a.sk4;
    w = *(const uint32_t *)((const char *)(which ? a.v4 : a.k4) + b * s4[0] + h * s4[1] + at * s4[2] + 4 * e);
    step = step_f32<T>(a.step[b * a.ss[0] + h * a.ss[1] + (at * 2 + which) * a.ng + e / 8]);
  }
  const int64_t *st = which ? a.sv : a.sk;
  T *dst = (T *)(which ? a.v : a.k) + b * st[0] + h * st[1] + t * st[2] + 8 * e;
  if constexpr (sizeof(T) == 4) {
    float x[8];
    values8_f32(w, step, x);
    ((f32x4 *)dst)[0] = f32x4{x[0], x[1], x[2], x[3]};
    ((f32x4 *)dst)[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    *(s16x8 *)dst = values8<T>(w, step);
  }
}

// ---- attention ----------------------------------------------------------------
struct Cache4Args {
  CacheArgs a;           // k, v: the codes; sk, sv in bytes
  const uint16_t *step;
  int64_t ss[2];
  int32_t ng;            // steps of a key or value row
};

// Queries and probabilities enter the products as sums of 16-bit numbers: a 32-bit number
// is three bf16 exactly (8 bits each).
template <typename T> struct Pieces {
  using K = bf16;                                                   // the product's type
  static constexpr int Q = 1, P = 2;
};
template <> struct Pieces<f16> { using K = f16; static constexpr int Q = 1, P = 2; };
template <> struct Pieces<float> { using K = bf16; static constexpr int Q = 3, P = 3; };

// x as N bf16 numbers, each what the ones before leave (the last rounded, the others cut)
template <int N> __device__ __forceinline__ void split8(const float *x, s16x8 *out) {
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
  for (int n = 0; n + 1 < N; ++n) {
    u32x4 hw;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = __float_as_uint(r[2 * j]), b = __float_as_uint(r[2 * j + 1]);
      hw[j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      r[2 * j] -= __uint_as_float(a & 0xffff0000u);
      r[2 * j + 1] -= __uint_as_float(b & 0xffff0000u);
    }
    out[n] = __builtin_bit_cast(s16x8, hw);
  }
  out[N - 1] = pack8<bf16>(r);
}
// elements d .. d + 7 of a query row (zeros past the head dim), the scale's sign applied
template <typename T> __device__ __forceinline__ void load_q8(const CacheArgs &a, const T *row, int d, s16x8 *out) {
  if constexpr (sizeof(T) == 4) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const u32x4 w = d < a.D ? ((const u32x4 *)(row + d))[i] : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = __uint_as_float((w[e] & a.qand) ^ a.qxor);
    }
    split8<3>(x, out);
  } else {
    u32x4 w = d < a.D ? *(const u32x4 *)(row + d) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = (w[e] & a.qand) ^ a.qxor;
    out[0] = __builtin_bit_cast(s16x8, w);
  }
}

// A chunk of 64 rows in LDS: codes of keys, codes of values, steps. A row of codes is CPR
// units of 16 bytes, unit c at c ^ swk(row) (values: swv), which keeps the reads below
// off each other's banks as far as 16-byte units can: none for keys, two lanes to a bank for values.
template <int DP> struct Part4 {
  static constexpr int KC = 64, RB = DP / 2, CPR = RB / 16, NG = DP <= kGroup4 ? 1 : DP / kGroup4;
  static constexpr int TILE = KC * RB, STEPS = KC * 4 * NG, STAGE = 2 * TILE + STEPS, LOADS = 2 * CPR + NG;
  static constexpr int NS = DP <= 64 ? 4 : DP == 128 ? 3 : 2;  // stages of the ring
  __device__ static __forceinline__ int swk(int row) {
    return CPR == 1 ? 0 : CPR == 4 ? (row >> 2) & 3 : CPR == 8 ? (row >> 1) & 7 : (row >> 3) & 1;
  }
  __device__ static __forceinline__ int swv(int row) {
    return CPR == 1 ? 0 : CPR == 4 ? (row >> 4) & 3 : CPR == 8 ? ((row >> 4) & 3) | (row & 2) << 1 : (row >> 4) & 1;
  }
};

// Steps of four keys from `at` on (a multiple of 4): number e of 2 NG of key r
template <typename T, int NG> struct Steps4 {
  u32x4 w[NG];
  __device__ __forceinline__ void load(const char *steps, int at) {
#pragma unroll
    for (int i = 0; i < NG; ++i) w[i] = ((const u32x4 *)(steps + at * 4 * NG))[i];
  }
  __device__ __forceinline__ float get(int r, int e) const { return step_half<T>(w[(r * NG + e / 2) / 4][(r * NG + e / 2) % 4], e); }
};

// Up to 16 rows: a wave per (tile, share of the keys). Codes go to LDS through a ring of
// the wave's own and are made 16-bit numbers on their way into the matrix units (one
// instruction for two), the steps applied in 32 bits: to the scores of a group's product,
// and to the probabilities before the value product, one set of them for each group.
// Keys past what a row sees have p = 0, codes are finite whatever they are, and a step
// that is NaN counts as 0 there, so nothing that is not seen comes through.
//   scores: S^T = K Q^T, 16 keys x 16 rows a product; lane (g, p) has keys 16 m + 4 g + r of row p
//   values: O^T = V^T P, 16 columns x 16 rows over 32 keys; a transposing read gives lane
//   (g, i) one column's 16 keys 16 a + 4 g + b, a, b < 4: the order that P has anyway.
// QUAD (up to 4 rows): the columns of Q are 4 rows x 4 quarters of the chunk, zero outside
// the quarter's own lanes, so a product of 16 x 16 has the scores of 64 keys and no lane
// holds one twice: a quarter of the exponentials and splits. Each (row, quarter) has a
// softmax of its own, joined at the end.
template <typename T, int DP, bool QUAD> __global__ __launch_bounds__(64) void cache4_part_kernel(Cache4Args c4) {
  using C = Part4<DP>;
  using K = typename Pieces<T>::K;
  constexpr int KC = C::KC, NM = QUAD ? 1 : KC / 16, NG = C::NG, NQ = Pieces<T>::Q, NP = Pieces<T>::P, NT = DP / 16;
  constexpr int NF = QUAD ? DP / 8 : DP / 32, PITCH = DP == 192 ? 256 : DP;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const CacheArgs &a = c4.a;
  const int lane = threadIdx.x, g = lane >> 4, p = lane & 15, quarter = p >> 2;
  const uint32_t id = blockIdx.x;
  const int tile = id % a.rt_own, hk = id / a.rt_own / a.np_own % a.Hkv, b = id / a.rt_own / a.np_own / a.Hkv;
  const int split = id / a.rt_own % a.np_own, rho = tile * a.tr_own + (QUAD ? p & 3 : p);
  const RowInfo ri = row_info(a, b, hk, rho);
  int keys, low;
  own_bounds(a, b, tile * a.tr_own, min(tile * a.tr_own + a.tr_own, a.TG), keys, low);
  const int64_t slot = (((int64_t)b * a.Hkv + hk) * a.rt_own + tile) * a.np_own * a.tr_own + split * a.tr_own;
  const int lim = ri.valid ? ri.lim : keys;
  int c0, c1;
  share_of((keys + KC - 1) / KC, split, a.np_own, c0, c1);

  s16x8 fr[NF][NQ];
  const T *qrow = (const T *)a.q + ri.b * a.sq[0] + ri.hq * a.sq[1] + ri.t * a.sq[2];
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    load_q8<T>(a, qrow, QUAD ? 8 * f : DP == 32 ? 8 * g : 64 * (f / 2) + 16 * g + 8 * (f % 2), fr[f]);
    if (QUAD && g != quarter) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) fr[f][n] = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
    }
  }

  const int64_t kstep = a.sk[2], vstep = a.sv[2];
  const char *kb = (const char *)a.k + b * a.sk[0] + hk * a.sk[1], *vb = (const char *)a.v + b * a.sv[0] + hk * a.sv[1];
  const char *sb = (const char *)(c4.step + b * c4.ss[0] + hk * c4.ss[1]);
  uint32_t koff[C::CPR], voff[C::CPR];
#pragma unroll
  for (int n = 0; n < C::CPR; ++n) {
    const int u = n * 64 + lane, row = u / C::CPR, c = u % C::CPR, last = a.D / 32 - 1;
    const int ck = c ^ C::swk(row), cv = c ^ C::swv(row);  // (columns past the head dim: the row's last unit)
    koff[n] = (uint32_t)(row * kstep + (ck < last ? ck : last) * 16);
    voff[n] = (uint32_t)(row * vstep + (cv < last ? cv : last) * 16);
  }
  auto issue = [&](int c, int stage) {
    const unsigned st = (unsigned)(uintptr_t)smem + stage * C::STAGE;
    const uint32_t row0 = (uint32_t)c * KC;
    const uint32_t klim = tail_limit<KC>(row0, keys, (uint32_t)kstep, (uint32_t)a.D / 2), vlim = tail_limit<KC>(row0, keys, (uint32_t)vstep, (uint32_t)a.D / 2);
#pragma unroll
    for (int n = 0; n < C::CPR; ++n) g2lds16_s(kb + row0 * kstep, koff[n] > klim ? klim : koff[n], st + n * 1024);
#pragma unroll
    for (int n = 0; n < C::CPR; ++n) g2lds16_s(vb + row0 * vstep, voff[n] > vlim ? vlim : voff[n], st + C::TILE + n * 1024);
    const uint32_t words = min((uint32_t)KC, keys - row0) * NG;  // (rows past the end: the last step)
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const uint32_t u = n * 64 + lane;
      g2lds4(sb + ((int64_t)row0 * NG + (u < words ? u : words - 1)) * 4, smem + stage * C::STAGE + 2 * C::TILE + n * 256);
    }
  };
  // this lane's keys: 16 m + 4 g + r (QUAD: 16 quarter + 4 g + r)
  const int key0 = QUAD ? 16 * quarter + 4 * g : 4 * g;
  const int vrow = 16 * (p >> 2) + 4 * g + (p & 3), vswz = C::swv(vrow), krow = QUAD ? lane : p, kswz = C::swk(krow);

  SoftmaxState<DP> sm;
  sm.init();
  for (int n = 0; n < C::NS - 1; ++n)
    if (c0 + n < c1) issue(c0 + n, n);
  int stage = 0;
  for (int c = c0; c < c1; ++c) {
    wait_ring<C::LOADS>(min(C::NS - 2, c1 - 1 - c));
    lds_wait_all();  // the previous chunk's reads, whose stage is written next
    if (c + C::NS - 1 < c1) issue(c + C::NS - 1, stage == 0 ? C::NS - 1 : stage - 1);
    const char *Ks = smem + stage * C::STAGE, *Vs = Ks + C::TILE, *Ss = Vs + C::TILE;
    stage = stage == C::NS - 1 ? 0 : stage + 1;

    f32x4 s[NM];
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      Steps4<T, NG> st;
      st.load(Ss, key0 + 16 * m);
      const char *row = Ks + (krow + 16 * m) * C::RB;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
        auto mul = [&](uint32_t w, const s16x8 *q) {
          const s16x8 x = codes8<K>(w);
#pragma unroll
          for (int n = NQ - 1; n >= 0; --n) acc = Mfma16<K>::run(x, q[n], acc);
        };
        if constexpr (QUAD) {
#pragma unroll
          for (int u = 2 * j; u < (DP == 32 ? 1 : 2 * j + 2); ++u) {
            const u32x4 w = *(const u32x4 *)(row + ((u ^ kswz) << 4));
#pragma unroll
            for (int i = 0; i < 4; ++i) mul(w[i], fr[4 * u + i]);
          }
        } else if constexpr (DP == 32) {
          mul(*(const uint32_t *)(row + 4 * g), fr[0]);
        } else {
          const u32x2 w = *(const u32x2 *)(row + (((2 * j + (g >> 1)) ^ kswz) << 4) + (g & 1) * 8);
          mul(w[0], fr[2 * j]);
          mul(w[1], fr[2 * j + 1]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) s[m][r] = j ? __builtin_fmaf(acc[r], st.get(r, j), s[m][r]) : acc[r] * st.get(r, 0);
      }
    }
    if ((c + 1) * (int64_t)KC > low) {
#pragma unroll
      for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (key0 + 16 * m + r >= lim - c * KC) s[m][r] = -INFINITY;
    }
    float x[NM][4];
    sm.template step<NM>(s, a.scale2, x);

#pragma unroll
    for (int j = 0; j < NG; ++j) {
      s16x8 pk[2][NP];  // keys of the transposing read's first and second word
      if constexpr (QUAD) {
        Steps4<T, NG> st;
        st.load(Ss, key0);
        float y[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          y[r] = x[0][r] * fmaxf(st.get(r, NG + j), 0.f);
          y[4 + r] = 0.f;
        }
        s16x8 one[NP];
        split8<NP>(y, one);
#pragma unroll
        for (int n = 0; n < NP; ++n) {
          const u32x4 w = __builtin_bit_cast(u32x4, one[n]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            u32x4 z;
            z[0] = quarter == 2 * h ? w[0] : 0u;
            z[1] = quarter == 2 * h ? w[1] : 0u;
            z[2] = quarter == 2 * h + 1 ? w[0] : 0u;
            z[3] = quarter == 2 * h + 1 ? w[1] : 0u;
            pk[h][n] = __builtin_bit_cast(s16x8, z);
          }
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float y[8];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            Steps4<T, NG> st;
            st.load(Ss, key0 + 16 * (2 * h + i));
#pragma unroll
            for (int r = 0; r < 4; ++r) y[4 * i + r] = x[2 * h + i][r] * fmaxf(st.get(r, NG + j), 0.f);
          }
          split8<NP>(y, pk[h]);
        }
      }
      constexpr int TG4 = NT < 4 ? NT : 4;  // 16-column tiles of a group
      i32x2 w[TG4];
#pragma unroll
      for (int t = 0; t < TG4; ++t) {
        const int tt = 4 * j + t;
        const char *at = Vs + vrow * C::RB + (((tt >> 1) ^ vswz) << 4) + (tt & 1) * 8;
        w[t] = __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) i32x2 *)(uintptr_t)(uint32_t)(uintptr_t)at);
      }
#pragma unroll
      for (int t = 0; t < TG4; ++t) {
        const s16x8 v0 = codes8<bf16>((uint32_t)w[t][0]), v1 = codes8<bf16>((uint32_t)w[t][1]);
#pragma unroll
        for (int n = NP - 1; n >= 0; --n) {
          sm.o[4 * j + t] = Mfma16<bf16>::run(v0, pk[0][n], sm.o[4 * j + t]);
          sm.o[4 * j + t] = Mfma16<bf16>::run(v1, pk[1][n], sm.o[4 * j + t]);
        }
      }
    }
  }

  float lt = sm.total(), m = sm.m;
  if constexpr (QUAD) {
    // the four quarters of a row, lanes p & 3 of each
    float mq = fmaxf(m, shfl_xor_f(m, 4));
    mq = fmaxf(mq, shfl_xor_f(mq, 8));
    const float f = m == -INFINITY ? (lt == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - mq);  // (NaN sums are kept)
    m = mq;
    lt *= f;
    lt += shfl_xor_f(lt, 4);
    lt += shfl_xor_f(lt, 8);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float y = sm.o[t][r] * f;
        y += shfl_xor_f(y, 4);
        sm.o[t][r] = y + shfl_xor_f(y, 8);
      }
    if (p >= 4) return;
  }
  if (a.direct) {
    if (rho >= a.TG) return;
    const float l = ri.valid ? lt : 0.f, inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int t = 0; t < NT; ++t) store_row<T>(a, ri, sm.o[t], inv, 16 * t + 4 * g);
    if (g == 0 && a.lse) a.lse[((int64_t)ri.b * a.Hq + ri.hq) * a.T + ri.t] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
    return;
  }
  if (g == 0) a.stat[slot + p] = float2{m, lt};
  if (ri.valid && lt != 0.f) {  // (a NaN sum is kept)
    float *dst = a.part + (slot + p) * PITCH;
#pragma unroll
    for (int t = 0; t < NT; ++t) *(f32x4 *)(dst + 16 * t + 4 * g) = sm.o[t];
  }
}

// Many rows: a workgroup per (tile of NW x 16 QT rows, share of the keys). Its threads
// make 16-bit numbers of the codes, steps and all (exact), into two stages of LDS, and
// from there it is the tile of a 16-bit cache. 32-bit rows are three bf16 pieces of
// queries and of probabilities: six products of the matrix units' fastest type cost less
// than two of the slow 32-bit one.
template <typename K, int DP, int QT, int NM, int N>
__device__ __forceinline__ void qk_pieces(const char *tile, const RowFrag<K, DP> (&fr)[N][QT], f32x4 (&acc)[QT][NM], int g, int p) {
  qk_tile<K, DP, QT, NM>(tile, fr[0], acc, g, p);
  if constexpr (N > 1) {
#pragma unroll
    for (int n = 1; n < N; ++n) {
      f32x4 more[QT][NM];
      qk_tile<K, DP, QT, NM>(tile, fr[n], more, g, p);
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int m = 0; m < NM; ++m) acc[qt][m] += more[qt][m];
    }
  }
}

template <typename T, int DP, int NW> struct Tile4 {
  using K = typename Pieces<T>::K;
  static constexpr int KC = 64, NT = NW * 64, CPR = DP / 8, TILE = KC * DP * 2, STAGE = 2 * TILE, LDS = 2 * STAGE;
  static constexpr int BYTES = KC * DP / NT, LB = BYTES < 16 ? BYTES : 16, NL = BYTES / LB;  // codes of a thread: NL loads of LB bytes
  static constexpr int UPR = DP / 2 / LB;                                                    // loads of a row
  static_assert(LDS <= 160 * 1024, "LDS");
};

template <typename T, int DP, int NW, int QT>
__global__ __launch_bounds__(NW * 64) void cache4_tile_kernel(Cache4Args c4) {
  using C = Tile4<T, DP, NW>;
  using K = typename C::K;
  constexpr int KC = C::KC, NM = KC / 16, N = Pieces<T>::Q;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const CacheArgs &a = c4.a;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, p = lane & 15;
  const int tr = a.tr_own;
  // (the last tokens' tiles see the most keys: they start first)
  const uint32_t per = (uint32_t)(a.Hkv * a.np_own * a.B), u0 = blockIdx.x % per;
  const int tile = a.rt_own - 1 - (int)(blockIdx.x / per), hk = u0 / a.np_own % a.Hkv, b = u0 / a.np_own / a.Hkv, split = u0 % a.np_own;
  RowInfo ri[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    ri[qt] = row_info(a, b, hk, tile * tr + (w * QT + qt) * 16 + p);
    ri[qt].valid = ri[qt].valid && (w * QT + qt) * 16 < tr;
  }
  int keys, low;  // keys that any row sees; below `low` every row of the wave sees every key
  own_bounds(a, b, tile * tr, min(tile * tr + tr, a.TG), keys, low);
  const int r0 = tile * tr + w * QT * 16;
  if (w > 0 && r0 < a.TG) {
    int k;
    own_bounds(a, b, r0, a.TG, k, low);
    low = min(low, keys);
  }
  const int64_t slot = ((((int64_t)b * a.Hkv + hk) * a.rt_own + tile) * a.np_own + split) * tr;
  int c0, c1;
  share_of((keys + KC - 1) / KC, split, a.np_own, c0, c1);

  RowFrag<K, DP> fr[N][QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt)
#pragma unroll
    for (int ks = 0; ks < DP / 32; ++ks) {
      s16x8 x[N];
      load_q8<T>(a, (const T *)a.q + ri[qt].b * a.sq[0] + ri[qt].hq * a.sq[1] + ri[qt].t * a.sq[2], 32 * ks + 8 * g, x);
#pragma unroll
      for (int n = 0; n < N; ++n) fr[n][qt].h[ks] = x[n];
    }

  // this thread's loads: row, tensor (keys, then values; the same across a wave), place in the row
  int row[C::NL], place[C::NL];
  uint32_t off[C::NL], cw[C::NL][C::LB / 4];
  float st[C::NL];
  bool val[C::NL];
#pragma unroll
  for (int n = 0; n < C::NL; ++n) {
    const int u = n * C::NT + tid, last = a.D / 2 / C::LB - 1, c = u % C::UPR;
    val[n] = u / (KC * C::UPR);
    row[n] = u / C::UPR % KC;
    place[n] = c;
    off[n] = (uint32_t)(row[n] * (val[n] ? a.sv[2] : a.sk[2]) + (c < last ? c : last) * C::LB);
  }
  const char *kb = (const char *)a.k + b * a.sk[0] + hk * a.sk[1], *vb = (const char *)a.v + b * a.sv[0] + hk * a.sv[1];
  const uint16_t *sb = c4.step + b * c4.ss[0] + hk * c4.ss[1];
  auto load = [&](int c) {
    const uint32_t row0 = (uint32_t)c * KC;
#pragma unroll
    for (int n = 0; n < C::NL; ++n) {
      const int64_t step = val[n] ? a.sv[2] : a.sk[2];
      const uint32_t lim = tail_limit<KC>(row0, keys, (uint32_t)step, (uint32_t)a.D / 2) == 0xffffffffu ? 0xffffffffu
                                                                                                       : (uint32_t)((keys - 1 - row0) * step + a.D / 2 - C::LB);
      const char *src = (val[n] ? vb : kb) + row0 * step + (off[n] > lim ? lim : off[n]);
      if constexpr (C::LB == 16) {
        const u32x4 y = *(const u32x4 *)src;
#pragma unroll
        for (int i = 0; i < 4; ++i) cw[n][i] = y[i];
      } else if constexpr (C::LB == 8) {
        const u32x2 y = *(const u32x2 *)src;
        cw[n][0] = y[0];
        cw[n][1] = y[1];
      } else {
        cw[n][0] = *(const uint32_t *)src;
      }
      const bool in = row0 + row[n] < (uint32_t)keys;
      const int j = min(place[n] * C::LB * 2 / kGroup4, c4.ng - 1);
      const uint16_t bits = sb[((int64_t)(in ? row0 + row[n] : keys - 1) * 2 + (val[n] ? 1 : 0)) * c4.ng + j];
      const float y = step_f32<T>(bits);
      st[n] = !in ? 0.f : val[n] ? fmaxf(y, 0.f) : y;  // (rows past the end are zeros; a value's NaN is its key's too)
    }
  };
  auto store = [&](int stage) {
#pragma unroll
    for (int n = 0; n < C::NL; ++n) {
      char *tl = smem + stage * C::STAGE + (val[n] ? C::TILE : 0) + row[n] * DP * 2;
#pragma unroll
      for (int i = 0; i < C::LB / 4; ++i)
        *(s16x8 *)(tl + ((place[n] * (C::LB / 4) + i) ^ swz(row[n], C::CPR)) * 16) = values8<K>(cw[n][i], st[n]);
    }
  };

  SoftmaxState<DP> sm[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) sm[qt].init();
  if (c0 < c1) {
    load(c0);
    store(0);
    if (c0 + 1 < c1) load(c0 + 1);
  }
  int stage = 0;
  for (int c = c0; c < c1; ++c) {
    lds_barrier();  // chunk c is written, and every wave has read chunk c - 1, whose place is filled next
    const char *Ks = smem + stage * C::STAGE, *Vs = Ks + C::TILE;
    stage ^= 1;
    if (c + 1 < c1) store(stage);
    if (c + 2 < c1) load(c + 2);
    if (w * QT * 16 >= tr) continue;
    f32x4 s[QT][NM];
    qk_pieces<K, DP, QT, NM, N>(Ks, fr, s, g, p);
    if ((c + 1) * (int64_t)KC > low) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) mask_keys<NM>(s[qt], (ri[qt].valid ? ri[qt].lim : keys) - c * KC, g);
    }
    float x[QT][NM][4];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) sm[qt].template step<NM>(s[qt], a.scale2, x[qt]);
    if constexpr (N == 1) {
      pv_tile<K, DP, KC, QT>(Vs, x, sm, g, p);
    } else {
      // (pieces cut off one after the other; what a product takes rounded is exact)
#pragma unroll
      for (int n = 0; n < N; ++n) {
        float y[QT][NM][4];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
          for (int m = 0; m < NM; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              y[qt][m][r] = n + 1 < N ? __uint_as_float(__float_as_uint(x[qt][m][r]) & 0xffff0000u) : x[qt][m][r];
              x[qt][m][r] -= y[qt][m][r];
            }
        pv_tile<K, DP, KC, QT>(Vs, y, sm, g, p);
      }
    }
  }

#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int i = (w * QT + qt) * 16 + p;
    if (i >= tr) continue;
    const float lt = sm[qt].total();
    if (a.direct) {
      if (tile * tr + i >= a.TG) continue;
      const float l = ri[qt].valid ? lt : 0.f, inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) store_row<T>(a, ri[qt], sm[qt].o[t], inv, 16 * t + 4 * g);
      if (g == 0 && a.lse) a.lse[((int64_t)ri[qt].b * a.Hq + ri[qt].hq) * a.T + ri[qt].t] = l == 0.f ? -INFINITY : (sm[qt].m + __log2f(l)) * kLn2;
      continue;
    }
    if (g == 0) a.stat[slot + i] = float2{sm[qt].m, lt};
    if (ri[qt].valid && lt != 0.f) {  // (a NaN sum is kept)
      float *dst = a.part + (slot + i) * DP;
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) *(f32x4 *)(dst + 16 * t + 4 * g) = sm[qt].o[t];
    }
  }
}

// ---- host ---------------------------------------------------------------------
struct Plan4 {
  int64_t DP, pitch, tr, rt, np, rows;
  bool few, quad;
  size_t part, total;
};
static Plan4 plan4(const fbsa_attn4_desc *d) {
  Plan4 p;
  const int64_t TG = d->T * (d->Hq / d->Hkv), seqs = d->B * d->Hkv;
  p.few = TG <= 16;
  p.DP = d->D <= 32 ? 32 : d->D <= 64 ? 64 : d->D <= 128 ? 128 : p.few && d->D <= 192 ? 192 : 256;
  p.pitch = p.DP == 192 ? 256 : p.DP;
  p.quad = TG <= 4 && (p.DP <= 64 || (p.DP == 128 && d->dtype != FBSA_F32));
  p.tr = p.quad ? 4 : p.few ? 16 : tile_rows(d->dtype, TG);
  p.rt = cdiv(TG, p.tr);
  const int64_t tiles = seqs * p.rt, room = kCUs * (p.DP <= 128 ? 2 : 1);
  const int64_t want = p.few ? cdiv((p.DP >= 192 ? 4 : 8) * kCUs, tiles) : d->B > 1 ? cdiv(4 * room, tiles) : tiles >= room ? 1 : room / tiles;
  p.np = std::max<int64_t>(1, std::min({want, cdiv(d->S, p.few ? 64 : 128), (int64_t)kMaxShares / 2}));
  p.rows = tiles * p.np * p.tr;
  const size_t parts = p.np == 1 ? 0 : (size_t)p.rows;
  p.part = up256(parts * 8);
  p.total = p.part + up256(parts * p.pitch * 4);
  if (p.total == 0) p.total = 256;  // (0 says that a descriptor is refused)
  return p;
}

template <typename T, int DP, bool QUAD> static int launch_part4(const Cache4Args &c, int64_t wgs, hipStream_t s) {
  constexpr size_t lds = (size_t)Part4<DP>::NS * Part4<DP>::STAGE;
  const int e = lds_optin((const void *)cache4_part_kernel<T, DP, QUAD>, lds, "hipFuncSetAttribute(cache4_part)");
  if (e) return e;
  hipLaunchKernelGGL((cache4_part_kernel<T, DP, QUAD>), dim3((unsigned)wgs), dim3(64), lds, s, c);
  return hip_check(hipGetLastError(), "cache4_part_kernel launch");
}
template <typename T, int DP, int NW, int QT> static int launch_tile4(const Cache4Args &c, int64_t wgs, hipStream_t s) {
  using C = Tile4<T, DP, NW>;
  const int e = lds_optin((const void *)cache4_tile_kernel<T, DP, NW, QT>, C::LDS, "hipFuncSetAttribute(cache4_tile)");
  if (e) return e;
  hipLaunchKernelGGL((cache4_tile_kernel<T, DP, NW, QT>), dim3((unsigned)wgs), dim3(NW * 64), C::LDS, s, c);
  return hip_check(hipGetLastError(), "cache4_tile_kernel launch");
}
template <typename T, int DP> static int launch_attn4(const Cache4Args &c, const Plan4 &pl, hipStream_t s) {
  const int64_t wgs = (int64_t)c.a.B * c.a.Hkv * pl.rt * pl.np;
  if constexpr (DP <= 64 || (DP == 128 && sizeof(T) == 2)) {
    if (pl.quad) return launch_part4<T, DP, true>(c, wgs, s);
  }
  if (pl.few) return launch_part4<T, DP, false>(c, wgs, s);
  if constexpr (DP != 192) {
    if (pl.tr <= 64) return launch_tile4<T, DP, 4, 1>(c, wgs, s);
    if constexpr (sizeof(T) == 2) {
      constexpr int NW = DP == 32 ? 4 : 8;
      return launch_tile4<T, DP, NW, 8 / NW>(c, wgs, s);
    }
  }
  return fail(FBSA_EUNSUPPORTED, "fbsa_cache4_attn: no kernel");
}
template <typename T> static int dispatch_attn4(const Cache4Args &c, const Plan4 &pl, hipStream_t s) {
  switch (pl.DP) {
    case 32: return launch_attn4<T, 32>(c, pl, s);
    case 64: return launch_attn4<T, 64>(c, pl, s);
    case 128: return launch_attn4<T, 128>(c, pl, s);
    case 192: return launch_attn4<T, 192>(c, pl, s);
    default: return launch_attn4<T, 256>(c, pl, s);
  }
}

static bool aligned_to(const void *p, int64_t n) { return (uintptr_t)p % (uintptr_t)n == 0; }

// strides of codes (bytes) and steps, shared by the three entry points
static int check_held(const char *fn, int64_t D, const int64_t *sk4, const int64_t *sv4, const int64_t *ss) {
  if (D < 32 || D > 256 || D % 32) return fail(FBSA_EUNSUPPORTED, "%s: head dim %lld is not a multiple of 32 up to 256", fn, (long long)D);
  for (int x = 0; x < 3; ++x)
    if (sk4[x] < 0 || sv4[x] < 0 || sk4[x] % 16 || sv4[x] % 16)
      return fail(FBSA_EINVAL, "%s: strides of the codes must be non-negative multiples of 16 bytes", fn);
  // (64 rows are addressed with 32-bit offsets from the first)
  if (sk4[2] >= 1LL << 26 || sv4[2] >= 1LL << 26) return fail(FBSA_EUNSUPPORTED, "%s: a row stride of the codes is 64 MiB or more", fn);
  if (ss[0] < 0 || ss[1] < 0 || ss[0] % 2 || ss[1] % 2) return fail(FBSA_EINVAL, "%s: strides of the steps must be even and not negative", fn);
  return FBSA_OK;
}

static int check_rows4(const char *fn, const fbsa_rows4_desc *d) {
  if (!d) return fail(FBSA_EINVAL, "%s: null descriptor", fn);
  if (d->dtype < FBSA_F32 || d->dtype > FBSA_F16) return fail(FBSA_EINVAL, "%s: bad dtype %d", fn, d->dtype);
  if (d->flags) return fail(FBSA_EINVAL, "%s: unknown flags 0x%x", fn, d->flags);
  if (d->B < 1 || d->H < 1 || d->T < 1 || d->S < 1)
    return fail(FBSA_EINVAL, "%s: sizes must be positive (B=%lld H=%lld T=%lld S=%lld)", fn, (long long)d->B, (long long)d->H, (long long)d->T, (long long)d->S);
  const int64_t lim = 0x7fff0000LL;
  if (d->S > lim || d->T > lim || d->B > lim || d->H > 65535 || d->B * d->H > 65535)
    return fail(FBSA_EUNSUPPORTED, "%s: sizes exceed the grid or 32-bit row indices", fn);
  const int e = check_held(fn, d->D, d->sk4, d->sv4, d->ss);
  if (e) return e;
  const int64_t es = d->dtype == FBSA_F32 ? 4 : 2;
  for (int x = 0; x < 3; ++x)
    if (d->sk[x] < 0 || d->sv[x] < 0 || d->sk[x] * es % 16 || d->sv[x] * es % 16)
      return fail(FBSA_EINVAL, "%s: strides of the rows must be non-negative multiples of 16 bytes", fn);
  // (2 lanes' groups of up to 32 to a row, fewer than 2^32 threads)
  if (d->B * d->H * d->T > 0x3ff0000LL) return fail(FBSA_EUNSUPPORTED, "%s: grid too large", fn);
  return FBSA_OK;
}

static int check_attn4(const fbsa_attn4_desc *d) {
  static const char *fn = "fbsa_cache4_attn";
  if (!d) return fail(FBSA_EINVAL, "%s: null descriptor", fn);
  if (d->dtype < FBSA_F32 || d->dtype > FBSA_F16) return fail(FBSA_EINVAL, "%s: bad dtype %d", fn, d->dtype);
  if (d->flags) return fail(FBSA_EINVAL, "%s: unknown flags 0x%x", fn, d->flags);
  if (d->B < 1 || d->Hq < 1 || d->Hkv < 1 || d->T < 1 || d->S < 1)
    return fail(FBSA_EINVAL, "%s: sizes must be positive (B=%lld Hq=%lld Hkv=%lld T=%lld S=%lld)", fn, (long long)d->B, (long long)d->Hq,
                (long long)d->Hkv, (long long)d->T, (long long)d->S);
  if (d->Hq % d->Hkv) return fail(FBSA_EINVAL, "%s: Hq=%lld not a multiple of Hkv=%lld", fn, (long long)d->Hq, (long long)d->Hkv);
  if (!isfinite(d->scale * kLog2e)) return fail(FBSA_EINVAL, "%s: scale times log2(e) is not finite", fn);
  const int64_t lim = 0x7fff0000LL;
  if (d->S > lim || d->B > lim || d->Hq > 65535 || d->T > lim || d->T * (d->Hq / d->Hkv) > lim || d->B > lim / d->Hq ||
      d->B * d->Hq > lim / d->T || d->B * d->Hkv > 65535)
    return fail(FBSA_EUNSUPPORTED, "%s: sizes exceed the grid or 32-bit row indices", fn);
  const int e = check_held(fn, d->D, d->sk4, d->sv4, d->ss);
  if (e) return e;
  const int64_t es = d->dtype == FBSA_F32 ? 4 : 2;
  for (int x = 0; x < 3; ++x)
    if (d->sq[x] < 0 || d->so[x] < 0 || d->sq[x] * es % 16 || d->so[x] * es % 16)
      return fail(FBSA_EINVAL, "%s: strides of q and o must be non-negative multiples of 16 bytes", fn);
  // (fewer than 2^32 threads: up to 512 a tile and share, 64 or 256 a row that is joined)
  const Plan4 pl = plan4(d);
  if (pl.rows > lim || d->B * d->Hq * d->T > 0x3ff0000LL || d->B * d->Hkv * pl.rt * pl.np > 0x7f0000LL)
    return fail(FBSA_EUNSUPPORTED, "%s: grid too large", fn);
  return FBSA_OK;
}

static void fill_rows4(Rows4Args &a, const fbsa_rows4_desc *d) {
  for (int x = 0; x < 3; ++x) { a.sk4[x] = d->sk4[x]; a.sv4[x] = d->sv4[x]; a.sk[x] = d->sk[x]; a.sv[x] = d->sv[x]; }
  a.ss[0] = d->ss[0]; a.ss[1] = d->ss[1];
  a.B = (int)d->B; a.H = (int)d->H; a.T = (int)d->T; a.S = (int)d->S; a.D = (int)d->D; a.ng = (int)cdiv(d->D, kGroup4);
}
template <typename T, int LPR> static int launch_rows4(const Rows4Args &a, bool read, hipStream_t s) {
  const unsigned wgs = (unsigned)cdiv((int64_t)a.B * a.H * a.T, 256 / (2 * LPR));
  if (read) hipLaunchKernelGGL((cache4_read_kernel<T, LPR>), dim3(wgs), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((cache4_append_kernel<T, LPR>), dim3(wgs), dim3(256), 0, s, a);
  return hip_check(hipGetLastError(), read ? "cache4_read_kernel launch" : "cache4_append_kernel launch");
}
template <typename T> static int rows4_of(const Rows4Args &a, bool read, hipStream_t s) {
  if (a.D <= 32) return launch_rows4<T, 4>(a, read, s);
  if (a.D <= 64) return launch_rows4<T, 8>(a, read, s);
  if (a.D <= 128) return launch_rows4<T, 16>(a, read, s);
  return launch_rows4<T, 32>(a, read, s);
}
static int run_rows4(const Rows4Args &a, int dtype, bool read, hipStream_t s) {
  return dtype == FBSA_BF16 ? rows4_of<bf16>(a, read, s) : dtype == FBSA_F16 ? rows4_of<f16>(a, read, s) : rows4_of<float>(a, read, s);
}
static int check_pointers4(const char *fn, const void *k4, const void *v4, const void *step, const void *k, const void *v,
                           const int32_t *first, const int32_t *count) {
  if (!k4 || !v4 || !step || !k || !v) return fail(FBSA_EINVAL, "%s: null tensor pointer", fn);
  if (!aligned_to(k4, 16) || !aligned_to(v4, 16) || !aligned_to(k, 16) || !aligned_to(v, 16))
    return fail(FBSA_EINVAL, "%s: tensors must be 16-byte aligned", fn);
  if (!aligned_to(step, 4) || !aligned_to(first, 4) || !aligned_to(count, 4)) return fail(FBSA_EINVAL, "%s: steps, places or counts misaligned", fn);
  return FBSA_OK;
}

}  // namespace fbsa

using namespace fbsa;

extern "C" {

int fbsa_cache4_append(const fbsa_rows4_desc *d, void *k4, void *v4, void *step, const void *k_new, const void *v_new, const int32_t *start,
                       const int32_t *count, void *stream) {
  int e = check_rows4("fbsa_cache4_append", d);
  if (e || (e = check_pointers4("fbsa_cache4_append", k4, v4, step, k_new, v_new, start, count))) return e;
  if (!start) return fail(FBSA_EINVAL, "fbsa_cache4_append: null tensor pointer");
  Rows4Args a = {};
  fill_rows4(a, d);
  a.k4 = k4; a.v4 = v4; a.step = (uint16_t *)step; a.k = (void *)k_new; a.v = (void *)v_new; a.first = start; a.count = count;
  return run_rows4(a, d->dtype, false, (hipStream_t)stream);
}

int fbsa_cache4_read(const fbsa_rows4_desc *d, const void *k4, const void *v4, const void *step, const int32_t *first, const int32_t *count,
                     void *k, void *v, void *stream) {
  int e = check_rows4("fbsa_cache4_read", d);
  if (e || (e = check_pointers4("fbsa_cache4_read", k4, v4, step, k, v, first, count))) return e;
  Rows4Args a = {};
  fill_rows4(a, d);
  a.k4 = (void *)k4; a.v4 = (void *)v4; a.step = (uint16_t *)step; a.k = k; a.v = v; a.first = first; a.count = count;
  return run_rows4(a, d->dtype, true, (hipStream_t)stream);
}

size_t fbsa_cache4_attn_workspace_bytes(const fbsa_attn4_desc *d) { return check_attn4(d) ? 0 : plan4(d).total; }

int fbsa_cache4_attn(const fbsa_attn4_desc *d, const void *q, const void *k4, const void *v4, const void *step, const int32_t *lens,
                     const int32_t *count, const void *out_gate, void *o, float *lse, void *workspace, size_t workspace_bytes, void *stream) {
  int e = check_attn4(d);
  if (e) return e;
  if (!q || !k4 || !v4 || !step || !lens || !o) return fail(FBSA_EINVAL, "fbsa_cache4_attn: null tensor pointer");
  const int64_t es = d->dtype == FBSA_F32 ? 4 : 2;
  if (!aligned_to(q, 16) || !aligned_to(k4, 16) || !aligned_to(v4, 16) || !aligned_to(o, 16))
    return fail(FBSA_EINVAL, "fbsa_cache4_attn: tensors must be 16-byte aligned");
  if (!aligned_to(step, 4) || !aligned_to(lens, 4) || !aligned_to(count, 4) || !aligned_to(lse, 4) || !aligned_to(out_gate, es))
    return fail(FBSA_EINVAL, "fbsa_cache4_attn: step/lens/count/lse/out_gate misaligned");
  const Plan4 pl = plan4(d);
  if (!workspace || workspace_bytes < pl.total)
    return fail(FBSA_EWORKSPACE, "fbsa_cache4_attn: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, pl.total);
  if (!aligned_to(workspace, 256)) return fail(FBSA_EINVAL, "fbsa_cache4_attn: workspace must be 256-byte aligned");
  Cache4Args c = {};
  CacheArgs &a = c.a;
  a.q = q; a.k = k4; a.v = v4; a.og = out_gate; a.o = o; a.lse = lse; a.lens = lens; a.count = count;
  c.step = (const uint16_t *)step;
  c.ss[0] = d->ss[0]; c.ss[1] = d->ss[1];
  c.ng = (int)cdiv(d->D, kGroup4);
  for (int x = 0; x < 3; ++x) { a.sq[x] = d->sq[x]; a.sk[x] = d->sk4[x]; a.sv[x] = d->sv4[x]; a.so[x] = d->so[x]; a.sog[x] = d->sog[x]; }
  a.B = (int)d->B; a.Hq = (int)d->Hq; a.Hkv = (int)d->Hkv; a.T = (int)d->T; a.S = (int)d->S; a.D = (int)d->D;
  a.G = (int)(d->Hq / d->Hkv); a.TG = a.T * a.G;
  a.tr_own = (int)pl.tr; a.tr_pre = 16; a.rt_own = (int)pl.rt; a.np_own = (int)pl.np;
  a.direct = pl.np == 1;
  a.scale2 = d->scale == 0.f ? 1.f : fabsf(d->scale) * kLog2e;
  a.qand = d->scale == 0.f ? 0u : 0xffffffffu;
  a.qxor = d->scale < 0.f ? (d->dtype == FBSA_F32 ? 0x80000000u : 0x80008000u) : 0u;
  a.stat = (float2 *)workspace; a.part = (float *)((char *)workspace + pl.part);
  hipStream_t s = (hipStream_t)stream;
  e = d->dtype == FBSA_BF16 ? dispatch_attn4<bf16>(c, pl, s) : d->dtype == FBSA_F16 ? dispatch_attn4<f16>(c, pl, s) : dispatch_attn4<float>(c, pl, s);
  return e || a.direct ? e : launch_cache_join(a, d->dtype, pl.pitch, s);
}

}  // extern "C"
