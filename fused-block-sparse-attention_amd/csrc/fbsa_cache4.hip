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
// Attention: rows and tiles as in the cache of 16 and 32 bits (fbsa_cache.hip); the shares
// of the keys are formed on the device from the sequences' lengths.
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

// The largest magnitude of a group's N lanes (4 or 8)
template <int N> __device__ __forceinline__ float group_max(float x) {
  auto with = [&](auto CTRL) {
    const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(CTRL)::value, 0xf, 0xf, false);
    x = fmaxf(x, __builtin_bit_cast(float, y));
  };
  with(std::integral_constant<int, 0xb1>{});                         // lane ^ 1
  with(std::integral_constant<int, 0x4e>{});                         // lane ^ 2
  if constexpr (N >= 8) with(std::integral_constant<int, 0x141>{});  // 7 - lane of eight
  return x;
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
// The codes of 8 elements: x / step goes to the converter, which rounds to the nearest
// code, ties to the even one, and saturates; what matters is that a quotient on a border
// is formed as the border and one beside it is not. With step = m 2^e, 1 <= m <= 63/32:
// z = x 2^-e exactly, t = z / m to a unit in the last place, and t + (z - t m) / m is
// within 0.5 + 2^-20 units of the quotient (the residual is exact). A quotient beside a
// border c (c m has 9 bits, z 24) is at least 1 / m >= 0.507 units from it, one on it is exact.
__device__ __forceinline__ uint32_t codes_of(const float (&y)[8], float step) {
  if (!(step > 0.f)) return 0;  // (zeros, and rows held as NaN)
  const uint32_t bits = __float_as_uint(step);
  const float m = __uint_as_float((bits & 0x007fffffu) | 0x3f800000u), pw = __uint_as_float((254u << 23) - (bits & 0x7f800000u)), r = 1.f / m;
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float z = y[i] * pw, t = z * r;
    q[i] = __builtin_fmaf(__builtin_fmaf(-t, m, z), r, t);
  }
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[0], q[1], 1.f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[2], q[3], 1.f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[4], q[5], 1.f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[6], q[7], 1.f, 3);
}

// Rows of a block: EL elements a lane, LPR lanes to a key or value row and the two side by
// side, RPB rows at a time, U times.
template <int EL_, int LPR> struct Rows4 {
  static constexpr int EL = EL_, RPB = 256 / (2 * LPR), U = 4;
};

// New rows: key and value of a row side by side, so that all its lanes know of a NaN or
// an infinity in either. Bound by memory, long prompts: 65531 fp32 rows of 8 heads, d 96,
// 94 us, 4.9 TB/s (four elements a lane, whole lines a load, 112: codes leave two bytes at
// a time); a step's rows by latency, 3 us.
template <typename T, int LPR> __global__ __launch_bounds__(256) void cache4_append_kernel(Rows4Args a) {
  using C = Rows4<8, LPR>;
  const int tid = threadIdx.x, lane = tid & 63, which = (tid / LPR) & 1, e = tid % LPR;  // key or value; elements 8 e ...
  const int h = (int)(blockIdx.y % (uint32_t)a.H), b = (int)(blockIdx.y / (uint32_t)a.H);
  const int t0 = blockIdx.x * (C::RPB * C::U) + tid / (2 * LPR), first = a.first[b], count = min(a.count ? a.count[b] : a.T, a.T);
  const int64_t *st = which ? a.sv : a.sk, *s4 = which ? a.sv4 : a.sk4;
  const T *src = (const T *)(which ? a.v : a.k) + b * st[0] + h * st[1] + 8 * e;
  const int64_t tstep = st[2];
  float y[C::U][8];
  bool live[C::U];
#pragma unroll
  for (int i = 0; i < C::U; ++i) {
    const int t = t0 + i * C::RPB;
    const int64_t at = (int64_t)first + t;
    live[i] = 8 * e < a.D && t < count && at >= 0 && at < a.S;
#pragma unroll
    for (int j = 0; j < 8; ++j) y[i][j] = 0.f;
    if (live[i]) {
      if constexpr (sizeof(T) == 4) {
        const f32x4 p = ((const f32x4 *)(src + t * tstep))[0], q = ((const f32x4 *)(src + t * tstep))[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) { y[i][j] = p[j]; y[i][4 + j] = q[j]; }
      } else {
        const s16x8 p = *(const s16x8 *)(src + t * tstep);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[i][j] = to_f32<T>(__builtin_bit_cast(T, (short)p[j]));
      }
    }
  }
  char *dst = (char *)(which ? a.v4 : a.k4) + b * s4[0] + h * s4[1] + 4 * e;
  const int64_t rstep = s4[2];
  uint16_t *sd = a.step + b * a.ss[0] + h * a.ss[1] + which * a.ng + e / 8;
#pragma unroll
  for (int i = 0; i < C::U; ++i) {
    float most = 0.f, sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      most = fmaxf(most, fabsf(y[i][j]));       // (passes NaN over)
      sum = __builtin_fmaf(y[i][j], 0.f, sum);  // 0, or NaN
    }
    const uint64_t vote = __ballot(sum != 0.f);
    constexpr uint64_t ROW = LPR == 32 ? ~0ull : (1ull << (2 * LPR % 64)) - 1;
    const bool bad = (vote >> (lane / (2 * LPR) * (2 * LPR)) & ROW) != 0;
    most = group_max<(LPR < 8 ? LPR : 8)>(most);
    if (!live[i]) continue;
    const float step = bad ? __uint_as_float(0x7fc00000u) : step_of<T>(most);
    const int64_t at = (int64_t)first + t0 + i * C::RPB;
    *(uint32_t *)(dst + at * rstep) = codes_of(y[i], step);
    if (e % 8 == 0) {
      if constexpr (__is_same(T, f16)) sd[at * 2 * a.ng] = __builtin_bit_cast(uint16_t, (f16)step);
      else sd[at * 2 * a.ng] = (uint16_t)(__float_as_uint(step) >> 16);
    }
  }
}

// Rows first[b] + t of each sequence as numbers of type T; rows outside the cache, and
// those from count[b] on, are zeros. 16 bytes of values a lane, so that a store is whole
// lines, past the caches (nothing here reads them again): 262144 bf16 rows of 8 heads, d
// 64, 119 us, 5.7 TB/s, 126 with ordinary stores.
template <typename T, int LPR> __global__ __launch_bounds__(256) void cache4_read_kernel(Rows4Args a) {
  using C = Rows4<16 / sizeof(T), LPR>;
  constexpr int EL = C::EL, RPB = C::RPB, U = C::U;
  const int tid = threadIdx.x, which = (tid / LPR) & 1, e = tid % LPR;
  const int h = (int)(blockIdx.y % (uint32_t)a.H), b = (int)(blockIdx.y / (uint32_t)a.H);
  if (EL * e >= a.D) return;
  const int t0 = blockIdx.x * (RPB * U) + tid / (2 * LPR), first = a.first ? a.first[b] : 0, count = a.count ? a.count[b] : a.T;
  const int64_t *st = which ? a.sv : a.sk, *s4 = which ? a.sv4 : a.sk4;
  const char *src = (const char *)(which ? a.v4 : a.k4) + b * s4[0] + h * s4[1] + EL / 2 * e;
  const int64_t rstep = s4[2], tstep = st[2];
  const uint16_t *sd = a.step + b * a.ss[0] + h * a.ss[1] + which * a.ng + e / (kGroup4 / EL);
  uint32_t w[U], s[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int t = t0 + i * RPB;
    const int64_t at = (int64_t)first + t;
    w[i] = s[i] = 0;
    if (t < count && at >= 0 && at < a.S) {
      w[i] = EL == 8 ? *(const uint32_t *)(src + at * rstep) : *(const uint16_t *)(src + at * rstep);
      s[i] = sd[at * 2 * a.ng];
    }
  }
  T *dst = (T *)(which ? a.v : a.k) + b * st[0] + h * st[1] + EL * e;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int t = t0 + i * RPB;
    if (t >= a.T) continue;
    const float step = step_f32<T>(s[i]);
    if constexpr (sizeof(T) == 4) {
      const f32x2 x = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.f, 0), y = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.f, 1);
      __builtin_nontemporal_store(f32x4{x[0] * step, x[1] * step, y[0] * step, y[1] * step}, (f32x4 *)(dst + t * tstep));
    } else {
      __builtin_nontemporal_store(values8<T>(w[i], step), (s16x8 *)(dst + t * tstep));
    }
  }
}

// ---- attention ----------------------------------------------------------------
struct Cache4Args {
  CacheArgs a;           // k, v: the codes; sk, sv in bytes
  const uint16_t *step;
  int64_t ss[2];
  int32_t ng;            // steps of a key or value row
  int32_t want;          // shares that a KV head's chunks are cut into
  int2 *used;            // a tile's first share and its number of them (several tiles to a KV head)
};

// An address that is the same on every lane, in scalar registers from here on: without the
// empty statements the compiler keeps what it forms with 64-bit products in vector registers
// and reads it back for each load (one token over 32 sequences, d 256: 28 us so, 45 without).
__device__ __forceinline__ const char *uniform(const char *x) {
  uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)((uintptr_t)x >> 32));
  asm("" : "+s"(lo));
  asm("" : "+s"(hi));
  return (const char *)(uintptr_t)((uint64_t)hi << 32 | lo);
}
// 4 bytes a lane to LDS, as g2lds16_s its 16 (the asm has m0 as a register it writes)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void g2lds4_s(const void *sbase, unsigned voff, void *lds_wave_base) {
  const unsigned m = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)lds_wave_base);
  const uint64_t bp = (uint64_t)(uintptr_t)sbase;
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((unsigned)(bp >> 32));
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((unsigned)bp);
  const uint64_t sb = ((uint64_t)hi << 32) | (uint64_t)lo;
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" : : "v"(voff), "s"(sb), "s"(m) : "memory", "m0");
}
#pragma clang diagnostic pop

template <typename N> __device__ __forceinline__ N wave_sum(N x) {
  auto with = [&](auto CTRL) { x += __builtin_bit_cast(N, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(CTRL)::value, 0xf, 0xf, false)); };
  with(std::integral_constant<int, 0xb1>{});   // lane ^ 1
  with(std::integral_constant<int, 0x4e>{});   // lane ^ 2
  with(std::integral_constant<int, 0x141>{});  // 7 - lane of eight
  with(std::integral_constant<int, 0x140>{});  // 15 - lane of sixteen
  x += __shfl_xor(x, 16, 64);
  x += __shfl_xor(x, 32, 64);
  return __builtin_bit_cast(N, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}
// sums of lanes 0 .. lane
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // one lane to the right, of sixteen
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // the last of sixteen to the next sixteen
  return x + __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
}
// Share i of a KV head's chunks, which are cut into pieces of about the same number: tile
// (numbered from the one that sees the most keys on, the sequences of a place side by
// side), piece, number of pieces and of the tile's first one. The lengths are on the
// device, so every wave counts (the same number of pieces for each leaves the longest
// sequence's to end last: 3 sequences of 2000 to 30000 rows, 200 tokens, 2 heads over 1, d
// 256: 58.7 us against 43.7; 4 of 1000 to 16000, 128 tokens, 16 over 2, d 128: 78 against
// 72). False: there is none.
__device__ __forceinline__ int chunks4(const CacheArgs &a, int u) {
  if (u >= a.B * a.rt_own) return 0;
  const int tile = a.rt_own - 1 - u / a.B, b = a.rt_own == 1 ? u : u % a.B;
  const int n = seq_len(a, b), c = seq_count(a, b);
  if (a.rt_own == 1) return c > 0 ? (int)(((uint32_t)n + 63u) / 64u) : 0;
  const int real = min(tile * a.tr_own + a.tr_own, c * a.G);
  if (tile * a.tr_own >= real) return 0;
  const int64_t keys = (int64_t)n - c + (real - 1) / a.G + 1;  // (own_bounds)
  return keys < 0 ? 0 : (int)((keys + 63) / 64);
}
// FIT: pieces of LEAST chunks or more, in `want` of them, which run at a time. Where there
// are more tiles than half of that, what is a quarter longer than a place's share of the
// chunks is cut, the others stay whole (16 sequences, 512 tokens, 8 heads over 1, d 128: one
// of 30000 rows and 15 of 1000 211 us against 1205 uncut, all of 4000 210 against 184). A
// quarter is between the two: at none (1.0 for 0.8) those of 4000 take 244, lengths of 1000
// to 30000 889 us in place of 937; at two thirds (0.6) 206 and 1063.
// Otherwise each tile may round its own up.
template <bool FIT, int LEAST> __device__ __forceinline__ bool share4(const Cache4Args &c4, int i, int lane, int &u, int &split, int &np, int &before) {
  const CacheArgs &a = c4.a;
  const int units = a.B * a.rt_own;
  if (units == 1) {
    u = 0; split = i; np = a.np_own; before = 0;
    return i < np;
  }
  if (a.direct) {
    u = i; split = 0; np = 1; before = i;
    return i < units;
  }
  const int one = chunks4(a, lane);  // (of most calls, all there are)
  auto chunks = [&](int u0) { return u0 ? chunks4(a, u0 + lane) : one; };
  int each;
  if constexpr (FIT) {
    float total = 0.f;  // (near enough, as is half a piece a tile for the rounding: the count below tells)
    for (int u0 = 0; u0 < units; u0 += 64) total += (float)chunks(u0);
    const bool fit = 2 * units <= c4.want;
    const int most = fit ? c4.want : c4.want + units;
    each = max(LEAST, (int)(wave_sum(total) / (fit ? (float)c4.want - 0.5f * (float)units : 0.8f * (float)c4.want)));
    for (;; each += 1 + each / 16) {  // (ends: one piece a tile is no more than `most`)
      int pieces = 0;
      for (int u0 = 0; u0 < units; u0 += 64) pieces += u0 + lane < units ? max(1, (chunks(u0) + each - 1) / each) : 0;
      if (wave_sum(pieces) <= most) break;
    }
  } else {
    int total = 0;  // (below 2^31: check_attn4)
#pragma unroll 4
    for (int u0 = 0; u0 < units; u0 += 64) total += chunks(u0);
    each = max(LEAST, (wave_sum(total) + c4.want - 1) / c4.want);
  }
  before = 0;
  for (int u0 = 0; u0 < units; u0 += 64) {
    const int mine = u0 + lane < units ? max(1, (chunks(u0) + each - 1) / each) : 0;
    const int upto = wave_scan(mine);
    const uint64_t past = __ballot(before + upto > i);
    if (past) {
      const int l = __builtin_ctzll(past);
      u = u0 + l;
      np = __builtin_amdgcn_readlane(mine, l);
      before += __builtin_amdgcn_readlane(upto, l) - np;
      split = i - before;
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// ---- softmax -----------------------------------------------------------------
// SoftmaxState's step for scores of any size. The largest of a row is a rounded product
// with the scale, and the product within an fma is not: from 2^28 on the two are up to 16
// apart, which is more than exponentials in fp16 have room for, and from 2^31 on more than
// 32-bit ones do (all of a row were 0 or infinite). There neighbouring scores are 16 apart
// or more, too, so all the weight is the largest's; such a row's scale is the next power
// of two, whose products are exact: its largest is the reference.
constexpr float kFar4 = 0x1p28f;
__device__ __forceinline__ float far_scale(float scale2) { return __uint_as_float((__float_as_uint(scale2) + 0x7fffffu) & 0xff800000u); }
// ROWS < 16: a row's scores are in lane columns ROWS apart too, and share its reference.
// scale: the row's, scale2 at first. UP: the reference is 2^UP below the largest, for
// exponentials that fp16 is to hold: at UP = 7 a probability loses bits from 2^-21 on and
// is 0 from 2^-32 on (2^-14 and 2^-25 at 0, which many small ones beside a large one came
// to). They reach 2^14, and with the products' roundings 2^15 (a rounding of 4 or 8 goes
// with scores and references that are multiples of 8 or 16), below fp16's 2^16.
template <int NM, int ROWS, int UP, int DP>
__device__ __forceinline__ void softmax4(SoftmaxState<DP> &sm, float &scale, const f32x4 (&s)[NM], float scale2, float (&x)[NM][4]) {
  constexpr float TAU = UP ? 14.f : SoftmaxState<DP>::TAU;
  float mx = -INFINITY;
#pragma unroll
  for (int k = 0; k < NM; ++k) mx = fmaxf(mx, fmaxf(fmaxf(s[k][0], s[k][1]), fmaxf(s[k][2], s[k][3])));
  if (__ballot(mx * scale - sm.m > TAU)) {
    float mc = fmaxf(mx, shfl_xor_f(mx, 16));
    mc = fmaxf(mc, shfl_xor_f(mc, 32));
#pragma unroll
    for (int y = ROWS; y < 16; y <<= 1) mc = fmaxf(mc, shfl_xor_f(mc, y));
    if (mc * scale - sm.m > TAU) {
      scale = fabsf(mc * scale2) >= kFar4 ? far_scale(scale2) : scale2;
      mc = mc * scale - (float)UP;
      const float alpha = __builtin_amdgcn_exp2f(sm.m - mc);
      sm.l *= alpha;
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) sm.o[t] *= alpha;
      sm.m = mc;
    }
  }
  const float ref = sm.m == -INFINITY ? 0.f : sm.m;
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < NM; ++k)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[k][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k][r], scale, -ref));
      sum += x[k][r];
    }
  sm.l += sum;
}
// a row's normaliser in natural logarithms, of its reference and sum
__device__ __forceinline__ float lse4(float scale2, float m, float l) {
  if (fabsf(m) >= kFar4) m *= scale2 / far_scale(scale2);
  return l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

// Queries and probabilities enter the products as sums of 16-bit numbers: a 32-bit number
// is three bf16 exactly (8 bits each).
template <typename T> struct Pieces {
  using K = bf16;                                                   // the product's type
  static constexpr int Q = 1, P = 2;
};
template <> struct Pieces<f16> { using K = f16; static constexpr int Q = 1, P = 2; };
template <> struct Pieces<float> { using K = bf16; static constexpr int Q = 3, P = 3; };

// x as N bf16 numbers, each what the ones before leave (the last rounded, the others cut).
// INF: numbers that may be infinite, which leave nothing (inf - inf is NaN, and made
// queries NaN whose every score is -inf)
template <int N, bool INF = false> __device__ __forceinline__ void split8(const float *x, s16x8 *out) {
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
      const bool ia = INF && fabsf(r[2 * j]) == INFINITY, ib = INF && fabsf(r[2 * j + 1]) == INFINITY;
      r[2 * j] = ia ? 0.f : r[2 * j] - __uint_as_float(a & 0xffff0000u);
      r[2 * j + 1] = ib ? 0.f : r[2 * j + 1] - __uint_as_float(b & 0xffff0000u);
    }
    out[n] = __builtin_bit_cast(s16x8, hw);
  }
  out[N - 1] = pack8<bf16>(r);
}
// elements d .. d + 7 of a query row (zeros past the head dim, or where `in` says), the scale's sign applied
// and of 32-bit ones the largest magnitude so far
template <typename T, bool INF> __device__ __forceinline__ void load_q8(const CacheArgs &a, const T *row, int d, bool in, s16x8 *out, float &top) {
  u32x4 w[sizeof(T) / 2];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
    w[i] = u32x4{0, 0, 0, 0};
    if (in && d < a.D) w[i] = ((const u32x4 *)(row + d))[i];
    if (a.qand != 0xffffffffu || a.qxor) {  // (a scale below or of zero)
#pragma unroll
      for (int e = 0; e < 4; ++e) w[i][e] = (w[i][e] & a.qand) ^ a.qxor;
    }
  }
  if constexpr (sizeof(T) == 4) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e / 4][e % 4]);
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
    split8<3, INF>(x, out);
  } else {
    out[0] = __builtin_bit_cast(s16x8, w[0]);
  }
}
// A wave's queries by `load`; 32-bit ones among which one is infinite a second time, with
// its pieces looked at (each looked at from the start costs short caches 12% of a call)
template <typename T, typename F> __device__ __forceinline__ void load_queries(F load) {
  float top = 0.f;
  load(std::false_type{}, top);
  if constexpr (sizeof(T) == 4) {
    if (__ballot(top == INFINITY)) load(std::true_type{}, top);
  }
}

// A chunk of 64 rows in LDS: keys' codes, values' codes, and steps twice. A row of codes
// is CPR units of 16 bytes, unit c at c ^ swk(row) (values: swv), which keeps the reads
// below off each other's banks as far as 16-byte units can: no two lanes on a bank for
// keys, two for values.
template <int DP> struct Part4 {
  static constexpr int KC = 64, RB = DP / 2, CPR = RB / 16, NG = DP <= kGroup4 ? 1 : DP / kGroup4;
  static constexpr int TILE = KC * RB, STEPS = KC * 4 * NG, LDS = 2 * TILE + 2 * STEPS;
  // Load i of a tile has rows RL i .. (six units to a row: no whole number of them), and
  // of the units' places only so many are different: number i % KV of keys, i / VD of values
  static constexpr int RL = 64 % CPR ? 0 : 64 / CPR, KV = CPR == 8 ? 2 : CPR == 6 ? 6 : 1, VD = CPR == 8 ? 2 : CPR <= 2 ? CPR : 1, VV = CPR / VD;
  __device__ static __forceinline__ int swk(int row) {
    return CPR == 1 ? 0 : CPR == 4 ? (row >> 2) & 3 : CPR == 8 ? (row >> 1) & 7 : (row >> 3) & 1;
  }
  __device__ static __forceinline__ int swv(int row) {
    return CPR == 1 ? 0 : CPR == 4 ? (row >> 4) & 3 : CPR == 8 ? ((row >> 4) & 3) | (row & 2) << 1 : (row >> 4) & 1;
  }
};

// Steps of four rows from `at` on (a multiple of 4): of group j of row r's key, or value
template <typename T, int NG> struct Steps4 {
  u32x4 w[NG];
  __device__ __forceinline__ void load(const char *steps, int at) {
#pragma unroll
    for (int i = 0; i < NG; ++i) w[i] = ((const u32x4 *)(steps + at * 4 * NG))[i];
  }
  __device__ __forceinline__ float key(int r, int j) const { return step_half<T>(w[(r * NG + j / 2) / 4][(r * NG + j / 2) % 4], j); }
  __device__ __forceinline__ float value(int r, int j) const { return step_half<T>(w[(r * NG + (NG + j) / 2) / 4][(r * NG + (NG + j) / 2) % 4], NG + j); }
};

// Few rows (16 QT): a wave per (sequence, KV head, share of the keys). Codes go to LDS
// (keys of the next chunk while this one's values are used, and the other way round) and
// are made 16-bit numbers on their way into the matrix units, one instruction for two;
// the steps are applied in 32 bits: to the scores of a group's product, and to the
// probabilities before the value product, one set of them for each group. Keys past what
// a row sees have p = 0, codes are finite whatever they are, and a value's
// step is 0 where it is NaN, so nothing that is not seen comes through.
//   scores: S^T = K Q^T, 16 keys x 16 columns a product; lane (g, p) has four keys of column p
//   values: O^T = V^T P, 16 columns x 16 rows over 32 keys; a transposing read gives lane
//   (g, i) one column's 16 keys 16 a + 4 g + b, a, b < 4: the order that P has anyway.
// SUB > 1: up to 16 / SUB rows. The columns of Q are those rows SUB times, once for each
// SUB-th of the chunk and zero outside the lanes that hold its keys, so a product has the
// scores of 16 SUB keys and no lane holds one twice: a SUB-th of the exponentials and
// splits. For the value product the first part's columns take the others' probabilities.
// One token over 262144 rows, 8 heads, d 64: 25 us, 5.7 TB/s; 32 sequences, 16 heads over
// 2, d 256: 23 us, 3.4 TB/s, one wave's chain from load to product.
// W > 1: a workgroup's waves share a sequence's chunks and join their parts in LDS, where
// that spares short caches the second launch.
// QT > 1: that many 16-row tiles, for which the codes are made numbers once; P times the
// step is then rounded once in bf16, to half a step of what the result is rounded to (two
// pieces: 16 sequences of 8192 to 16384 rows, 24 rows a head, d 128 34.7 us against 31.2, d
// 64 25.0 against 23.5; one of 65536, d 128 37.0 against 32.9).
// waves to a SIMD: one where 256 registers are too few
constexpr int part4_waves(bool f32, int dp, int sub, int qt) {
  const int regs = qt * (dp / 4 + dp / 8 * sub * (f32 ? 3 : 1) + 32 / sub) + 64 + dp / 4;
  return regs < 256 || (dp == 256 && sub == 2) ? 2 : 1;
}
template <typename T, int DP, int SUB, int QT, int W>
__global__ __launch_bounds__(64 * W, part4_waves(sizeof(T) == 4, DP, SUB, QT)) void cache4_part_kernel(Cache4Args c4) {
  using C = Part4<DP>;
  using K = typename Pieces<T>::K;
  static_assert(SUB == 1 || QT == 1, "parts of the chunk are for one tile");
  constexpr int KC = C::KC, NM = 4 / SUB, ROWS = 16 / SUB, LPS = 4 / SUB;  // LPS: lane groups that hold a part's keys
  constexpr int NG = C::NG, NQ = Pieces<T>::Q, NP = QT > 1 && __is_same(T, bf16) ? 1 : Pieces<T>::P, NT = DP / 16;
  constexpr int NF = DP / 32 * SUB, FG = DP == 32 ? NF : 2 * SUB;  // products of a score; of a group
  constexpr int PITCH = DP == 192 ? 256 : DP;
  extern __shared__ __attribute__((aligned(16))) char smem_all[];
  const CacheArgs &a = c4.a;
  const int wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char *smem = smem_all + wave * C::LDS;
  const int lane = threadIdx.x & 63, g = lane >> 4, p = lane & 15, sub = p / ROWS;
  // (a share's heads side by side: 32 sequences, 16 heads over 2, d 256: 29.4 us against 32.6)
  const int share = (int)(blockIdx.x / (uint32_t)a.Hkv), hk = (int)(blockIdx.x - (uint32_t)share * a.Hkv);
  int b, split, np, before;
  if constexpr (W > 1) {
    b = share; split = wave; np = W;
  } else {
    if (!share4<false, 1>(c4, share, lane, b, split, np, before)) return;
    if (split == 0 && hk == 0 && lane == 0 && !a.direct) c4.used[b] = int2{before, np};
  }
  const int n = __builtin_amdgcn_readfirstlane(seq_len(a, b)), count = __builtin_amdgcn_readfirstlane(seq_count(a, b));
  const int keys = count > 0 ? n : 0;
  int low = n - count + 1;  // below it every row sees every key
  low = low < 0 ? 0 : low;
  // rows: token, head, keys seen (a row that is none sees what the last one sees, so it asks for no masking)
  const T *qrow[QT];
  int tok[QT], head[QT], lim[QT];
  bool valid[QT];
  const float inv_g = 1.f / (float)a.G;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int rho = qt * 16 + p % ROWS, x = rho < a.TG ? rho : 0;
    tok[qt] = (int)(((float)x + 0.5f) * inv_g);  // (x / G: both below 2^7, exact)
    head[qt] = hk * a.G + x - tok[qt] * a.G;
    valid[qt] = rho < a.TG && tok[qt] < count;
    lim[qt] = valid[qt] ? clampi(n - count + tok[qt] + 1, 0, n) : keys;
    qrow[qt] = (const T *)a.q + b * a.sq[0] + head[qt] * a.sq[1] + tok[qt] * a.sq[2];
  }
  int c0, c1;
  share_of((int)(((uint32_t)keys + KC - 1) / KC), split, np, c0, c1);

  const int64_t kstep = a.sk[2], vstep = a.sv[2];
  // the next chunk to load
  const char *knext = uniform((const char *)a.k + b * a.sk[0] + hk * a.sk[1] + (int64_t)c0 * KC * kstep);
  const char *vnext = uniform((const char *)a.v + b * a.sv[0] + hk * a.sv[1] + (int64_t)c0 * KC * vstep);
  const char *snext = uniform((const char *)(c4.step + b * c4.ss[0] + hk * c4.ss[1]) + (int64_t)c0 * C::STEPS);
  uint32_t koff[C::KV], voff[C::VV];
  {
    const int last = a.D / 32 - 1;  // (columns past the head dim: the row's last unit; 64 strides of less than 2^26: check_held)
    auto off = [&](int i, int row, int c, int64_t step) {
      return (uint32_t)(C::RL ? row - C::RL * i : row) * (uint32_t)step + (c < last ? c : last) * 16;
    };
#pragma unroll
    for (int i = 0; i < C::KV; ++i) {
      const int u = i * 64 + lane, row = u / C::CPR;
      koff[i] = off(i, row, u % C::CPR ^ C::swk(row), kstep);
    }
#pragma unroll
    for (int i = 0; i < C::VV; ++i) {
      const int u = i * C::VD * 64 + lane, row = u / C::CPR;
      voff[i] = off(i * C::VD, row, u % C::CPR ^ C::swv(row), vstep);
    }
  }
  auto issue_codes = [&](const char *src, int64_t step, auto offset, int left, char *dst) {
    if (left >= KC) {
#pragma unroll
      for (int i = 0; i < C::CPR; ++i) g2lds16_s(src + i * C::RL * step, offset(i), dst + i * 1024);
    } else {  // (rows past the end: the end of the last one)
      const uint32_t lim0 = (uint32_t)(left - 1) * (uint32_t)step + (uint32_t)a.D / 2 - 16;
#pragma unroll
      for (int i = 0; i < C::CPR; ++i) {
        const uint32_t o = offset(i) + (uint32_t)(i * C::RL) * (uint32_t)step;
        g2lds16_s(src, o > lim0 ? lim0 : o, dst + i * 1024);
      }
    }
  };
  auto issue_keys = [&](int c) {  // and steps
    const int left = keys - c * KC;  // (c is a chunk of the sequence: at least 1)
    issue_codes(knext, kstep, [&](int i) { return koff[i % C::KV]; }, left, smem);
    const uint32_t words = (uint32_t)min(KC, left) * NG;  // (rows past the end: the last step)
    char *sd = smem + 2 * C::TILE + (c & 1) * C::STEPS;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const uint32_t u = i * 64 + lane;
      g2lds4_s(snext, (u < words ? u : words - 1) * 4, sd + i * 256);
    }
    knext += KC * kstep;
    snext += C::STEPS;
  };
  auto issue_values = [&](int c) {
    issue_codes(vnext, vstep, [&](int i) { return voff[i / C::VD]; }, keys - c * KC, smem + C::TILE);
    vnext += KC * vstep;
  };
  if (c0 < c1) {
    issue_keys(c0);
    issue_values(c0);
  }

  s16x8 fr[QT][NF][NQ];
  load_queries<T>([&](auto INF, float &top) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        // product f of the group's FG: elements 8 f .. of this lane's, a LPS-th of the group
        load_q8<T, decltype(INF)::value>(a, qrow[qt], (DP == 32 ? 0 : 64 * (f / FG)) + (g % LPS) * 8 * FG + 8 * (f % FG), SUB == 1 || g / LPS == sub, fr[qt][f], top);
      }
  });
  // this lane's scores: keys 16 (sub NM + m) + 4 g + r; the row that it reads of 16-row tile m
  const int key0 = 16 * sub * NM + 4 * g, krow = 16 * (g / LPS) * NM + p, kswz = C::swk(p);
  const int vrow = 16 * (p >> 2) + 4 * g + (p & 3), vswz = C::swv(vrow);

  SoftmaxState<DP> sm[QT];
  float scale[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    sm[qt].init();
    scale[qt] = a.scale2;
  }
  for (int c = c0; c < c1; ++c) {
    wait_vmcnt<C::CPR>();  // keys and steps are here, the values may be under way
    lds_wait_all();
    const char *Ks = smem, *Vs = smem + C::TILE, *Ss = Vs + C::TILE + (c & 1) * C::STEPS;
    f32x4 s[QT][NM];
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      Steps4<T, NG> st;
      st.load(Ss, key0 + 16 * m);
      const char *row = Ks + (krow + 16 * m) * C::RB;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        f32x4 acc[QT];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) acc[qt] = f32x4{0.f, 0.f, 0.f, 0.f};
        uint32_t w[FG];  // this lane's codes of the group: 4 FG bytes
        if constexpr (FG >= 4) {
#pragma unroll
          for (int u = 0; u < FG / 4; ++u) {
            const int unit = DP == 32 ? 0 : 2 * j + (g % LPS) * (FG / 4) + u;
            const u32x4 x = *(const u32x4 *)(row + ((unit ^ kswz) << 4));
#pragma unroll
            for (int i = 0; i < 4; ++i) w[4 * u + i] = x[i];
          }
        } else if constexpr (FG == 2) {
          // (16 elements of four lane groups, or of two at d 32)
          const int unit = DP == 32 ? 0 : 2 * j + (g >> 1);
          const u32x2 x = *(const u32x2 *)(row + ((unit ^ kswz) << 4) + (g & 1) * 8);
          w[0] = x[0];
          w[1] = x[1];
        } else {
          w[0] = *(const uint32_t *)(row + 4 * g);
        }
#pragma unroll
        for (int i = 0; i < FG; ++i) {
          const s16x8 x = codes8<K>(w[i]);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
#pragma unroll
            for (int y = NQ - 1; y >= 0; --y) acc[qt] = Mfma16<K>::run(x, fr[qt][j * FG + i][y], acc[qt]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float y = st.key(r, j);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) s[qt][m][r] = j ? __builtin_fmaf(acc[qt][r], y, s[qt][m][r]) : acc[qt][r] * y;
        }
      }
    }
    lds_wait_all();  // the keys' reads, whose place is filled next
    const bool more = c + 1 < c1;
    if (more) issue_keys(c + 1);
    if ((c + 1) * (int64_t)KC > low) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int m = 0; m < NM; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (key0 + 16 * m + r >= lim[qt] - c * KC) s[qt][m][r] = -INFINITY;
      // (a value's step that is NaN, as its key's is: 0 for the rows that do not see it)
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        uint16_t *v = (uint16_t *)(smem + 2 * C::TILE + (c & 1) * C::STEPS) + lane * 2 * NG + NG + j;
        if ((*v & 0x7fff) > (__is_same(T, f16) ? 0x7c00 : 0x7f80)) *v = 0;
      }
    }
    float x[QT][NM][4];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) softmax4<NM, ROWS, 0>(sm[qt], scale[qt], s[qt], a.scale2, x[qt]);

    if (more) wait_vmcnt<C::CPR + NG>();
    else wait_vmcnt<0>();
    lds_wait_all();
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      s16x8 pk[QT][2][NP];  // keys of the transposing read's first and second word
      float y[QT][NM][4];
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        Steps4<T, NG> st;
        st.load(Ss, key0 + 16 * m);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float z = st.value(r, j);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) y[qt][m][r] = x[qt][m][r] * z;
        }
      }
      if constexpr (SUB == 1) {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
          for (int h = 0; h < 2; ++h) split8<NP>(&y[qt][2 * h][0], pk[qt][h]);
      } else {
        // the columns of the first part take the others' (theirs hold what no one reads)
        float z[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          z[r] = y[0][0][r];
          z[4 + r] = SUB == 2 ? y[0][NM - 1][r] : 0.f;
        }
        s16x8 one[NP];
        split8<NP>(z, one);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const u32x4 w = __builtin_bit_cast(u32x4, one[i]);
          u32x4 v[2];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            auto from = [&](auto N, uint32_t x) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x120 + decltype(N)::value, 0xf, 0xf, false); };  // lane p + 16 - N
            if constexpr (SUB == 2) {
              v[0][e] = w[e];
              v[1][e] = from(std::integral_constant<int, 8>{}, w[e]);
            } else {
              v[0][e] = e < 2 ? w[e] : from(std::integral_constant<int, 12>{}, w[e % 2]);
              v[1][e] = e < 2 ? from(std::integral_constant<int, 8>{}, w[e % 2]) : from(std::integral_constant<int, 4>{}, w[e % 2]);
            }
          }
          pk[0][0][i] = __builtin_bit_cast(s16x8, v[0]);
          pk[0][1][i] = __builtin_bit_cast(s16x8, v[1]);
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
        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
          for (int i = NP - 1; i >= 0; --i) {
            sm[qt].o[4 * j + t] = Mfma16<bf16>::run(v0, pk[qt][0][i], sm[qt].o[4 * j + t]);
            sm[qt].o[4 * j + t] = Mfma16<bf16>::run(v1, pk[qt][1][i], sm[qt].o[4 * j + t]);
          }
      }
    }
    lds_wait_all();  // the values' reads
    if (more) issue_values(c + 1);
  }

  if constexpr (W > 1) {
    // the waves' parts through LDS, each in its own ring's place (O's rows are as long
    // as the two tiles), added up in order by threads of four columns each
    static_assert(QT == 1, "one tile's O in a wave's ring");
    constexpr int RING = C::LDS, STAT = 2 * C::TILE;
    float lt = sm[0].total();
#pragma unroll
    for (int x = ROWS; x < 16; x <<= 1) lt += shfl_xor_f(lt, x);
    if (p < ROWS) {
      if (g == 0) ((float2 *)(smem + STAT))[p] = float2{sm[0].m, lt};
#pragma unroll
      for (int t = 0; t < NT; ++t) *(f32x4 *)(smem + (p * DP + 16 * t + 4 * g) * 4) = sm[0].o[t];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.TG * (DP / 4); i += 64 * W) {
      const int row = i / (DP / 4), d = i % (DP / 4) * 4;
      float m = -INFINITY, l = 0.f;
      float2 st[W];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        st[w] = ((const float2 *)(smem_all + w * RING + STAT))[row];
        m = fmaxf(m, st[w].x);
      }
      const float ref = m == -INFINITY ? 0.f : m;
      f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (st[w].y == 0.f) continue;  // (a NaN sum is kept)
        const float f = st[w].x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(st[w].x - ref);
        l += f * st[w].y;
        acc += f * *(const f32x4 *)(smem_all + w * RING + (row * DP + d) * 4);
      }
      RowInfo ri;
      ri.b = b;
      ri.t = (int)(((float)row + 0.5f) * inv_g);
      ri.hq = hk * a.G + row - ri.t * a.G;
      if (ri.t >= count) l = 0.f;
      store_row<T>(a, ri, acc, l == 0.f ? 0.f : 1.f / l, d);
      if (d == 0 && a.lse) a.lse[((int64_t)b * a.Hq + ri.hq) * a.T + ri.t] = lse4(a.scale2, m, l);
    }
    return;
  }
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    float lt = sm[qt].total();
    const float m = sm[qt].m;
    if constexpr (SUB > 1) {
#pragma unroll
      for (int x = ROWS; x < 16; x <<= 1) lt += shfl_xor_f(lt, x);
      if (p >= ROWS) return;
    }
    const int rho = qt * 16 + p;
    if (rho >= a.TG) continue;
    if (a.direct || np == 1) {
      RowInfo ri;
      ri.b = b; ri.t = tok[qt]; ri.hq = head[qt];
      const float l = valid[qt] ? lt : 0.f, inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int t = 0; t < NT; ++t) store_row<T>(a, ri, sm[qt].o[t], inv, 16 * t + 4 * g);
      if (g == 0 && a.lse) a.lse[((int64_t)b * a.Hq + head[qt]) * a.T + tok[qt]] = lse4(a.scale2, m, l);
      continue;
    }
    const int64_t at = ((int64_t)hk * a.np_own + share) * a.TG + rho;
    if (g == 0) a.stat[at] = float2{m, lt};
    if (valid[qt] && lt != 0.f) {  // (a NaN sum is kept)
      float *dst = a.part + at * PITCH;
#pragma unroll
      for (int t = 0; t < NT; ++t) *(f32x4 *)(dst + 16 * t + 4 * g) = sm[qt].o[t];
    }
  }
}

// Many rows: a workgroup per (tile of NW x 16 QT rows, share of the keys). Its threads
// make 16-bit numbers of the codes, steps and all (exact), in LDS, and from there it is
// the tile of a 16-bit cache. 2048 tokens over 16301 rows, 16 heads over 2, d 256: 541 us,
// 0.95 PFLOP/s, matrix units 39% busy, LDS 49%, vector issue 51%, eight waves in step. P is
// rounded to the operand type once: a second piece is another product for each of the value
// ones (that case 25% longer, 512 tokens of 2 sequences, d 128 18%, 48 rows a head, d 64
// 5%), and one rounding of P and one of the result make 0.0023 of the result where the
// second alone is 0.0017. 32-bit rows are three bf16 pieces of queries and of
// probabilities: six products of the matrix units' fastest type cost less than two of the
// slow 32-bit one.
template <typename K, int DP, int QT, int NM, int N>
__device__ __forceinline__ void qk_pieces(const char *tile, const RowFrag<K, DP> (&fr)[N * QT], f32x4 (&s)[QT][NM], int g, int p) {
  if constexpr (N == 1) {
    qk_tile<K, DP, QT, NM>(tile, fr, s, g, p);
  } else {  // (a fragment of K read once, the smallest pieces' products added first)
    f32x4 acc[N * QT][NM];
    qk_tile<K, DP, N * QT, NM>(tile, fr, acc, g, p);
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        s[qt][m] = acc[(N - 1) * QT + qt][m];
#pragma unroll
        for (int n = N - 2; n >= 0; --n) s[qt][m] += acc[n * QT + qt][m];
      }
  }
}
// O += V^T P with P as N bf16 pieces, a fragment of V read once
template <int DP, int KC, int N>
__device__ __forceinline__ void pv_pieces(const char *tile, const float (&x)[KC / 16][4], SoftmaxState<DP> &sm, int g, int p) {
  constexpr int CPR = DP / 8, K2 = KC / 32, NTL = DP / 16, VL = NTL < 8 ? NTL : 8, RPT = 2 * K2, W = NTL < 4 ? NTL : 4;
  s16x8 pk[K2][N];
#pragma unroll
  for (int k2 = 0; k2 < K2; ++k2) split8<N>(&x[2 * k2][0], pk[k2]);
  s16x4 lo[NTL][K2], hi[NTL][K2];
  unsigned vb[VL];
#pragma unroll
  for (int l = 0; l < VL; ++l) vb[l] = (unsigned)(uintptr_t)tile + tile_vbase(l, g, p, CPR);
  auto rd = [&](auto TT) {
    constexpr int t = decltype(TT)::value;
    static_for<K2>([&](auto KK) {
      constexpr int k2 = decltype(KK)::value, off = (t / 8) * 256 + k2 * 512 * CPR;
      lo[t][k2] = lds_read_tr16_at<off>(vb[t % 8]);
      hi[t][k2] = lds_read_tr16_at<off + 256 * CPR>(vb[t % 8]);
    });
  };
  static_for<W>(rd);
  static_for<NTL>([&](auto TT) {
    constexpr int t = decltype(TT)::value;
    constexpr int last = t + W - 1 < NTL - 1 ? t + W - 1 : NTL - 1, n = (last - t) * RPT;
    lds_wait_le<(n < 15 ? n : 15)>();
#pragma unroll
    for (int k2 = 0; k2 < K2; ++k2) {
      lds_ready(lo[t][k2]);
      lds_ready(hi[t][k2]);
      const s16x4 a = lo[t][k2], b = hi[t][k2];
      const s16x8 av = s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
#pragma unroll
      for (int i = N - 1; i >= 0; --i) sm.o[t] = Mfma16<bf16>::run(av, pk[k2][i], sm.o[t]);
    }
    if constexpr (t + W < NTL) rd(std::integral_constant<int, t + W>{});
  });
}

template <typename T, int DP, int NW> struct Tile4 {
  using K = typename Pieces<T>::K;
  static constexpr int KC = 64, NT = NW * 64, CPR = DP / 8, TILE = KC * DP * 2, STAGE = 2 * TILE;
  // One stage where two leave a CU fewer workgroups of four waves, which hide each other's
  // barriers (16 sequences of 2000 to 16384 rows, 64 rows a head, d 256: 87 us with two, 50 with one)
  static constexpr int STAGES = DP >= 128 && NW == 4 && sizeof(T) == 2 ? 1 : 2, LDS = STAGES * STAGE;
  static constexpr int BYTES = KC * DP / NT, LB = BYTES / 2 < 16 ? BYTES / 2 : 16, NL = BYTES / LB;  // codes of a thread: NL loads of LB bytes, half of keys
  static constexpr int UPR = DP / 2 / LB;                                                    // loads of a row
  static_assert(LDS <= 160 * 1024, "LDS");
};

template <typename T, int DP, int NW, int QT>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 4 && DP == 256 ? 1 : 2) void cache4_tile_kernel(Cache4Args c4) {
  using C = Tile4<T, DP, NW>;
  using K = typename C::K;
  constexpr int KC = C::KC, NM = KC / 16, N = Pieces<T>::Q, UP = __is_same(T, f16) ? 7 : 0;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const CacheArgs &a = c4.a;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, p = lane & 15;
  const int tr = a.tr_own;
  const int i = (int)(blockIdx.x / (uint32_t)a.Hkv), hk = (int)(blockIdx.x - (uint32_t)i * a.Hkv);
  int u, split, np, before;
  if (!share4<true, 2>(c4, i, lane, u, split, np, before)) return;
  if (split == 0 && hk == 0 && tid == 0 && !a.direct) c4.used[u] = int2{before, np};
  const int tile = a.rt_own - 1 - u / a.B, b = u % a.B;
  const int64_t slot = ((int64_t)hk * a.np_own + i) * tr;
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
  int c0, c1;
  share_of((int)(((uint32_t)keys + KC - 1) / KC), split, np, c0, c1);

  static_assert(N == 1 || QT == 1, "pieces of one fragment");
  RowFrag<K, DP> fr[N * QT];
  load_queries<T>([&](auto INF, float &top) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int ks = 0; ks < DP / 32; ++ks) {
        s16x8 x[N];
        load_q8<T, decltype(INF)::value>(a, (const T *)a.q + ri[qt].b * a.sq[0] + ri[qt].hq * a.sq[1] + ri[qt].t * a.sq[2], 32 * ks + 8 * g, true, x, top);
#pragma unroll
        for (int n = 0; n < N; ++n) fr[n * QT + qt].h[ks] = x[n];
      }
  });

  // this thread's loads: half of keys, half of values, at the same rows and places
  constexpr int NH = C::NL / 2;
  int row[NH], place[NH], sj[NH];
  uint32_t koff[NH], voff[NH], cw[C::NL][C::LB / 4], sw[C::NL];
  bool in[NH];
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    const int u = n * C::NT + tid, last = a.D / 2 / C::LB - 1, c = u % C::UPR, at = (c < last ? c : last) * C::LB;
    row[n] = u / C::UPR;
    place[n] = c;
    sj[n] = at * 2 / kGroup4;
    koff[n] = (uint32_t)(row[n] * a.sk[2] + at);
    voff[n] = (uint32_t)(row[n] * a.sv[2] + at);
  }
  const char *kb = (const char *)a.k + b * a.sk[0] + hk * a.sk[1], *vb = (const char *)a.v + b * a.sv[0] + hk * a.sv[1];
  const uint16_t *sb = c4.step + b * c4.ss[0] + hk * c4.ss[1];
  const int64_t kchunk = a.sk[2] * KC, vchunk = a.sv[2] * KC;
  const int ng = c4.ng;
  auto fetch = [&](const char *src, uint32_t (&y)[C::LB / 4]) {
    if constexpr (C::LB == 16) {
      const u32x4 x = *(const u32x4 *)src;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = x[i];
    } else if constexpr (C::LB == 8) {
      const u32x2 x = *(const u32x2 *)src;
      y[0] = x[0];
      y[1] = x[1];
    } else {
      y[0] = *(const uint32_t *)src;
    }
  };
  auto load = [&](int c) {
    const int left = keys - c * KC;  // rows from the chunk's first on (below 2^31)
    const char *kc = kb + c * kchunk, *vc = vb + c * vchunk;
    const uint16_t *sc = sb + (int64_t)c * KC * 2 * ng;
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      in[n] = row[n] < left;
      // (rows past the end: the first one's codes, and steps of zero)
      fetch(kc + (in[n] ? koff[n] : 0u), cw[n]);
      fetch(vc + (in[n] ? voff[n] : 0u), cw[NH + n]);
      const uint32_t at = in[n] ? (uint32_t)(row[n] * 2 * ng + sj[n]) : 0u;
      sw[n] = sc[at];
      sw[NH + n] = sc[at + ng];
    }
  };
  auto store = [&](int stage) {
#pragma unroll
    for (int n = 0; n < C::NL; ++n) {
      const float y = step_f32<T>(sw[n]);
      // (a value's NaN is its key's too)
      const float st = !in[n % NH] ? 0.f : n < NH ? y : fmaxf(y, 0.f);
      char *tl = smem + stage * C::STAGE + (n < NH ? 0 : C::TILE) + row[n % NH] * DP * 2;
      // a load's words are 16-byte units side by side, and lanes next to each other would
      // write to a few banks: each starts at another word
      constexpr int NWD = C::LB / 4;
      const int first = NWD == 4 ? (C::UPR == 8 ? place[n % NH] + (place[n % NH] >> 2) : place[n % NH]) & 3 : place[n % NH] & (NWD - 1);
      uint32_t x[NWD];
#pragma unroll
      for (int i = 0; i < NWD; ++i) x[i] = first & 1 ? cw[n][(i + 1) % NWD] : cw[n][i];
      if constexpr (NWD == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t y0 = x[i], y1 = x[i + 2];
          x[i] = first & 2 ? y1 : y0;
          x[i + 2] = first & 2 ? y0 : y1;
        }
      }
#pragma unroll
      for (int i = 0; i < NWD; ++i)
        *(s16x8 *)(tl + ((place[n % NH] * NWD + ((i + first) & (NWD - 1))) ^ swz(row[n % NH], C::CPR)) * 16) = values8<K>(x[i], st);
    }
  };

  SoftmaxState<DP> sm[QT];
  float scale[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    sm[qt].init();
    scale[qt] = a.scale2;
  }
  if (c0 < c1) {
    load(c0);
    if constexpr (C::STAGES == 2) {
      store(0);
      if (c0 + 1 < c1) load(c0 + 1);
    }
  }
  int stage = 0;
  for (int c = c0; c < c1; ++c) {
    if constexpr (C::STAGES == 2) {
      lds_barrier();  // chunk c is written, and every wave has read chunk c - 1, whose place is filled next
      if (c + 1 < c1) store(stage ^ 1);
      if (c + 2 < c1) load(c + 2);
    } else {
      if (c > c0) lds_barrier();  // every wave has read chunk c - 1
      store(0);
      lds_barrier();
      if (c + 1 < c1) load(c + 1);
    }
    const char *Ks = smem + stage * C::STAGE, *Vs = Ks + C::TILE;
    if constexpr (C::STAGES == 2) stage ^= 1;
    if (w * QT * 16 >= tr) continue;
    f32x4 s[QT][NM];
    qk_pieces<K, DP, QT, NM, N>(Ks, fr, s, g, p);
    if ((c + 1) * (int64_t)KC > low) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) mask_keys<NM>(s[qt], (ri[qt].valid ? ri[qt].lim : keys) - c * KC, g);
    }
    float x[QT][NM][4];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) softmax4<NM, 16, UP>(sm[qt], scale[qt], s[qt], a.scale2, x[qt]);
    if constexpr (N == 1) {
      pv_tile<K, DP, KC, QT>(Vs, x, sm, g, p);
    } else {
      pv_pieces<DP, KC, N>(Vs, x[0], sm[0], g, p);
    }
  }

#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int i = (w * QT + qt) * 16 + p;
    if (i >= tr) continue;
    const float lt = sm[qt].total();
    if (a.direct || np == 1) {
      if (tile * tr + i >= a.TG) continue;
      const float l = ri[qt].valid ? lt : 0.f, inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) store_row<T>(a, ri[qt], sm[qt].o[t], inv, 16 * t + 4 * g);
      if (g == 0 && a.lse) a.lse[((int64_t)ri[qt].b * a.Hq + ri[qt].hq) * a.T + ri[qt].t] = lse4(a.scale2, sm[qt].m, l);
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

// A row's parts added up: 8 threads to a part's 32 columns (a block has CW columns of a
// row), so NG parts at a time, each thread with a running maximum of its own parts; then
// across the threads in a fixed order.
template <typename T, int TEAM, int CW> __global__ __launch_bounds__(256) void cache4_join_kernel(Cache4Args c4, int pitch) {
  constexpr int LG = CW / 4, NG = TEAM / LG, U = 4;
  __shared__ f32x4 s_acc[256];
  __shared__ float2 s_ml[256];
  const CacheArgs &a = c4.a;
  const int tid = threadIdx.x, in = tid % TEAM, gi = in / LG, e = in % LG;
  const uint32_t row = blockIdx.x * (256 / TEAM) + tid / TEAM, rows = (uint32_t)a.B * a.Hkv * a.TG;
  if (TEAM < 256 && row >= rows) return;
  const uint32_t seq = row / (uint32_t)a.TG;
  const int rho = (int)(row - seq * (uint32_t)a.TG), b = (int)(seq / (uint32_t)a.Hkv), hk = (int)(seq - (uint32_t)b * a.Hkv);
  const RowInfo ri = row_info(a, b, hk, rho);
  const int col = blockIdx.y * CW + 4 * e;
  // part i of the row: first + i * tr_own
  const int tile = rho / a.tr_own;
  const int2 u = a.B * a.rt_own > 1 ? c4.used[(a.rt_own - 1 - tile) * a.B + b] : int2{0, a.np_own};
  const int64_t first = ((int64_t)hk * a.np_own + u.x) * a.tr_own + (rho - tile * a.tr_own);
  int n = u.y;
  if (n == 1) return;  // (written by the one that had it all)
  if (!ri.valid) n = 0;
  float m = -INFINITY, l = 0.f;
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int i = gi; i < n; i += U * NG) {
    float2 st[U];
    f32x4 y[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {  // (one that there is not: the first again, left out)
      const int64_t at = first + (int64_t)(i + j * NG < n ? i + j * NG : i) * a.tr_own;
      st[j] = a.stat[at];
      y[j] = *(const f32x4 *)(a.part + at * pitch + col);
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (i + j * NG >= n || st[j].y == 0.f) continue;  // (a part of no keys has no O)
      const float mn = fmaxf(m, st[j].x), ref = mn == -INFINITY ? 0.f : mn;
      const float f0 = __builtin_amdgcn_exp2f(m - ref), f1 = st[j].x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(st[j].x - ref);
      l = l * f0 + st[j].y * f1;
      acc = acc * f0 + y[j] * f1;
      m = mn;
    }
  }
  // threads e of the groups: neighbours first
  auto add = [&](float m2, float l2, f32x4 a2) {
    const float mn = fmaxf(m, m2), ref = mn == -INFINITY ? 0.f : mn;
    const float f0 = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - ref), f1 = m2 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m2 - ref);
    l = l * f0 + l2 * f1;
    acc = acc * f0 + a2 * f1;
    m = mn;
  };
#pragma unroll
  for (int x = LG; x < 64; x <<= 1) {
    f32x4 a2;
#pragma unroll
    for (int r = 0; r < 4; ++r) a2[r] = shfl_xor_f(acc[r], x);
    add(shfl_xor_f(m, x), shfl_xor_f(l, x), a2);
  }
  if constexpr (TEAM == 256) {
    if ((tid & 63) < LG) {
      s_acc[tid] = acc;
      s_ml[tid] = float2{m, l};
    }
    __syncthreads();
    if (tid >= LG) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) add(s_ml[w * 64 + tid].x, s_ml[w * 64 + tid].y, s_acc[w * 64 + tid]);
  } else if (gi) {
    return;
  }
  store_row<T>(a, ri, acc, l == 0.f ? 0.f : 1.f / l, col);
  if (col == 0 && a.lse) a.lse[((int64_t)b * a.Hq + ri.hq) * a.T + ri.t] = lse4(a.scale2, m, l);
}

// ---- host ---------------------------------------------------------------------
struct Plan4 {
  int64_t DP, pitch, tr, rt, np, want, rows;
  int sub, qt;  // 0: the tile kernel
  bool direct;  // each row's one share is its whole answer
  bool joined;  // the waves of a workgroup share a sequence's chunks
  size_t used, part, total;
};
// (queries take D SUB / 8 registers, 32-bit ones three times as many; O D / 4 for each 16 rows)
constexpr int most_sub4(bool f32, int64_t dp) { return f32 ? (dp <= 64 ? 4 : dp == 128 ? 2 : 1) : dp <= 128 ? 4 : 2; }
// Waves of a workgroup that joins its own parts: with four, which take half as much LDS and
// so many short sequences better, more calls are left to two launches (8 heads, d 128: 64
// sequences of 2048 to 4096 rows 43.9 us against 55.8, of 256 to 512 14.1 against 10.0; fp32
// d 64, 4 heads: 32 of 512 to 1024 9.2 and 9.3; over 100 shapes within 2% in the mean)
constexpr int kJoined4 = 8;
constexpr int most_tiles4(bool f32, int64_t dp) { return dp <= (f32 ? 64 : 128) ? 2 : 1; }
static Plan4 plan4(const fbsa_attn4_desc *d) {
  Plan4 p;
  const int64_t TG = d->T * (d->Hq / d->Hkv), seqs = d->B * d->Hkv;
  const bool f32 = d->dtype == FBSA_F32;
  p.DP = d->D <= 32 ? 32 : d->D <= 64 ? 64 : d->D <= 128 ? 128 : d->D <= 192 ? 192 : 256;
  // Two 16-row tiles to a wave against the tile kernel, 16 sequences of 2000 to 16384
  // rows, 24 rows a head: d 64 21.0 us against 23.2, d 128 27.6 against 33.5, fp32 d 64
  // 25.5 against 36.5; three tiles lose (48 rows, d 128: 42.0 against 36.1)
  const bool few = TG <= 16 * most_tiles4(f32, p.DP);
  if (!few && p.DP == 192) p.DP = 256;
  p.pitch = p.DP == 192 ? 256 : p.DP;
  p.sub = !few ? 0 : (int)std::min<int64_t>(most_sub4(f32, p.DP), TG <= 4 ? 4 : TG <= 8 ? 2 : 1);
  p.qt = few ? (int)cdiv(TG, 16) : 0;
  p.tr = few ? TG : tile_rows(d->dtype, TG);
  p.rt = cdiv(TG, p.tr);
  p.joined = false;
  if (few) {
    // Shares of the chunks: as many as run at a time with two waves to a SIMD, or one
    // where a wave has more to do or rows are long (32 sequences, 16 heads over 2, d 256:
    // 28.9 us against 30.3; one of 131072 rows 27.8 against 31.4; d 64, 262144 rows: 40.0
    // against 29.9). Sequences round theirs up.
    const int64_t each = std::max<int64_t>(1, kCUs * (p.qt > 1 || p.DP >= 192 ? 4 : 8) / d->Hkv), nc = cdiv(d->S, 64);
    p.want = each;
    // One share a sequence where the card goes through them several times and a wave with
    // the longest is soon done beside the counting that shares take (30000 sequences of up
    // to 130 rows, 24 heads over 1: 107 us against 3702; 1024 of up to 1024, 8 heads, fp32 d
    // 256: 351 against 426; but 1099 of 64 rows and one of 16384, 8 heads, d 64: 213 against 47)
    p.np = d->B == 1 ? std::min(each, nc) : d->B >= std::max(4 * each, 8 * nc) ? d->B : std::min(each + d->B, nc * d->B);
    p.rows = d->Hkv * p.np * TG;
    // (kernels of one wave to a SIMD have no such form)
    // One launch against two, where the waves have few chunks each, or the card many
    // workgroups (8 heads, d 64, 1024 rows 6.8 us against 7.7, 4096 10.8 against 8.0; 32
    // sequences of those 15.5 against 18.5, of 8192 rows 24.1 against 25.9; 32 x 2 heads, d
    // 256, 256 rows 9.9 against 12.6, 2048 22.3 against 19.3). Twice the chunks for a lone
    // sequence lose up to half (fp32, 4096 rows 9.2 against 14.1); 256 and more (sequence,
    // head) pairs take four times as many (64 x 8 heads, d 64, 4096 rows 22.3 against 28.8 with
    // as few; more than four times: 64 x 8 heads, d 128, 8192 rows 88 against 118, others alike)
    const int64_t chunks = std::max<int64_t>(1, 256 / p.DP) * std::min<int64_t>(4, std::max<int64_t>(1, seqs / 64));
    p.joined = TG <= 16 && part4_waves(f32, (int)p.DP, p.sub, 1) == 2 && nc > 1 && nc <= kJoined4 * chunks;
  } else {
    // As many as a CU holds (48 rows, d 128, 16 sequences: two to a CU 36.1 us, four
    // 41.0; d 64: 29.6 and 27.8), of 128 keys at least
    const int64_t room = kCUs * (p.DP <= 64 ? (f32 ? 3 : 4) : p.DP == 128 ? (f32 || p.tr > 64 ? 2 : 3) : f32 || p.tr > 64 ? 1 : 2);
    // One share a tile where the card goes through them several times (see above), and for
    // one sequence's tiles as soon as they are half of what runs at a time: those that see the
    // most start first, and shares join through memory (16 heads over 2, d 256: 1040 tokens
    // over 16301 rows 499 us against 530 cut as share4 does, 2048 571 against 581; 2048 tokens
    // that see themselves alone, tiles of few keys to all, 75 against 89, 32 heads over 8, d
    // 128 58 against 89). The last round of workgroups may be all but empty: 1040 tokens over
    // 16301 rows take nearly as long as 2048, 2064 926 us.
    const int64_t each = std::max<int64_t>(1, room / d->Hkv), units = d->B * p.rt, nc = cdiv(d->S, 128);
    p.want = each;
    p.np = units >= std::max(4 * each, 16 * nc) || (d->B == 1 && p.rt > 1 && 2 * units > each) ? units : std::min(2 * units <= each || units == 1 ? each : each + units, nc * units);
    p.rows = d->Hkv * p.np * p.tr;
  }
  p.direct = p.joined || p.np == d->B * p.rt;
  const size_t parts = p.direct ? 0 : (size_t)p.rows;
  p.used = up256(parts * 8);
  p.part = p.used + (p.direct ? 0 : up256((size_t)(d->B * p.rt) * 8));
  p.total = p.part + up256(parts * p.pitch * 4);
  if (p.total == 0) p.total = 256;  // (0 says that a descriptor is refused)
  return p;
}

template <typename T, int DP, int SUB, int QT, int W> static int launch_part4(const Cache4Args &c, const Plan4 &pl, hipStream_t s) {
  constexpr size_t lds = (size_t)W * Part4<DP>::LDS;
  static_assert(lds <= 160 * 1024, "LDS");
  const int e = lds_optin((const void *)cache4_part_kernel<T, DP, SUB, QT, W>, lds, "hipFuncSetAttribute(cache4_part)");
  if (e) return e;
  hipLaunchKernelGGL((cache4_part_kernel<T, DP, SUB, QT, W>), dim3((unsigned)((W > 1 ? c.a.B : pl.np) * c.a.Hkv)), dim3(64 * W), lds, s, c);
  return hip_check(hipGetLastError(), "cache4_part_kernel launch");
}
template <typename T, int DP, int SUB> static int launch_few4(const Cache4Args &c, const Plan4 &pl, hipStream_t s) {
  if constexpr (part4_waves(sizeof(T) == 4, DP, SUB, 1) == 2) {
    if (pl.joined) return launch_part4<T, DP, SUB, 1, kJoined4>(c, pl, s);
  }
  return launch_part4<T, DP, SUB, 1, 1>(c, pl, s);
}
template <typename T> static int launch_join4(const Cache4Args &c, const Plan4 &pl, hipStream_t s) {
  const int64_t rows = (int64_t)c.a.B * c.a.Hkv * c.a.TG;
  const int pitch = (int)pl.pitch;
  // many rows: a wave each (of up to 128 columns); few: a workgroup for 128 or 32 columns, as
  // many workgroups as there are CUs or more. (By waves and workgroups, a call: 4 sequences of
  // 32 heads, d 128, 32768 rows 33.2 us and 27.5; 64 of 5 x 16, d 256 91 and 100. By 128 columns
  // and 32: one of 16 heads, d 128, 131072 rows 42.1 and 22.1; 32 of 16, d 256 36.7 and 46.2.)
  if (rows >= 2048) {
    const unsigned wgs = (unsigned)cdiv(rows, 4);
    if (pitch == 32) hipLaunchKernelGGL((cache4_join_kernel<T, 64, 32>), dim3(wgs), dim3(256), 0, s, c, pitch);
    else if (pitch == 64) hipLaunchKernelGGL((cache4_join_kernel<T, 64, 64>), dim3(wgs), dim3(256), 0, s, c, pitch);
    else hipLaunchKernelGGL((cache4_join_kernel<T, 64, 128>), dim3(wgs, (unsigned)(pitch / 128)), dim3(256), 0, s, c, pitch);
  } else if (pitch >= 128 && rows * pitch >= 32 * 4 * kCUs) {
    hipLaunchKernelGGL((cache4_join_kernel<T, 256, 128>), dim3((unsigned)rows, (unsigned)(pitch / 128)), dim3(256), 0, s, c, pitch);
  } else {
    hipLaunchKernelGGL((cache4_join_kernel<T, 256, 32>), dim3((unsigned)rows, (unsigned)cdiv(c.a.D, 32)), dim3(256), 0, s, c, pitch);
  }
  return hip_check(hipGetLastError(), "cache4_join_kernel launch");
}
template <typename T, int DP, int NW, int QT> static int launch_tile4(const Cache4Args &c, int64_t wgs, hipStream_t s) {
  using C = Tile4<T, DP, NW>;
  const int e = lds_optin((const void *)cache4_tile_kernel<T, DP, NW, QT>, C::LDS, "hipFuncSetAttribute(cache4_tile)");
  if (e) return e;
  hipLaunchKernelGGL((cache4_tile_kernel<T, DP, NW, QT>), dim3((unsigned)wgs), dim3(NW * 64), C::LDS, s, c);
  return hip_check(hipGetLastError(), "cache4_tile_kernel launch");
}
template <typename T, int DP> static int launch_attn4(const Cache4Args &c, const Plan4 &pl, hipStream_t s) {
  const int64_t wgs = c.a.Hkv * pl.np;
  constexpr int MOST = most_sub4(sizeof(T) == 4, DP);
  if constexpr (MOST >= 4) {
    if (pl.sub == 4) return launch_few4<T, DP, 4>(c, pl, s);
  }
  if constexpr (MOST >= 2) {
    if (pl.sub == 2) return launch_few4<T, DP, 2>(c, pl, s);
  }
  if constexpr (most_tiles4(sizeof(T) == 4, DP) == 2) {
    if (pl.qt == 2) return launch_part4<T, DP, 1, 2, 1>(c, pl, s);
  }
  if (pl.qt == 1) return launch_few4<T, DP, 1>(c, pl, s);
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

template <typename T> static int run_attn4(const Cache4Args &c, const Plan4 &pl, hipStream_t s) {
  const int e = dispatch_attn4<T>(c, pl, s);
  return e || c.a.direct ? e : launch_join4<T>(c, pl, s);
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
  // (a launch has fewer than 2^32 threads along an axis, the first of which holds T alone, at
  // least 8 rows to 256; a call's rows in all stay below what one axis takes of them)
  if (d->B * d->H * d->T > 0x7ff0000LL) return fail(FBSA_EUNSUPPORTED, "%s: grid too large", fn);
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
  // (up to 2^127: the power of two above it is a number, far_scale)
  if (!(fabsf(d->scale * kLog2e) <= 0x1p127f)) return fail(FBSA_EINVAL, "%s: scale times log2(e) is beyond 2^127", fn);
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
  if (d->B * cdiv(d->S, 64) > lim) return fail(FBSA_EUNSUPPORTED, "%s: more than 2^31 chunks of 64 rows in all", fn);
  // (fewer than 2^32 threads along an axis: up to 512 a tile and share, 64 or 256 a row that is joined)
  const Plan4 pl = plan4(d);
  if (pl.rows > lim || d->B * d->Hq * d->T > 0x3ff0000LL || (!pl.qt && d->Hkv * pl.np > 0x7f0000LL))
    return fail(FBSA_EUNSUPPORTED, "%s: grid too large", fn);
  return FBSA_OK;
}

static void fill_rows4(Rows4Args &a, const fbsa_rows4_desc *d) {
  for (int x = 0; x < 3; ++x) { a.sk4[x] = d->sk4[x]; a.sv4[x] = d->sv4[x]; a.sk[x] = d->sk[x]; a.sv[x] = d->sv[x]; }
  a.ss[0] = d->ss[0]; a.ss[1] = d->ss[1];
  a.B = (int)d->B; a.H = (int)d->H; a.T = (int)d->T; a.S = (int)d->S; a.D = (int)d->D; a.ng = (int)cdiv(d->D, kGroup4);
}
// LPR: 8 elements a lane, to read as many as are 16 bytes
template <typename T, int LPR> static int launch_rows4(const Rows4Args &a, bool read, hipStream_t s) {
  using A = Rows4<8, LPR>;
  constexpr int LPR_READ = LPR * (int)sizeof(T) / 2;
  using R = Rows4<16 / sizeof(T), LPR_READ>;
  const dim3 wgs((unsigned)cdiv(a.T, read ? R::RPB * R::U : A::RPB * A::U), (unsigned)(a.B * a.H));
  if (read) hipLaunchKernelGGL((cache4_read_kernel<T, LPR_READ>), wgs, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((cache4_append_kernel<T, LPR>), wgs, dim3(256), 0, s, a);
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
  a.direct = pl.direct;
  c.want = (int)pl.want;
  c.used = (int2 *)((char *)workspace + pl.used);
  a.scale2 = d->scale == 0.f ? 1.f : fabsf(d->scale) * kLog2e;
  a.qand = d->scale == 0.f ? 0u : 0xffffffffu;
  a.qxor = d->scale < 0.f ? (d->dtype == FBSA_F32 ? 0x80000000u : 0x80008000u) : 0u;
  a.stat = (float2 *)workspace; a.part = (float *)((char *)workspace + pl.part);
  hipStream_t s = (hipStream_t)stream;
  switch (d->dtype) {
    case FBSA_BF16: return run_attn4<bf16>(c, pl, s);
    case FBSA_F16: return run_attn4<f16>(c, pl, s);
    default: return run_attn4<float>(c, pl, s);
  }
}

}  // extern "C"
