// What the attention kernels over caches share (gfx950): their arguments, the rows
// of a tile, the online softmax, and the products of a tile of many rows.
#pragma once
#include <math.h>

#include "fbsa_common.h"
#include "fbsa_internal.h"
#include "fbsa_tiles.h"

namespace fbsa {

struct CacheArgs {
  const void *q, *k, *v, *kp, *vp, *og;
  void *o;
  float *lse;
  const float *w;
  float *wo;
  const int32_t *lens, *count;
  int64_t sq[3], sk[3], sv[3], so[3], sog[3], skp[2], svp[2], sw[2], swo[2];
  int32_t B, Hq, Hkv, T, S, P, D, G;
  int32_t TG;                // rows per (sequence, KV head): T * G
  int32_t tr_own, tr_pre;    // rows of a tile
  int32_t rt_own, rt_pre;    // tiles of a (sequence, KV head); of a KV head's prefix rows
  int32_t np_own, np_pre;    // shares of a tile's keys
  int32_t few_own, few_pre;  // tiles of 16 rows, a wave each
  int32_t direct;            // a tile's one share is its whole answer: no parts
  float scale2;              // |scale| * log2(e); the sign is the query's (zero: queries of zeros, scale 1)
  uint32_t qand, qxor;       // applied to the query's words
  float *part;               // [tile, share][row] unnormalised O (DP floats): prefix tiles, then own
  float2 *stat;              // [tile, share][row] row maximum (log2 domain), row sum
  float *wpart;              // [row share][B][Hkv][S] weights, where the rows are shared out
  float *lse2;               // [B][Hkv][TG] log2-domain lse for the weights: +inf, probabilities of 0, for rows that see nothing
  float *sc;                 // [B][Hkv][TG][S rounded up to 32] log2-domain scores (up to 16 rows, with weights)
};

// Row rho of a (sequence, KV head): token rho / G, head rho % G. The keys it
// sees of its own cache are [0, lim).
struct RowInfo {
  int b, t, hq, lim;
  bool valid;
};
__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }
__device__ __forceinline__ int seq_len(const CacheArgs &a, int b) { return clampi(a.lens[b], 0, a.S); }
__device__ __forceinline__ int seq_count(const CacheArgs &a, int b) { return a.count ? clampi(a.count[b], 0, a.T) : a.T; }
__device__ __forceinline__ RowInfo row_info(const CacheArgs &a, int b, int hk, int rho) {
  RowInfo r;
  const int n = seq_len(a, b), c = seq_count(a, b);
  r.valid = rho < a.TG;
  const int x = r.valid ? rho : 0;
  r.b = b;
  r.t = x / a.G;
  r.hq = hk * a.G + x % a.G;
  r.valid = r.valid && r.t < c;
  // (a length of up to 2^31 - 1 rows plus 1 may leave 32 bits: clamped before the 1 is added)
  const int64_t m = (int64_t)n - c + r.t + 1;
  r.lim = m < 0 ? 0 : m > n ? n : (int)m;
  return r;
}

// Rows [r0, r1) of a (sequence, KV head): the keys that the last real one sees (0
// if none is real), and those that the first sees.
__device__ __forceinline__ void own_bounds(const CacheArgs &a, int b, int r0, int r1, int &keys, int &low) {
  const int n = seq_len(a, b), c = seq_count(a, b), real = min(r1, c * a.G);
  keys = low = 0;
  if (r0 >= real) return;
  const int64_t k1 = (int64_t)n - c + (real - 1) / a.G + 1, k0 = (int64_t)n - c + r0 / a.G + 1;
  keys = __builtin_amdgcn_readfirstlane(k1 < 0 ? 0 : (int)k1);  // (at most n)
  low = __builtin_amdgcn_readfirstlane(k0 < 0 ? 0 : (int)k0);
}
// chunks [c0, c1) of share `split` of np: nc / np each, one more for the first nc % np
__device__ __forceinline__ void share_of(int nc, int split, int np, int &c0, int &c1) {
  const int per = (int)((uint32_t)nc / (uint32_t)np), more = nc - per * np;
  c0 = split * per + min(split, more);
  c1 = c0 + per + (split < more ? 1 : 0);
}

template <typename T, int DP>
__device__ __forceinline__ void load_frag(RowFrag<T, DP> &fr, const T *row, int g, const CacheArgs &a) {
  // (elements past the head dim are zeros: the tile's columns there hold copies of the row's last chunk)
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int ks = 0; ks < DP / 4; ++ks) {
      const uint32_t x = 4 * ks + g < a.D ? ((const uint32_t *)row)[4 * ks + g] : 0u;
      fr.f[ks] = __uint_as_float((x & a.qand) ^ a.qxor);
    }
  } else {
#pragma unroll
    for (int ks = 0; ks < DP / 32; ++ks) {
      u32x4 x = 32 * ks + 8 * g < a.D ? *(const u32x4 *)(row + 32 * ks + 8 * g) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (x[e] & a.qand) ^ a.qxor;
      fr.h[ks] = __builtin_bit_cast(s16x8, x);
    }
  }
}

// A wave's online softmax over 16 rows (one to a lane column, 4 lanes to a row).
// The running reference moves only when a score passes it by 2^TAU, so few
// chunks rescale the accumulators.
template <int DP> struct SoftmaxState {
  static constexpr float TAU = 8.f;
  float m = -INFINITY, l = 0.f;
  f32x4 o[DP / 16];
  __device__ __forceinline__ void init() {
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // s: raw products (scaled by scale2 > 0 here), masked ones -inf; out: exponentials.
  template <int NM> __device__ __forceinline__ void step(const f32x4 (&s)[NM], float scale2, float (&x)[NM][4]) {
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < NM; ++k) mx = fmaxf(mx, fmaxf(fmaxf(s[k][0], s[k][1]), fmaxf(s[k][2], s[k][3])));
    mx *= scale2;
    if (__ballot(mx > m + TAU)) {
      float mc = fmaxf(mx, shfl_xor_f(mx, 16));
      mc = fmaxf(mc, shfl_xor_f(mc, 32));
      if (mc > m + TAU) {
        const float alpha = __builtin_amdgcn_exp2f(m - mc);
        l *= alpha;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) o[t] *= alpha;
        m = mc;
      }
    }
    const float ref = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < NM; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[k][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k][r], scale2, -ref));
        sum += x[k][r];
      }
    l += sum;
  }
  __device__ __forceinline__ float total() const {  // the row's sum, on its four lanes
    const float lt = l + shfl_xor_f(l, 16);
    return lt + shfl_xor_f(lt, 32);
  }
  // Whether O is finite (a NaN score makes all of it NaN). Products of two: half the
  // instructions, and values of 2^63 may count as infinite, which costs time only.
  __device__ __forceinline__ bool finite() const {
    float z[2] = {0.f, 0.f};
#pragma unroll
    for (int t = 0; t < DP / 16; ++t)
#pragma unroll
      for (int r = 0; r < 2; ++r) z[r] = __builtin_fmaf(o[t][2 * r], o[t][2 * r + 1], z[r]);
    return fabsf(z[0] + z[1]) < INFINITY;
  }
};
// keys at or past lim (counted from the chunk's first) drop out of the softmax
template <int NM> __device__ __forceinline__ void mask_keys(f32x4 (&s)[NM], int lim, int g) {
#pragma unroll
  for (int m = 0; m < NM; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (16 * m + 4 * g + r >= lim) s[m][r] = -INFINITY;
}

// o[d .. d + 3] = acc * inv [* sigmoid(gate)] of a row; inv 0: a row that sees
// nothing, 0 whatever its gate holds
template <typename T> __device__ __forceinline__ void store_row(const CacheArgs &a, const RowInfo &ri, f32x4 acc, float inv, int d) {
  if (d >= a.D) return;
  T *orow = (T *)a.o + ri.b * a.so[0] + ri.hq * a.so[1] + ri.t * a.so[2] + d;
  float y[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = acc[r] * inv;
  if (inv == 0.f) {
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = 0.f;
  } else if (a.og) {
    const T *og = (const T *)a.og + ri.b * a.sog[0] + ri.hq * a.sog[1] + ri.t * a.sog[2] + d;
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] *= 1.f / (1.f + __expf(-to_f32<T>(og[r])));
  }
  if constexpr (sizeof(T) == 4) {
    *(f32x4 *)orow = f32x4{y[0], y[1], y[2], y[3]};
  } else {
    s16x4 pk;
#pragma unroll
    for (int r = 0; r < 4; ++r) pk[r] = bits16<T>((T)y[r]);
    *(s16x4 *)orow = pk;
  }
}

// first row of the own tiles' parts
__device__ __forceinline__ int64_t own_slot(const CacheArgs &a) { return (int64_t)a.Hkv * a.rt_pre * a.np_pre * a.tr_pre; }
template <typename T, int DP, int QT, int NM>
__device__ __forceinline__ void qk_tile(const char *tile, const RowFrag<T, DP> (&fr)[QT], f32x4 (&acc)[QT][NM], int g, int p) {
  constexpr int CPR = DP * (int)sizeof(T) / 16;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt)
#pragma unroll
    for (int m = 0; m < NM; ++m) acc[qt][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  if constexpr (sizeof(T) == 2) {
    constexpr int KS = DP / 32, NK = NM * KS, KL = KS < 4 ? KS : 4, W = NK < 8 ? NK : 8;
    unsigned kb[KL];
#pragma unroll
    for (int l = 0; l < KL; ++l) kb[l] = (unsigned)(uintptr_t)tile + tile_kbase(l, g, p, CPR);
    s16x8 x[NK];
    auto rd = [&](auto K) {
      constexpr int k = decltype(K)::value, m = k / KS, ks = k % KS;
      x[k] = lds_read_b128_at<(ks / 4) * 256 + m * 256 * CPR>(kb[ks % 4]);
    };
    static_for<W>(rd);
    static_for<NK>([&](auto K) {
      constexpr int k = decltype(K)::value;
      constexpr int last = k + W - 1 < NK - 1 ? k + W - 1 : NK - 1;  // last read issued so far
      lds_wait_le<last - k>();
      lds_ready(x[k]);
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) acc[qt][k / KS] = Mfma16<T>::run(x[k], fr[qt].h[k % KS], acc[qt][k / KS]);
      if constexpr (k + W < NK) rd(std::integral_constant<int, k + W>{});
    });
  } else {
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      const int row = 16 * m + p;
#pragma unroll
      for (int ks = 0; ks < DP / 4; ++ks) {
        const float x = *(const float *)(tile + (row * CPR + (ks ^ swz(row, CPR))) * 16 + g * 4);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) acc[qt][m] = mfma_f32_16x16x4(x, fr[qt].f[ks], acc[qt][m]);
        if constexpr (DP >= 256) if (ks % 16 == 15) asm volatile("" ::: "memory");  // at most 16 loads ahead
      }
      if constexpr (DP >= 128) asm volatile("" ::: "memory");
    }
  }
}
template <typename T, int DP, int KC, int QT>
__device__ __forceinline__ void pv_tile(const char *tile, const float (&x)[QT][KC / 16][4], SoftmaxState<DP> (&sm)[QT], int g, int p) {
  constexpr int CPR = DP * (int)sizeof(T) / 16;
  if constexpr (sizeof(T) == 2) {
    constexpr int K2 = KC / 32, NTL = DP / 16, VL = NTL < 8 ? NTL : 8, RPT = 2 * K2, W = NTL < 4 ? NTL : 4;
    s16x8 pk[QT][K2];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int k2 = 0; k2 < K2; ++k2) {
        float y[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) { y[r] = x[qt][2 * k2][r]; y[4 + r] = x[qt][2 * k2 + 1][r]; }
        pk[qt][k2] = pack8<T>(y);
      }
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
        for (int qt = 0; qt < QT; ++qt) sm[qt].o[t] = Mfma16<T>::run(av, pk[qt][k2], sm[qt].o[t]);
      }
      if constexpr (t + W < NTL) rd(std::integral_constant<int, t + W>{});
    });
  } else {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) mm_tr_acc<T, DP, KC>(tile, x[qt], sm[qt].o, g, p);
  }
}

static inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
static inline size_t up256(size_t x) { return (x + 255) / 256 * 256; }

constexpr int kMaxShares = 512;  // np_own + np_pre
constexpr int64_t kCUs = 256;

// Rows of a tile: as many tiles as workgroups of 64 or 128 rows would be, of even
// sizes (160 rows are two tiles of 80, whose spare waves leave the CU to others)
static inline int64_t tile_rows(int dtype, int64_t rows) {
  const int64_t most = dtype == FBSA_F32 || rows <= 64 ? 64 : 128, n = cdiv(rows, most);
  return cdiv(cdiv(rows, n), 16) * 16;
}

}  // namespace fbsa
