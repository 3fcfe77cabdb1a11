// Attention over a cache of keys and values for gfx950 (CDNA4): the newest
// tokens of each sequence over the rows it holds, with or without a prefix that
// every sequence of the batch shares, and the attention weight that each row
// received.
//
// Query t of head h of sequence b sees the prefix rows and its own rows
// s < m(b, t). With x_s = scale q.k_s:  lse = log sum_s exp(x_s),
// p_s = exp(x_s - lse), o = sum_s p_s v_s [* sigmoid(out_gate)], and each own
// row's weight grows by its p_s summed over the group's heads and the tokens.
//
// The query rows that read one KV head (G heads x T tokens of a sequence; for
// the prefix those of every sequence) are stacked, ordered (token, head) so that a
// tile's rows see about the same keys.
//   part     up to 16 rows: a wave per (tile, share of the keys), memory bound
//   tile     more: a workgroup per (64- or 128-row tile, share of the keys)
//   combine, join   a row's parts (unnormalised fp32 O, row maximum, row sum) added
//            in a fixed order; O, lse; after `part` the weights too, from its scores
//   weight, weight_rows  after `tile`: scores formed again, the keys in registers
// Lengths are read on the device; nothing depends on launch order.
#include <math.h>

#include <algorithm>

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

// keys per chunk of a wave's ring: 32; 16 where a row is 512 bytes or more, so that
// more waves fit a CU's LDS
template <typename T, int DP> struct CacheCfg {
  static constexpr int ES = sizeof(T);
  static constexpr int KC = DP * ES >= 512 ? 16 : 32;
  static constexpr int TILE = KC * DP * ES;
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

// Per-lane byte offsets of a copy of a KC-row tile (swizzled chunks) by NW waves;
// columns past the head dim read the row's last chunk.
template <typename T, int DP, int KC, int NW> struct TilePlan {
  static constexpr int ES = sizeof(T), CPR = DP * ES / 16, LPT = KC * CPR / (64 * NW);
  static_assert(LPT * 64 * NW == KC * CPR, "a tile is whole loads of every wave");
  uint32_t off[LPT];
  __device__ __forceinline__ void init(int64_t stride, int D, int w, int lane) {
    const int last = D * ES / 16 - 1;
#pragma unroll
    for (int n = 0; n < LPT; ++n) {
      const int u = (n * NW + w) * 64 + lane, row = u / CPR, c = (u % CPR) ^ swz(row, CPR);
      off[n] = (uint32_t)(((int64_t)row * stride) * ES + (c < last ? c : last) * 16);
    }
  }
  // rows [row0, ...) of a tensor of `rows` rows: rows past the end read its last one
  __device__ __forceinline__ void issue(unsigned st, const char *base, uint32_t row0, uint32_t rows, int64_t step, int rowbytes, int w) const {
    const char *src = base + (int64_t)row0 * step;
    static_assert(KC <= 64, "the strides' limit in check_cache");
    const uint32_t lim = tail_limit<KC>(row0, rows, (uint32_t)step, (uint32_t)rowbytes);
#pragma unroll
    for (int n = 0; n < LPT; ++n) g2lds16_s(src, off[n] > lim ? lim : off[n], st + (n * NW + w) * 1024);
  }
};

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
  // s: raw products (scaled by scale2 > 0 here), masked ones -inf; out: exponentials
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

// ---- infinities. The matrix instructions add 0 * v for every key of a chunk that a
// row does not see, and for the empty half of a split p: NaN where v is infinite or
// NaN; a key's infinities past the head dim's columns do the same to its scores.
// Where a row's O is not finite its share of the keys is therefore gone through once
// more: infinite values are zeros in the products, which are otherwise the same
// instructions in the same order (so finite results are the same bits), and the rows
// that see them get p * v added outside. Finite caches pay for the look at O: over
// 154 shapes up to 8% of a call (4 us of 47), 0.5% in the mean. 262144 rows of 8
// heads, d 64: 105 us finite, 175 with one infinite value, 512 with one in every 64 rows.
template <typename T> __device__ __forceinline__ void zero_infinities(s16x4 &x, bool &any) {
  constexpr short EXP = __is_same(T, bf16) ? 0x7f80 : 0x7c00;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if ((x[e] & EXP) == EXP) {
      x[e] = 0;
      any = true;
    }
}
// the scores of a chunk, as mm_rows_frag and qk_tile form them, without the columns past
// the head dim: copies of the row's last chunk there, whose infinities the query's zeros
// would turn to NaN
template <typename T, int DP, int QT, int NM>
__device__ __forceinline__ void careful_scores(const char *tile, const RowFrag<T, DP> (&fr)[QT], f32x4 (&acc)[QT][NM], int D, int g, int p) {
  constexpr int CPR = DP * (int)sizeof(T) / 16, KS = sizeof(T) == 2 ? DP / 32 : DP / 4, KL = KS < 4 ? KS : 4;
  const char *kb[KL];  // (few addresses and few loads ahead: registers count here, not time)
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int l = 0; l < KL; ++l) kb[l] = tile + tile_kbase(l, g, p, CPR);
  }
#pragma unroll
  for (int m = 0; m < NM; ++m) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) acc[qt][m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if constexpr (sizeof(T) == 2) {
        s16x8 x = *(const s16x8 *)(kb[ks % KL] + (ks / 4) * 256 + m * 256 * CPR);
        if (32 * ks + 8 * g >= D) x = s16x8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) acc[qt][m] = Mfma16<T>::run(x, fr[qt].h[ks], acc[qt][m]);
      } else {
        const float y = *(const float *)(tile + ((16 * m + p) * CPR + (ks ^ swz(p, CPR))) * 16 + g * 4), x = 4 * ks + g < D ? y : 0.f;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) acc[qt][m] = mfma_f32_16x16x4(x, fr[qt].f[ks], acc[qt][m]);
      }
      if (ks % 4 == 3) asm volatile("" ::: "memory");
    }
    asm volatile("" ::: "memory");
  }
}
// sm.o += V^T p of a chunk; row p sees the chunk's keys below lim. SPLIT: p as a pair of 16-bit numbers
template <typename T, int DP, int KC, int QT, bool SPLIT>
__device__ __forceinline__ void careful_values(const char *tile, const float (&x)[QT][KC / 16][4], SoftmaxState<DP> (&sm)[QT],
                                               const int (&lim)[QT], int g, int p) {
  constexpr int CPR = DP * (int)sizeof(T) / 16, NM = KC / 16, K2 = NM / 2;
  bool any = false;
  if constexpr (sizeof(T) == 2) {
    s16x8 pk[QT][K2 ? K2 : 1], pl[QT][K2 ? K2 : 1];
    s16x4 qk[QT], ql[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
      for (int k2 = 0; k2 < K2; ++k2) {
        float y[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) { y[r] = x[qt][2 * k2][r]; y[4 + r] = x[qt][2 * k2 + 1][r]; }
        if constexpr (SPLIT) pack8_split<T>(y, pk[qt][k2], pl[qt][k2]);
        else pk[qt][k2] = pack8<T>(y);
      }
      if constexpr (K2 == 0) pack4_split<T>(x[qt][0], qk[qt], ql[qt]);
    }
    static_assert(K2 > 0 || SPLIT, "16 keys to a chunk: split");
    constexpr int NTL = DP / 16, VL = NTL < 8 ? NTL : 8;
    unsigned vb[VL];
#pragma unroll
    for (int l = 0; l < VL; ++l) vb[l] = (unsigned)(uintptr_t)tile + tile_vbase(l, g, p, CPR);
    static_for<NTL>([&](auto TT) {
      constexpr int t = decltype(TT)::value;
      s16x4 v[NM];
      static_for<NM>([&](auto MM) {
        constexpr int m = decltype(MM)::value;
        v[m] = lds_read_tr16_at<(t / 8) * 256 + m * 256 * CPR>(vb[t % 8]);
      });
      lds_wait_all();
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        lds_ready(v[m]);
        zero_infinities<T>(v[m], any);
      }
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        if constexpr (K2 == 0) {
          sm[qt].o[t] = Mfma16<T>::run16(v[0], qk[qt], sm[qt].o[t]);
          sm[qt].o[t] = Mfma16<T>::run16(v[0], ql[qt], sm[qt].o[t]);
        } else {
#pragma unroll
          for (int half = 0; half < (SPLIT ? 2 : 1); ++half)
#pragma unroll
            for (int k2 = 0; k2 < K2; ++k2) {
              const s16x4 a = v[2 * k2], b = v[2 * k2 + 1];
              const s16x8 av = s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
              sm[qt].o[t] = Mfma16<T>::run(av, half ? pl[qt][k2] : pk[qt][k2], sm[qt].o[t]);
            }
        }
      }
    });
  } else {
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
#pragma unroll
      for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 16 * m + 4 * g + r;
          float a = *(const float *)(tile + (row * CPR + ((4 * t + (p >> 2)) ^ swz(row, CPR))) * 16 + (p & 3) * 4);
          if (!(fabsf(a) < INFINITY)) {
            a = 0.f;
            any = true;
          }
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) sm[qt].o[t] = mfma_f32_16x16x4(a, x[qt][m][r], sm[qt].o[t]);
          if (r == 3) asm volatile("" ::: "memory");
        }
    }
  }
  if (!__ballot(any)) return;
#pragma unroll 1
  for (int key = 0; key < KC; ++key) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float y = 0.f;  // this key's p of row p lies with the row's lane of group key / 4 % 4
#pragma unroll
      for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) y = key >> 4 == m && (key & 3) == r ? x[qt][m][r] : y;
      y = __shfl(y, (key >> 2 & 3) * 16 + p, 64);
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) {
        const int at = (16 * t + 4 * g) * (int)sizeof(T);
        const T *v = (const T *)(tile + (key * CPR + ((at >> 4) ^ swz(key, CPR))) * 16 + (at & 15));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float z = to_f32<T>(v[r]);
          if (key < lim[qt] && !(fabsf(z) < INFINITY)) sm[qt].o[t][r] += y * z;
        }
        asm volatile("" ::: "memory");
      }
    }
  }
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
__device__ __forceinline__ int64_t score_keys(const CacheArgs &a) { return ((int64_t)a.S + 31) / 32 * 32; }
__device__ __forceinline__ int64_t score_row(const CacheArgs &a, int b, int hk, int rho) {
  return (((int64_t)b * a.Hkv + hk) * a.TG + rho) * score_keys(a);
}

// ---- few rows (16 or fewer): a wave per (tile, share of the keys). K and V stream
// global -> LDS through a two-stage ring of the wave's own, so no wave waits for
// another; P enters the value product as a pair of 16-bit numbers (the matrix
// units are idle anyway: busy 5 to 7% of the time), online softmax in the log2
// domain, and where weights are wanted the scores are stored (4 bytes a row and key
// against 2 D to read the key again). Bound by memory: one token over 262144 rows, 8
// heads, d 64, 94 us, 5.7 TB/s; 32 sequences of 1000 to 8192 rows, 16 heads over 2, d 256,
// with weights, 61 to 63 us, 5.1 TB/s. A third and fourth stage changed nothing (d
// 256, 16 keys), nor did equal numbers of chunks to every wave whatever caches they
// lie in (85.8 -> 88.8 us a call: a wave that crosses caches starts its ring anew).
template <typename T, int DP> __global__ __launch_bounds__(64) void cache_part_kernel(CacheArgs a) {
  using C = CacheCfg<T, DP>;
  constexpr int KC = C::KC, NM = KC / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x, g = lane >> 4, p = lane & 15;
  const uint32_t npre = a.few_pre ? (uint32_t)a.Hkv * a.np_pre * a.rt_pre : 0;
  uint32_t id = blockIdx.x;
  const bool pre = id < npre;
  RowInfo ri;
  float *score = nullptr;  // this row's scores, where the weights are taken from them
  int64_t slot;  // the tile's first row among the parts
  int split, np, keys, low;  // keys that any row sees; below `low` every row sees every key
  const char *kb, *vb;
  int64_t kstep, vstep;
  if (pre) {
    const int tile = id % a.rt_pre, hk = id / a.rt_pre / a.np_pre;
    split = id / a.rt_pre % a.np_pre;
    np = a.np_pre;
    const uint32_t rho = tile * 16 + p, rows = (uint32_t)a.B * a.TG, x = rho < rows ? rho : 0;  // (below 2^31)
    ri = row_info(a, (int)(x / (uint32_t)a.TG), hk, (int)(x % (uint32_t)a.TG));
    ri.valid = ri.valid && rho < rows;
    ri.lim = keys = low = a.P;
    slot = (((int64_t)hk * a.rt_pre + tile) * np + split) * 16;
    kstep = a.skp[1] * C::ES;
    vstep = a.svp[1] * C::ES;
    kb = (const char *)a.kp + hk * a.skp[0] * C::ES;
    vb = (const char *)a.vp + hk * a.svp[0] * C::ES;
  } else {
    id -= npre;
    const int tile = id % a.rt_own, hk = id / a.rt_own / a.np_own % a.Hkv, b = id / a.rt_own / a.np_own / a.Hkv;
    split = id / a.rt_own % a.np_own;
    np = a.np_own;
    ri = row_info(a, b, hk, tile * 16 + p);
    own_bounds(a, b, tile * 16, min(tile * 16 + 16, a.TG), keys, low);
    if (a.sc) score = a.sc + score_row(a, b, hk, ri.valid ? p : 0);
    slot = own_slot(a) + (((int64_t)b * a.Hkv + hk) * a.rt_own + tile) * np * 16 + split * 16;
    kstep = a.sk[2] * C::ES;
    vstep = a.sv[2] * C::ES;
    kb = (const char *)a.k + (b * a.sk[0] + hk * a.sk[1]) * C::ES;
    vb = (const char *)a.v + (b * a.sv[0] + hk * a.sv[1]) * C::ES;
  }
  // (a row that is none -- past the end, or past the sequence's new tokens -- sees
  // what the tile sees, so that it asks for no masking; the combine drops it)
  const int lim = ri.valid ? ri.lim : keys;
  int c0, c1;
  share_of((keys + KC - 1) / KC, split, np, c0, c1);

  RowFrag<T, DP> fr;
  load_frag<T, DP>(fr, (const T *)a.q + ri.b * a.sq[0] + ri.hq * a.sq[1] + ri.t * a.sq[2], g, a);
  TilePlan<T, DP, KC, 1> pk, pv;
  pk.init(kstep / C::ES, a.D, 0, lane);
  pv.init(vstep / C::ES, a.D, 0, lane);
  auto issue = [&](int c) {
    const unsigned st = (unsigned)(uintptr_t)smem + (c & 1) * 2 * C::TILE;
    pk.issue(st, kb, (uint32_t)c * KC, keys, kstep, a.D * C::ES, 0);
    pv.issue(st + C::TILE, vb, (uint32_t)c * KC, keys, vstep, a.D * C::ES, 0);
  };

  auto store_scores = [&](int c, const f32x4 (&s)[NM]) {
    if (score && ri.valid) {
#pragma unroll
      for (int m = 0; m < NM; ++m) *(f32x4 *)(score + (int64_t)c * KC + 16 * m + 4 * g) = s[m] * a.scale2;
    }
  };

  SoftmaxState<DP> sm;
  sm.init();
  if (c0 < c1) issue(c0);
  wait_vmcnt<0>();  // the query rows too: the compiler then waits for nothing in the loop
  for (int c = c0; c < c1; ++c) {
    wait_vmcnt<0>();
    lds_wait_all();  // the previous chunk's reads, whose stage is written next
    if (c + 1 < c1) issue(c + 1);
    const char *Ks = smem + (c & 1) * 2 * C::TILE, *Vs = Ks + C::TILE;
    f32x4 s[NM];
    mm_rows_frag<T, DP, NM>(Ks, fr, s, g, p);
    if ((c + 1) * (int64_t)KC > low) mask_keys<NM>(s, lim - c * KC, g);
    store_scores(c, s);
    float x[NM][4];
    sm.template step<NM>(s, a.scale2, x);
    mm_tr_acc<T, DP, KC, 0, sizeof(T) == 2>(Vs, x, sm.o, g, p);
  }

  if (__builtin_expect(__ballot(ri.valid && !sm.finite()) != 0, 0)) {
    RowFrag<T, DP> frs[1] = {fr};
    // (addresses of its own: shared with the loop above they would cost that its
    // registers: fp32, d 256, 34372 keys 227 us, 190 so)
    int gg = g, pp = p;
    asm volatile("" : "+v"(gg), "+v"(pp));
    SoftmaxState<DP> sms[1];
    sms[0].init();
    lds_wait_all();  // the last chunk's reads, whose stage may be written first
    if (c0 < c1) issue(c0);
    for (int c = c0; c < c1; ++c) {
      wait_vmcnt<0>();
      lds_wait_all();
      if (c + 1 < c1) issue(c + 1);
      const char *Ks = smem + (c & 1) * 2 * C::TILE, *Vs = Ks + C::TILE;
      f32x4 s[1][NM];
      careful_scores<T, DP, 1, NM>(Ks, frs, s, a.D, gg, pp);
      mask_keys<NM>(s[0], lim - c * KC, g);
      store_scores(c, s[0]);
      float x[1][NM][4];
      sms[0].template step<NM>(s[0], a.scale2, x[0]);
      careful_values<T, DP, KC, 1, true>(Vs, x, sms, {lim - c * KC}, gg, pp);
    }
    sm = sms[0];
  }

  const float lt = sm.total();
  if (g == 0) a.stat[slot + p] = float2{sm.m, lt};
  if (ri.valid && lt != 0.f) {  // (a NaN sum is kept)
    float *dst = a.part + (slot + p) * DP;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) *(f32x4 *)(dst + 16 * t + 4 * g) = sm.o[t];
  }
}

// ---- many rows: a workgroup per (tile of NW x 16 QT rows, share of the keys).
// The K and V chunks are shared through a ring in LDS; each wave owns QT
// 16-row fragments, and a fragment of K or V read from LDS feeds QT products.
// P enters the value product rounded to the operand type, as in the block-sparse
// forward; the row sums are of the unrounded values. The bf16 results are then off by
// 0.0023 in relative L2, where their own rounding is 0.0017; P as a pair, as for up to
// 16 rows, would leave 0.0017 and take 12 to 25% more time (2048 tokens over 16301 rows
// 762 -> 914 us a call, 64 sequences behind 16301 shared rows 47 -> 53).
// Measured: 2048 tokens over 16301 rows, 16 heads over 2, d 256: 525 to 560 us, 0.92 to
// 0.98 PFLOP/s (matrix units and LDS each busy 47% of the time: eight waves in step
// at one barrier per 64 keys; 32 keys a chunk 610 us; four waves of 32 rows, one to a
// SIMD, 789). 512 rows a head over 16301 keys, beside 64 own caches: 40 us, of which
// about 17 are the chunks and the rest the start, 33 MB of parts and the own caches.
// 160 rows a head over 65536 keys, d 64: 44 us, exponentials and their like at half
// the vector issue.
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

template <typename T, int DP, int NW, int QT, int KC> struct TileCfg {
  static constexpr int ES = sizeof(T), TILE = KC * DP * ES, RING = 2 * 2 * TILE, LDS = RING + NW * 4;
  static_assert(LDS <= 160 * 1024, "LDS");
};

// (d 32: registers for three waves to a SIMD, as the loop needs, also where the second
// look would take more: 448 rows a head over 22876 keys 19.2 us against 21.3)
template <typename T, int DP, int NW, int QT, int KC>
__global__ __launch_bounds__(NW * 64, DP == 32 ? 3 : 1) void cache_tile_kernel(CacheArgs a, int64_t npre) {
  using C = TileCfg<T, DP, NW, QT, KC>;
  constexpr int NM = KC / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, p = lane & 15;
  const bool pre = blockIdx.x < npre;
  const int tr = pre ? a.tr_pre : a.tr_own;  // rows of a tile: the waves past them only load
  RowInfo ri[QT];
  int64_t slot;  // the tile's first row among the parts
  int split, np, keys, low;  // keys that any row sees; below `low` every row of the wave sees every key
  const char *kb, *vb;
  int64_t kstep, vstep;
  if (pre) {
    // (the tiles that share a share's keys run together on one XCD)
    const uint32_t id = (uint32_t)xcd_remap(blockIdx.x, npre);
    const int tile = id % a.rt_pre, hk = id / a.rt_pre / a.np_pre;
    split = id / a.rt_pre % a.np_pre;
    np = a.np_pre;
    const uint32_t rows = (uint32_t)a.B * a.TG;  // (below 2^31)
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const uint32_t rho = (uint32_t)tile * tr + (w * QT + qt) * 16 + p, x = rho < rows ? rho : 0;
      ri[qt] = row_info(a, (int)(x / (uint32_t)a.TG), hk, (int)(x % (uint32_t)a.TG));
      ri[qt].valid = ri[qt].valid && rho < rows && (w * QT + qt) * 16 < tr;
      ri[qt].lim = a.P;
    }
    keys = low = a.P;
    slot = (((int64_t)hk * a.rt_pre + tile) * np + split) * tr;
    kstep = a.skp[1] * C::ES;
    vstep = a.svp[1] * C::ES;
    kb = (const char *)a.kp + hk * a.skp[0] * C::ES;
    vb = (const char *)a.vp + hk * a.svp[0] * C::ES;
  } else {
    // (the last tokens' tiles see the most keys: they start first)
    const uint32_t id = blockIdx.x - (uint32_t)npre, per = (uint32_t)(a.Hkv * a.np_own * a.B), u = id % per;
    const int tile = a.rt_own - 1 - (int)(id / per), hk = u / a.np_own % a.Hkv, b = u / a.np_own / a.Hkv;
    split = u % a.np_own;
    np = a.np_own;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      ri[qt] = row_info(a, b, hk, tile * tr + (w * QT + qt) * 16 + p);
      ri[qt].valid = ri[qt].valid && (w * QT + qt) * 16 < tr;
    }
    own_bounds(a, b, tile * tr, min(tile * tr + tr, a.TG), keys, low);
    const int r0 = tile * tr + w * QT * 16;  // (the wave's first row: from it on, the later rows see more)
    if (w > 0 && r0 < a.TG) {
      int k;
      own_bounds(a, b, r0, a.TG, k, low);
      low = min(low, keys);
    }
    slot = own_slot(a) + ((((int64_t)b * a.Hkv + hk) * a.rt_own + tile) * np + split) * tr;
    kstep = a.sk[2] * C::ES;
    vstep = a.sv[2] * C::ES;
    kb = (const char *)a.k + (b * a.sk[0] + hk * a.sk[1]) * C::ES;
    vb = (const char *)a.v + (b * a.sv[0] + hk * a.sv[1]) * C::ES;
  }
  int c0, c1;
  share_of((keys + KC - 1) / KC, split, np, c0, c1);

  RowFrag<T, DP> fr[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt)
    load_frag<T, DP>(fr[qt], (const T *)a.q + ri[qt].b * a.sq[0] + ri[qt].hq * a.sq[1] + ri[qt].t * a.sq[2], g, a);
  TilePlan<T, DP, KC, NW> pk, pv;
  pk.init(kstep / C::ES, a.D, w, lane);
  pv.init(vstep / C::ES, a.D, w, lane);
  int ist = 0, cst = 0;  // ring places to fill and to read
  auto issue = [&](int c) {
    const unsigned st = (unsigned)(uintptr_t)smem + ist * 2 * C::TILE;
    pk.issue(st, kb, (uint32_t)c * KC, keys, kstep, a.D * C::ES, w);
    pv.issue(st + C::TILE, vb, (uint32_t)c * KC, keys, vstep, a.D * C::ES, w);
    ist ^= 1;
  };
  auto store_scores = [&](int c, const f32x4 (&s)[NM]) {
    if (!pre && a.sc && ri[0].valid) {  // (one tile of up to 16 rows: the first fragment)
      float *score = a.sc + score_row(a, ri[0].b, ri[0].hq / a.G, p);
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        const int64_t key = (int64_t)c * KC + 16 * m + 4 * g;
        if (key < score_keys(a)) *(f32x4 *)(score + key) = s[m] * a.scale2;
      }
    }
  };
  SoftmaxState<DP> sm[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) sm[qt].init();

  if (c0 < c1) issue(c0);
  wait_vmcnt<0>();  // the query rows too: the compiler then waits for nothing in the loop
  for (int c = c0; c < c1; ++c) {
    wait_vmcnt<0>();
    // every wave's part of chunk c has landed, and every wave has read chunk c - 1, whose place is filled next
    lds_barrier();
    if (c + 1 < c1) issue(c + 1);
    const char *Ks = smem + cst * 2 * C::TILE, *Vs = Ks + C::TILE;
    cst ^= 1;
    if (w * QT * 16 >= tr) continue;
    f32x4 s[QT][NM];
    qk_tile<T, DP, QT, NM>(Ks, fr, s, g, p);
    if ((c + 1) * (int64_t)KC > low) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) mask_keys<NM>(s[qt], (ri[qt].valid ? ri[qt].lim : keys) - c * KC, g);
    }
    store_scores(c, s[0]);
    float x[QT][NM][4];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) sm[qt].template step<NM>(s[qt], a.scale2, x[qt]);
    pv_tile<T, DP, KC, QT>(Vs, x, sm, g, p);
  }

  bool bad = false;
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) bad = bad || (ri[qt].valid && !sm[qt].finite());
  // (the chunks are every wave's: all go through them again if one has to)
  uint32_t *vote = (uint32_t *)(smem + C::RING);
  bad = __ballot(bad) != 0;
  if (lane == 0) vote[w] = bad;
  lds_barrier();
  if (__builtin_expect(__ballot(vote[lane % NW] != 0) != 0, 0)) {
    SoftmaxState<DP> sm2[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) sm2[qt].init();
    int gg = g, pp = p;
    asm volatile("" : "+v"(gg), "+v"(pp));  // (as above)
    ist = cst = 0;
    if (c0 < c1) issue(c0);
    for (int c = c0; c < c1; ++c) {
      wait_vmcnt<0>();
      lds_barrier();
      if (c + 1 < c1) issue(c + 1);
      const char *Ks = smem + cst * 2 * C::TILE, *Vs = Ks + C::TILE;
      cst ^= 1;
      if (w * QT * 16 >= tr) continue;
      f32x4 s[QT][NM];
      careful_scores<T, DP, QT, NM>(Ks, fr, s, a.D, gg, pp);
      float x[QT][NM][4];
      int lim[QT];
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        lim[qt] = (ri[qt].valid ? ri[qt].lim : keys) - c * KC;
        mask_keys<NM>(s[qt], lim[qt], g);
        if (qt == 0) store_scores(c, s[0]);
        sm2[qt].template step<NM>(s[qt], a.scale2, x[qt]);
      }
      careful_values<T, DP, KC, QT, false>(Vs, x, sm2, lim, gg, pp);
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) sm[qt] = sm2[qt];
  }

#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int i = (w * QT + qt) * 16 + p;
    if (i >= tr) continue;
    const float lt = sm[qt].total();
    if (!pre && a.direct) {
      const int rho = (a.rt_own - 1 - (int)((blockIdx.x - (uint32_t)npre) / (uint32_t)(a.Hkv * a.np_own * a.B))) * tr + i;
      if (rho >= a.TG) continue;
      const float l = ri[qt].valid ? lt : 0.f, inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) store_row<T>(a, ri[qt], ri[qt].valid ? sm[qt].o[t] : f32x4{0.f, 0.f, 0.f, 0.f}, inv, 16 * t + 4 * g);
      if (g == 0) {
        const float l2 = l == 0.f ? -INFINITY : sm[qt].m + __log2f(l);
        if (a.lse) a.lse[((int64_t)ri[qt].b * a.Hq + ri[qt].hq) * a.T + ri[qt].t] = l2 * kLn2;
        if (a.lse2) a.lse2[((int64_t)ri[qt].b * a.Hkv + ri[qt].hq / a.G) * a.TG + rho] = l == 0.f ? INFINITY : l2;
      }
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

// A row's parts: number i of its prefix tile's shares, then of its own tile's.
struct RowParts {
  int64_t pre0, own0;
  int npre, n;
  __device__ __forceinline__ int64_t at(const CacheArgs &a, int i) const {
    return i < npre ? pre0 + (int64_t)i * a.tr_pre : own0 + (int64_t)(i - npre) * a.tr_own;
  }
};
__device__ __forceinline__ RowParts row_parts(const CacheArgs &a, int b, int hk, int rho) {
  RowParts r;
  const uint32_t rp = (uint32_t)b * a.TG + rho, tr = a.tr_pre;  // (B * TG is below 2^31)
  r.npre = a.np_pre;
  r.n = a.np_pre + a.np_own;
  r.pre0 = a.np_pre ? ((int64_t)hk * a.rt_pre + rp / tr) * a.np_pre * tr + rp % tr : 0;
  r.own0 = own_slot(a) + (((int64_t)b * a.Hkv + hk) * a.rt_own + rho / a.tr_own) * a.np_own * a.tr_own + rho % a.tr_own;
  return r;
}

// A wave per row, where rows are many (12480 rows of few parts, d 64: 49 us a call
// with a workgroup each, 34 so): DP / 4 lanes to a part, so 64 / (DP / 4)
// parts at a time; their sums are joined across the lanes in order.
template <typename T, int DP> __global__ __launch_bounds__(256) void cache_join_kernel(CacheArgs a) {
  constexpr int LG = DP / 4, NG = 64 / LG;
  const int lane = threadIdx.x & 63;
  const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6), rows = (uint32_t)a.B * a.Hkv * a.TG;
  if (row >= rows) return;
  const int rho = (int)(row % a.TG), hk = (int)(row / a.TG % a.Hkv), b = (int)(row / a.TG / a.Hkv);
  const RowInfo ri = row_info(a, b, hk, rho);
  const RowParts rp = row_parts(a, b, hk, rho);
  const int n = ri.valid ? rp.n : 0, gi = lane / LG, e = lane % LG;
  float m = -INFINITY;
  for (int i = lane; i < n; i += 64) m = fmaxf(m, a.stat[rp.at(a, i)].x);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, shfl_xor_f(m, x));
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int i = gi; i < n; i += NG) {
    const int64_t at = rp.at(a, i);
    const float2 st = a.stat[at];
    if (st.y != 0.f) {  // (a part of no keys has no O)
      const float f = __builtin_amdgcn_exp2f(st.x - ref);
      l += f * st.y;
      acc += f * *(const f32x4 *)(a.part + at * DP + 4 * e);
    }
  }
#pragma unroll
  for (int x = LG; x < 64; x <<= 1) {
    l += shfl_xor_f(l, x);
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] += shfl_xor_f(acc[r], x);
  }
  if (gi == 0) store_row<T>(a, ri, acc, l == 0.f ? 0.f : 1.f / l, 4 * e);
  if (lane == 0) {
    const float l2 = l == 0.f ? -INFINITY : m + __log2f(l);
    if (a.lse) a.lse[((int64_t)b * a.Hq + ri.hq) * a.T + ri.t] = l2 * kLn2;
    if (a.lse2) a.lse2[row] = l == 0.f ? INFINITY : l2;
  }
}

constexpr int kMaxShares = 512;    // np_own + np_pre
constexpr int kWeightKeys = 1024;  // keys of a weight workgroup

// Bound by latency: a few microseconds for any few rows; 512 rows of 32 parts, d 256,
// with 64 caches' weights 9.4 us.
// Workgroups [0, rows): a row each. Groups of DP / 4 threads take every NG-th
// part, a float4 a thread, and are added in order at the end.
// Workgroups past them (WEIGHT): kWeightKeys keys of a (sequence, KV head): each row's
// lse from its parts' statistics, then weight + sum over rows of exp2(score - lse).
template <typename T, int DP, bool WEIGHT> __global__ __launch_bounds__(256) void cache_combine_kernel(CacheArgs a) {
  constexpr int LG = DP / 4, NG = 256 / LG;
  __shared__ float s_f[kMaxShares];
  __shared__ f32x4 s_acc[256];
  __shared__ float s_red[8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t rows = (uint32_t)a.B * a.Hkv * a.TG;
  if (WEIGHT && blockIdx.x >= rows) {
    const uint32_t per = (uint32_t)(a.S + kWeightKeys - 1) / kWeightKeys, u = blockIdx.x - rows;
    const int key0 = (int)(u % per) * kWeightKeys, hk = (int)(u / per % a.Hkv), b = (int)(u / per / a.Hkv);
    const int n = seq_len(a, b), c = seq_count(a, b);
    if (key0 >= n) return;
    __shared__ float s_lse[16];
    const int real = min(c * a.G, a.TG);  // rows of real queries
    const float *sc = a.sc + score_row(a, b, hk, 0);
    const int64_t step = score_row(a, 0, 0, 1);
    // four keys a thread, four rows' scores in flight (rows of scores are whole
    // multiples of 32); the first and the weights are asked for before the lse is known
    static_assert(kWeightKeys == 4 * 256, "four keys to a thread");
    const int key = key0 + 4 * tid, at = key < n ? key : key0;
    f32x4 x[4], w = f32x4{0.f, 0.f, 0.f, 0.f};
    auto load = [&](int r0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = *(const f32x4 *)(sc + (r0 + j < real ? r0 + j : r0) * step + at);
    };
    if (real) load(0);
    float w0[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w0[e] = a.w && key + e < n ? a.w[b * a.sw[0] + hk * a.sw[1] + key + e] : 0.f;
    // 16 lanes a row: the parts' statistics joined as they come
    {
      const int rho = tid >> 4;
      float m = -INFINITY, l = 0.f;
      auto join = [&](float m2, float l2) {
        if (l2 == 0.f) return;
        const float mn = fmaxf(m, m2);
        l = l * __builtin_amdgcn_exp2f(m - mn) + l2 * __builtin_amdgcn_exp2f(m2 - mn);
        m = mn;
      };
      if (rho < real) {
        const RowParts rp = row_parts(a, b, hk, rho);
        for (int i = tid & 15; i < rp.n; i += 16) {
          const float2 st = a.stat[rp.at(a, i)];
          join(st.x, st.y);
        }
      }
#pragma unroll
      for (int y = 1; y < 16; y <<= 1) {
        const float m2 = shfl_xor_f(m, y), l2 = shfl_xor_f(l, y);
        join(m2, l2);
      }
      if ((tid & 15) == 0) s_lse[rho] = l == 0.f ? -INFINITY : m + __log2f(l);
    }
    __syncthreads();
    if (key >= n) return;
    for (int r0 = 0; r0 < real; r0 += 4) {
      if (r0) load(r0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float l2 = r0 + j < real ? s_lse[r0 + j] : -INFINITY;
        // (a row's scores are written up to the last key that a row of its tile sees)
        const int64_t lim = (int64_t)n - c + (r0 + j) / a.G + 1;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (key + e < lim && l2 != -INFINITY) w[e] += __builtin_amdgcn_exp2f(x[j][e] - l2);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (key + e < n) a.wo[b * a.swo[0] + hk * a.swo[1] + key + e] = w0[e] + w[e];
    return;
  }
  const int rho = (int)(blockIdx.x % a.TG), hk = (int)(blockIdx.x / a.TG % a.Hkv), b = (int)(blockIdx.x / a.TG / a.Hkv);
  const RowInfo ri = row_info(a, b, hk, rho);
  const RowParts rp = row_parts(a, b, hk, rho);
  const int n = ri.valid ? rp.n : 0;
  // the first parts are asked for before their statistics are known
  constexpr int U = 4;
  const int gi = tid / LG, e = tid % LG;
  f32x4 ahead[U];
#pragma unroll
  for (int j = 0; j < U; ++j)
    if (gi + j * NG < n) ahead[j] = *(const f32x4 *)(a.part + rp.at(a, gi + j * NG) * DP + 4 * e);
  static_assert(kMaxShares <= 2 * 256, "two parts to a thread");
  float2 st[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) st[j] = tid + 256 * j < n ? a.stat[rp.at(a, tid + 256 * j)] : float2{-INFINITY, 0.f};
  float m = fmaxf(st[0].x, st[1].x);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, shfl_xor_f(m, x));
  if (lane == 0) s_red[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float f = st[j].y == 0.f ? -1.f : __builtin_amdgcn_exp2f(st[j].x - ref);  // (-1: a part of no keys has no O)
    if (st[j].y != 0.f) l += f * st[j].y;
    if (tid + 256 * j < n) s_f[tid + 256 * j] = f;
  }
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) l += shfl_xor_f(l, x);
  if (lane == 0) s_red[4 + wave] = l;
  __syncthreads();
  l = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < U; ++j)
    if (gi + j * NG < n) {
      const float f = s_f[gi + j * NG];
      if (f != -1.f) acc += f * ahead[j];
    }
  // (loads of several parts in flight: one that was not written is loaded and left out)
  for (int i = gi + U * NG; i < n; i += U * NG) {
    f32x4 y[U];
#pragma unroll
    for (int j = 0; j < U; ++j) y[j] = *(const f32x4 *)(a.part + rp.at(a, i + j * NG < n ? i + j * NG : i) * DP + 4 * e);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const float f = i + j * NG < n ? s_f[i + j * NG] : -1.f;
      if (f != -1.f) acc += f * y[j];
    }
  }
  s_acc[tid] = acc;
  __syncthreads();
  if (tid < LG) {
    for (int j = 1; j < NG; ++j) acc += s_acc[j * LG + tid];
    const float inv = l == 0.f ? 0.f : 1.f / l;
    store_row<T>(a, ri, acc, inv, 4 * tid);
  }
  if (tid == 0) {
    const float l2 = l == 0.f ? -INFINITY : m + __log2f(l);
    if (a.lse) a.lse[((int64_t)b * a.Hq + ri.hq) * a.T + ri.t] = l2 * kLn2;
    if (a.lse2) a.lse2[blockIdx.x] = l == 0.f ? INFINITY : l2;
  }
}

// ---- weights of many rows: p = exp2(score - lse) summed over the rows that see a
// key, scores formed again. A workgroup per 256 keys (fp32: 128) of a (sequence, KV
// head) and share of its rows: the keys stay in registers (64 to a wave, fp32 32, B
// operands), the query rows stream through a ring in LDS, a chunk's first half to
// waves 0-3 and its second to waves 4-7. A lane holds one column, a key, of the
// product, so the sum over rows is a register each. Row rho is token rho / G;
// key j is seen by the rows from G * (j - (len - count)) on. 2048 tokens over 16301
// rows, 16 heads over 2, d 256: 274 us, 0.94 PFLOP/s of these products (vector issue
// 57%, matrix units 44% busy).
template <typename T, int DP> struct WeightCfg {
  static constexpr int ES = sizeof(T), NT = 512, CPR = DP * ES / 16;
  // 16-key fragments of a wave: a row fragment read from LDS feeds KF products
  // (2048 tokens over 16301 rows, 16 heads over 2, d 256: KF 4 with 64 rows 286 us,
  // KF 2 with 128 rows 323, with 64 364); fp32 has registers for two
  static constexpr int KF = ES == 2 ? 4 : 2, KEYS = 4 * 16 * KF;
  static_assert(KEYS == (ES == 2 ? 256 : 128), "the launch's limit in check_cache");
  static constexpr int ROWS = DP * ES * KF <= 1024 ? 128 : 64, NM = ROWS / 32;  // NM 16-row tiles to a half
  static constexpr int LPT = ROWS * CPR / NT;        // 16-byte loads per thread and chunk
  static_assert(LPT * NT == ROWS * CPR, "a chunk is whole loads of every thread");
  static constexpr int STAGE = ROWS * DP * ES + ROWS * 4, LDS = 2 * STAGE;
};
template <typename T, int DP> __global__ __launch_bounds__(512) void cache_weight_kernel(CacheArgs a) {
  using C = WeightCfg<T, DP>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float s_sum[C::KEYS];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, p = lane & 15;
  const int kg = w & 3, half = w >> 2;
  const int hk = blockIdx.y % a.Hkv, b = blockIdx.y / a.Hkv;
  const int n = seq_len(a, b), cnt = seq_count(a, b), real = cnt * a.G;
  const int64_t key064 = (int64_t)blockIdx.x * C::KEYS;
  if (key064 >= n) return;
  const int key0 = (int)key064;

  // this wave's keys (a key past the length: the last one's values, not stored)
  RowFrag<T, DP> fr[C::KF];
  int first[C::KF];  // the first row that sees this lane's key
  const int64_t old = (int64_t)n - cnt;  // rows of the cache before the new tokens (negative: tokens before its start)
  auto first_row = [&](int64_t key) {
    const int64_t r = (key - old) * a.G;
    return (int)(r < 0 ? 0 : r > real ? real : r);
  };
#pragma unroll
  for (int f = 0; f < C::KF; ++f) {
    const int key = key0 + (kg * C::KF + f) * 16 + p, at = key < n ? key : n - 1;
    // (the keys take the query's sign, and zeros past the head dim)
    load_frag<T, DP>(fr[f], (const T *)a.k + b * a.sk[0] + hk * a.sk[1] + at * a.sk[2], g, a);
    first[f] = first_row(key);
  }
  const int r0 = first_row(key0) / C::ROWS * C::ROWS;
  const int nc = r0 < real ? (real - r0 + C::ROWS - 1) / C::ROWS : 0;
  const int c0 = (int)((int64_t)nc * blockIdx.z / gridDim.z), c1 = (int)((int64_t)nc * (blockIdx.z + 1) / gridDim.z);

  // loads of this thread: row and chunk within the stage, and the row's place in q,
  // stepped by a chunk at a time
  int rho[C::LPT], gg[C::LPT];
  int64_t off[C::LPT];
  const int last = a.D * C::ES / 16 - 1;
  const int dt = C::ROWS / a.G, dg = C::ROWS % a.G;
  const int64_t sh = a.sq[1] * C::ES, st = a.sq[2] * C::ES;
#pragma unroll
  for (int x = 0; x < C::LPT; ++x) {
    const int u = x * C::NT + tid, row = u / C::CPR, c = (u % C::CPR) ^ swz(row, C::CPR);
    rho[x] = r0 + c0 * C::ROWS + row;
    gg[x] = rho[x] % a.G;
    off[x] = (int64_t)(rho[x] / a.G) * st + gg[x] * sh + (c < last ? c : last) * 16;
  }
  const char *qb = (const char *)a.q + (b * a.sq[0] + (int64_t)hk * a.G * a.sq[1]) * C::ES;
  const float *lse = a.lse2 + ((int64_t)b * a.Hkv + hk) * a.TG;
  int ist = 0, cst = 0;
  auto issue = [&](int c) {
    char *stage = smem + ist * C::STAGE;
    ist ^= 1;
#pragma unroll
    for (int x = 0; x < C::LPT; ++x) {
      // (rows past the last real one: the first row's values, left out of the sums)
      g2lds16(qb + (rho[x] < real ? off[x] : 0), stage + (x * C::NT + w * 64) * 16);
      rho[x] += C::ROWS;
      gg[x] += dg;
      off[x] += dt * st + dg * sh;
      if (gg[x] >= a.G) {
        gg[x] -= a.G;
        off[x] += st - a.G * sh;
      }
    }
    if (w * 64 < C::ROWS) {
      const int r = r0 + c * C::ROWS + w * 64 + lane;
      g2lds4(lse + (r < real ? r : 0), stage + C::ROWS * DP * C::ES + w * 256);
    }
  };
  float sum[C::KF];
#pragma unroll
  for (int f = 0; f < C::KF; ++f) sum[f] = 0.f;
  const int most = first_row((int64_t)key0 + (kg + 1) * C::KF * 16 - 1);  // from here on every key of the wave is seen
  if (c0 < c1) issue(c0);
  wait_vmcnt<0>();  // the keys too: the compiler then waits for nothing in the loop
  for (int c = c0; c < c1; ++c) {
    wait_vmcnt<0>();
    lds_barrier();
    if (c + 1 < c1) issue(c + 1);
    const char *stage = smem + cst * C::STAGE, *tile = stage + half * 16 * C::NM * DP * C::ES;
    cst ^= 1;
    const int row0 = r0 + c * C::ROWS + half * 16 * C::NM;
    f32x4 l2[C::NM], s[C::KF][C::NM];
#pragma unroll
    for (int m = 0; m < C::NM; ++m) l2[m] = *(const f32x4 *)(stage + C::ROWS * DP * C::ES + (half * 16 * C::NM + 16 * m + 4 * g) * 4);
    qk_tile<T, DP, C::KF, C::NM>(tile, fr, s, g, p);
    if (row0 >= most && row0 + 16 * C::NM <= real) {
#pragma unroll
      for (int f = 0; f < C::KF; ++f)
#pragma unroll
        for (int m = 0; m < C::NM; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) sum[f] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[f][m][r], a.scale2, -l2[m][r]));
    } else {
#pragma unroll
      for (int f = 0; f < C::KF; ++f)
#pragma unroll
        for (int m = 0; m < C::NM; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = row0 + 16 * m + 4 * g + r;
            if (row >= first[f] && row < real) sum[f] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[f][m][r], a.scale2, -l2[m][r]));
          }
    }
  }
#pragma unroll
  for (int f = 0; f < C::KF; ++f) {
    sum[f] += shfl_xor_f(sum[f], 16);
    sum[f] += shfl_xor_f(sum[f], 32);
    if (half == 1 && g == 0) s_sum[(kg * C::KF + f) * 16 + p] = sum[f];
  }
  __syncthreads();
  if (half == 1 || g) return;
#pragma unroll
  for (int f = 0; f < C::KF; ++f) {
    const int i = (kg * C::KF + f) * 16 + p, key = key0 + i;
    if (key >= n) continue;
    const float y = sum[f] + s_sum[i];
    if (gridDim.z > 1) {
      a.wpart[((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * a.S + key] = y;
    } else {
      const float w0 = a.w ? a.w[b * a.sw[0] + hk * a.sw[1] + key] : 0.f;
      a.wo[b * a.swo[0] + hk * a.swo[1] + key] = w0 + y;
    }
  }
}
// ---- weights of up to 128 rows: the rows stay in LDS, and each wave streams keys of
// its own, KF fragments at a time straight into registers with the next ones on
// their way, so after the rows are staged no wave waits for another. A place past the
// last row holds that row with an lse of +inf: its probabilities are 0 (zeros there
// would make a NaN of a key's infinities; the last row sees every key, so its own
// scores are NaN where the copy's are). Against the
// kernel above, whose one or two chunks of such rows leave nothing to overlap: 56 rows a
// head over up to 123654 keys, 48 caches, d 32, 216 -> 118 us; 108 rows, d 64, fp32,
// 617 -> 377.
template <typename T, int DP> struct WeightRowsCfg {
  static constexpr int ES = sizeof(T), CPR = DP * ES / 16, MAXROWS = 128;  // (check_cache knows it)
  static constexpr int KF = ES == 2 ? (DP >= 256 ? 2 : 4) : (DP >= 128 ? 1 : 2), KEYS = 16 * KF;
};
template <typename T, int DP> __global__ __launch_bounds__(256) void cache_weight_rows_kernel(CacheArgs a) {
  using C = WeightRowsCfg<T, DP>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, p = lane & 15;
  const int hk = blockIdx.y % a.Hkv, b = blockIdx.y / a.Hkv;
  const int n = seq_len(a, b), cnt = seq_count(a, b), real = cnt * a.G, rp = (a.TG + 31) / 32 * 32;
  int t0, t1;
  share_of((n + C::KEYS - 1) / C::KEYS, blockIdx.x * 4 + w, gridDim.x * 4, t0, t1);
  float *s_lse = (float *)(smem + rp * DP * C::ES);
  for (int u = tid; u < rp * C::CPR; u += 256) {
    const int row = u / C::CPR, c = u % C::CPR;
    u32x4 x = u32x4{0, 0, 0, 0};
    const int at = row < real ? row : real - 1;
    if (real && c * 16 < a.D * C::ES)
      x = *(const u32x4 *)((const T *)a.q + b * a.sq[0] + (hk * a.G + at % a.G) * a.sq[1] + (at / a.G) * a.sq[2] + c * (16 / C::ES));
    *(u32x4 *)(smem + (row * C::CPR + (c ^ swz(row, C::CPR))) * 16) = x;
  }
  for (int row = tid; row < rp; row += 256) s_lse[row] = row < real ? a.lse2[((int64_t)b * a.Hkv + hk) * a.TG + row] : INFINITY;
  RowFrag<T, DP> next[C::KF];
  const T *kb = (const T *)a.k + b * a.sk[0] + hk * a.sk[1];
  // (the keys take the query's sign, and zeros past the head dim; a key past the
  // length is the last one, not stored)
  auto load = [&](int t) {
#pragma unroll
    for (int f = 0; f < C::KF; ++f) {
      const int64_t key = (int64_t)t * C::KEYS + f * 16 + p;
      load_frag<T, DP>(next[f], kb + (key < n ? key : n - 1) * a.sk[2], g, a);
    }
  };
  if (t0 < t1) load(t0);
  __syncthreads();
  const int64_t old = (int64_t)n - cnt;  // rows of the cache before the new tokens
  for (int t = t0; t < t1; ++t) {
    RowFrag<T, DP> fr[C::KF];
    float sum[C::KF], w0[C::KF];
    int64_t first[C::KF];  // the first row that sees this lane's key
#pragma unroll
    for (int f = 0; f < C::KF; ++f) {
      const int64_t key = (int64_t)t * C::KEYS + f * 16 + p;
      fr[f] = next[f];
      sum[f] = 0.f;
      first[f] = (key - old) * a.G;
      w0[f] = a.w && g == 0 && key < n ? a.w[b * a.sw[0] + hk * a.sw[1] + key] : 0.f;
    }
    if (t + 1 < t1) load(t + 1);
    const bool all = (int64_t)(t + 1) * C::KEYS - 1 <= old;  // every row sees every key of the wave's
    for (int r0 = 0; r0 < real; r0 += 32) {
      f32x4 s[C::KF][2], l2[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) l2[m] = *(const f32x4 *)(s_lse + r0 + 16 * m + 4 * g);
      qk_tile<T, DP, C::KF, 2>(smem + r0 * DP * C::ES, fr, s, g, p);
#pragma unroll
      for (int f = 0; f < C::KF; ++f)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[f][m][r], a.scale2, -l2[m][r]));
            if (all || r0 + 16 * m + 4 * g + r >= first[f]) sum[f] += x;
          }
    }
#pragma unroll
    for (int f = 0; f < C::KF; ++f) {
      sum[f] += shfl_xor_f(sum[f], 16);
      sum[f] += shfl_xor_f(sum[f], 32);
      const int64_t key = (int64_t)t * C::KEYS + f * 16 + p;
      if (g == 0 && key < n) a.wo[b * a.swo[0] + hk * a.swo[1] + key] = w0[f] + sum[f];
    }
  }
}

// the row shares' sums, in order
__global__ __launch_bounds__(256) void cache_weight_sum_kernel(CacheArgs a, int shares) {
  const int key = blockIdx.x * 256 + threadIdx.x;
  const int hk = blockIdx.y % a.Hkv, b = blockIdx.y / a.Hkv;
  if (key >= seq_len(a, b)) return;
  float y = 0.f;
  for (int z = 0; z < shares; ++z) y += a.wpart[((int64_t)z * gridDim.y + blockIdx.y) * a.S + key];
  const float w0 = a.w ? a.w[b * a.sw[0] + hk * a.sw[1] + key] : 0.f;
  a.wo[b * a.swo[0] + hk * a.swo[1] + key] = w0 + y;
}

static int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
static size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Tiles and shares of a call, from its sizes alone (lengths are on the device:
// the capacity stands for them).
constexpr int64_t kCUs = 256;

// Rows of a tile: as many tiles as workgroups of 64 or 128 rows would be, of even
// sizes (160 rows are two tiles of 80, whose spare waves leave the CU to others)
static int64_t tile_rows(int dtype, int64_t rows) {
  const int64_t most = dtype == FBSA_F32 || rows <= 64 ? 64 : 128, n = cdiv(rows, most);
  return cdiv(cdiv(rows, n), 16) * 16;
}

struct CachePlan {
  int64_t tr_own, tr_pre, rt_own, rt_pre, np_own, np_pre, rows, DP;
  int64_t nz;  // shares of the rows in the weights of many rows
  bool few_own, few_pre, direct, scores;  // scores: weights from stored scores (16 rows or fewer)
  size_t stat, part, lse2, wpart, sc, total;
};
static CachePlan cache_plan(const fbsa_cache_desc *d) {
  CachePlan p;
  const int64_t G = d->Hq / d->Hkv, TG = d->T * G;
  p.DP = d->D <= 32 ? 32 : d->D <= 64 ? 64 : d->D <= 128 ? 128 : 256;
  const int64_t pre_rows = d->B * TG;
  p.few_pre = pre_rows <= 16;
  // own tiles of few rows and keys beside a prefix that takes the tile kernel: they
  // go into its launch, a tile of 16 rows each, instead of one of their own (64
  // sequences, 16 heads over 2, d 256, up to 512 own rows: 38 us against 43; small
  // batches 25 to 35% less; fp32, whose single wave is slow: 157 us against 107 at
  // 1209 rows, so only short ones)
  const int64_t seqs = d->B * d->Hkv;
  const int64_t beside = std::min({cdiv(d->S, 256), std::max<int64_t>(1, 2 * kCUs / seqs), (int64_t)kMaxShares / 2});
  const bool merge = TG <= 16 && d->P && !p.few_pre && seqs <= 2 * kCUs && cdiv(d->S, beside) <= (d->dtype == FBSA_F32 ? 128 : 1024);
  p.scores = TG <= 16;
  p.few_own = TG <= 16 && !merge;
  p.tr_own = p.scores ? 16 : tile_rows(d->dtype, TG);
  p.tr_pre = p.few_pre ? 16 : tile_rows(d->dtype, pre_rows);
  p.rt_own = cdiv(TG, p.tr_own);
  p.rt_pre = d->P ? cdiv(pre_rows, p.tr_pre) : 0;
  // the wave kernel wants four waves to a CU (d 256: eight), the tile kernel as many workgroups as
  // a CU has room for (d 256: one). A share has at least so many keys that joining it
  // costs less than it saves (swept over some 200 drawn shapes: 16-bit wave tiles 64
  // keys up to 25% under 128, tile kernels 128 up to 30% under 64, fp32 32 up to 30%
  // under 64)
  const int64_t room = kCUs * (p.DP <= 128 ? 2 : 1);
  // (sequences of different lengths want them finer, so that the longest does not hold up the rest)
  auto shares = [&](bool few, bool ragged, int64_t tiles, int64_t keys) {
    const int64_t want = few ? cdiv((p.DP == 256 ? 8 : 4) * kCUs, tiles) : ragged ? cdiv(4 * room, tiles) : tiles >= room ? 1 : room / tiles;
    const int64_t most = cdiv(keys, d->dtype == FBSA_F32 ? 32 : few ? 64 : 128);
    const int64_t n = want < most ? want : most;
    return n < kMaxShares / 2 ? n : kMaxShares / 2;
  };
  p.np_own = merge ? beside : shares(p.few_own, d->B > 1, d->B * d->Hkv * p.rt_own, d->S);
  p.np_pre = d->P ? shares(p.few_pre, false, d->Hkv * p.rt_pre, d->P) : 0;
  p.direct = !p.few_own && !d->P && p.np_own == 1;
  p.rows = d->B * d->Hkv * p.rt_own * p.np_own * p.tr_own + d->Hkv * p.rt_pre * p.np_pre * p.tr_pre;
  // (tiles that write their results have no parts; 32 x 1024 tokens, 32 heads over 8, d 256: 1 GiB of them)
  const size_t parts = p.direct ? 0 : (size_t)p.rows;
  p.stat = 0;
  p.part = up256(parts * 8);
  p.lse2 = p.part + up256(parts * p.DP * 4);
  // (a share is at least four chunks of 64 rows)
  const int64_t wgs = d->B * d->Hkv * cdiv(d->S, d->dtype == FBSA_F32 ? 128 : 256), z = wgs >= kCUs ? 1 : kCUs / wgs, zmax = cdiv(TG, 256);
  p.nz = z < zmax ? z : zmax;
  const bool weight = d->flags & FBSA_CACHE_WEIGHT;
  p.wpart = p.lse2 + (weight && !p.scores ? up256((size_t)(d->B * d->Hkv * TG) * 4) : 0);
  p.sc = p.wpart + (weight && !p.scores && p.nz > 1 ? up256((size_t)p.nz * d->B * d->Hkv * d->S * 4) : 0);
  p.total = p.sc + (weight && p.scores ? up256((size_t)(d->B * d->Hkv * TG) * cdiv(d->S, 32) * 128) : 0);
  if (p.total == 0) p.total = 256;  // (0 says that a descriptor is refused)
  return p;
}

template <typename T, int DP, int NW, int QT, int KC>
static int launch_tiles(const CacheArgs &a, int64_t npre, int64_t nown, hipStream_t s) {
  using C = TileCfg<T, DP, NW, QT, KC>;
  const int e = lds_optin((const void *)cache_tile_kernel<T, DP, NW, QT, KC>, C::LDS, "hipFuncSetAttribute(cache_tile)");
  if (e) return e;
  hipLaunchKernelGGL((cache_tile_kernel<T, DP, NW, QT, KC>), dim3((unsigned)(npre + nown)), dim3(NW * 64), C::LDS, s, a, npre);
  return hip_check(hipGetLastError(), "cache_tile_kernel launch");
}
template <typename T, int DP> static int launch_tiles_of(const CacheArgs &a, int rows, int64_t npre, int64_t nown, hipStream_t s) {
  if constexpr (sizeof(T) == 4) {
    return launch_tiles<T, DP, 4, 1, DP >= 128 ? 16 : 32>(a, npre, nown, s);
  } else {
    if (rows <= 64) return launch_tiles<T, DP, 4, 1, 64>(a, npre, nown, s);
    constexpr int NW = DP == 32 ? 4 : 8;  // (a tile of 64 keys, d 32, is four waves' loads)
    return launch_tiles<T, DP, NW, 8 / NW, 64>(a, npre, nown, s);
  }
}

template <typename T, int DP> static int launch_cache(const CacheArgs &a, int64_t nz, hipStream_t s) {
  using C = CacheCfg<T, DP>;
  const size_t lds = (size_t)2 * 2 * C::TILE;
  int e = lds_optin((const void *)cache_part_kernel<T, DP>, lds, "hipFuncSetAttribute(cache_part)");
  if (e) return e;
  const int64_t rows = (int64_t)a.B * a.Hkv * a.TG;
  const int64_t nown = (int64_t)a.B * a.Hkv * a.rt_own * a.np_own, npre = (int64_t)a.Hkv * a.rt_pre * a.np_pre;
  // prefix and own tiles in one launch where one workgroup size serves both, or
  // where the own ones are few enough to sit beside the others in larger ones (90
  // rows a head over 138 shared keys and up to 728 own: 17 -> 12 us)
  const bool both = npre && !a.few_pre && !a.few_own && (a.TG <= 16 || (a.tr_own <= 64) == (a.tr_pre <= 64) || nown <= 2 * kCUs);
  const int tr = both && a.tr_own > a.tr_pre ? a.tr_own : a.tr_pre;
  if (npre && !a.few_pre && (e = launch_tiles_of<T, DP>(a, tr, npre, both ? nown : 0, s))) return e;
  if (!a.few_own && !both && (e = launch_tiles_of<T, DP>(a, a.tr_own, 0, nown, s))) return e;
  const int64_t parts = (a.few_own ? nown : 0) + (a.few_pre ? npre : 0);
  if (parts) {
    hipLaunchKernelGGL((cache_part_kernel<T, DP>), dim3((unsigned)parts), dim3(64), lds, s, a);
    if ((e = hip_check(hipGetLastError(), "cache_part_kernel launch"))) return e;
  }
  const int64_t wgs = a.sc ? (int64_t)a.B * a.Hkv * cdiv(a.S, kWeightKeys) : 0;
  if (!a.direct) {
    // many rows of few parts: a wave each (1152 rows of 26 parts, d 256: 71 us a call against 60)
    if (!a.sc && (rows >= 16384 || (rows >= 1024 && (a.np_own + a.np_pre) * DP <= 2048)))
      hipLaunchKernelGGL((cache_join_kernel<T, DP>), dim3((unsigned)cdiv(rows, 4)), dim3(256), 0, s, a);
    else if (a.sc)
      hipLaunchKernelGGL((cache_combine_kernel<T, DP, true>), dim3((unsigned)(rows + wgs)), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((cache_combine_kernel<T, DP, false>), dim3((unsigned)rows), dim3(256), 0, s, a);
    if ((e = hip_check(hipGetLastError(), "cache_combine_kernel launch"))) return e;
  }
  if (a.wo && !a.sc && a.TG <= WeightRowsCfg<T, DP>::MAXROWS) {
    using W = WeightRowsCfg<T, DP>;
    const size_t rp = (size_t)cdiv(a.TG, 32) * 32, need = rp * DP * W::ES + rp * 4;
    if ((e = lds_optin((const void *)cache_weight_rows_kernel<T, DP>, need, "hipFuncSetAttribute(cache_weight_rows)"))) return e;
    // eight workgroups a CU (four: up to 7% more on long caches), no more than there are key tiles
    const int64_t seqs = (int64_t)a.B * a.Hkv, wgs = std::min(std::max<int64_t>(1, cdiv(8 * kCUs, seqs)), cdiv(a.S, 4 * W::KEYS));
    hipLaunchKernelGGL((cache_weight_rows_kernel<T, DP>), dim3((unsigned)wgs, (unsigned)seqs), dim3(256), need, s, a);
    e = hip_check(hipGetLastError(), "cache_weight_rows_kernel launch");
  } else if (a.wo && !a.sc) {
    using W = WeightCfg<T, DP>;
    if ((e = lds_optin((const void *)cache_weight_kernel<T, DP>, W::LDS, "hipFuncSetAttribute(cache_weight)"))) return e;
    const unsigned seqs = (unsigned)(a.B * a.Hkv);
    hipLaunchKernelGGL((cache_weight_kernel<T, DP>), dim3((unsigned)cdiv(a.S, W::KEYS), seqs, (unsigned)nz), dim3(W::NT), W::LDS, s, a);
    if ((e = hip_check(hipGetLastError(), "cache_weight_kernel launch"))) return e;
    if (nz > 1) {
      hipLaunchKernelGGL(cache_weight_sum_kernel, dim3((unsigned)cdiv(a.S, 256), seqs), dim3(256), 0, s, a, (int)nz);
      e = hip_check(hipGetLastError(), "cache_weight_sum_kernel launch");
    }
  }
  return e;
}

template <typename T> static int dispatch_cache(const CacheArgs &a, const CachePlan &pl, hipStream_t s) {
  switch (pl.DP) {
    case 32: return launch_cache<T, 32>(a, pl.nz, s);
    case 64: return launch_cache<T, 64>(a, pl.nz, s);
    case 128: return launch_cache<T, 128>(a, pl.nz, s);
    default: return launch_cache<T, 256>(a, pl.nz, s);
  }
}

static bool aligned_to(const void *p, int64_t n) { return (uintptr_t)p % (uintptr_t)n == 0; }

static int check_cache(const fbsa_cache_desc *d) {
  static const char *fn = "fbsa_cache_attn";
  if (!d) return fail(FBSA_EINVAL, "%s: null descriptor", fn);
  if (d->dtype < FBSA_F32 || d->dtype > FBSA_F16) return fail(FBSA_EINVAL, "%s: bad dtype %d", fn, d->dtype);
  if (d->flags & ~FBSA_CACHE_WEIGHT) return fail(FBSA_EINVAL, "%s: unknown flags 0x%x", fn, d->flags);
  if (d->B < 1 || d->Hq < 1 || d->Hkv < 1 || d->T < 1 || d->S < 1 || d->P < 0)
    return fail(FBSA_EINVAL, "%s: sizes must be positive (B=%lld Hq=%lld Hkv=%lld T=%lld S=%lld P=%lld)", fn, (long long)d->B,
                (long long)d->Hq, (long long)d->Hkv, (long long)d->T, (long long)d->S, (long long)d->P);
  if (d->Hq % d->Hkv) return fail(FBSA_EINVAL, "%s: Hq=%lld not a multiple of Hkv=%lld", fn, (long long)d->Hq, (long long)d->Hkv);
  if (d->D < 8 || d->D > 256 || d->D % 8)
    return fail(FBSA_EUNSUPPORTED, "%s: head dim %lld is not a multiple of 8 up to 256", fn, (long long)d->D);
  if (!isfinite(d->scale * kLog2e)) return fail(FBSA_EINVAL, "%s: scale times log2(e) is not finite", fn);
  const int64_t lim = 0x7fff0000LL;
  if (d->S > lim || d->P > lim || d->B > lim || d->Hq > 65535 || d->T > lim || d->T * (d->Hq / d->Hkv) > lim ||
      d->B > lim / d->Hq || d->B * d->Hq > lim / d->T || d->B * d->Hkv > 65535)
    return fail(FBSA_EUNSUPPORTED, "%s: sizes exceed the grid or 32-bit row indices", fn);
  const int64_t es = d->dtype == FBSA_F32 ? 4 : 2;
  struct { const int64_t *s; int n; const char *name; } st[] = {{d->sq, 3, "q"}, {d->sk, 3, "k"}, {d->sv, 3, "v"}, {d->so, 3, "o"},
                                                                {d->skp, d->P ? 2 : 0, "k_prefix"}, {d->svp, d->P ? 2 : 0, "v_prefix"}};
  for (auto &t : st)
    for (int x = 0; x < t.n; ++x)
      if (t.s[x] < 0 || (t.s[x] * es) % 16)
        return fail(FBSA_EINVAL, "%s: %s stride[%d]=%lld must be a non-negative multiple of 16 bytes", fn, t.name, x, (long long)t.s[x]);
  // the copies address the rows of a chunk (at most 64) with unsigned 32-bit offsets from
  // its first: 63 strides of less than 64 MiB and a row fall short of 4 GiB by almost 64 MiB
  const int64_t rs[4] = {d->sk[2], d->sv[2], d->P ? d->skp[1] : 0, d->P ? d->svp[1] : 0};
  for (int64_t r : rs)
    if (r * es >= 1LL << 26) return fail(FBSA_EUNSUPPORTED, "%s: a row stride of %lld elements is 64 MiB or more", fn, (long long)r);
  // A launch has fewer than 2^32 threads along an axis: 64 a row where a wave joins
  // each; with weights 256 per 1024 keys beside a short step's rows, or 512 per 128 keys
  // (fp32; 16 bits: 256 keys) for more than 128 rows
  const CachePlan pl = cache_plan(d);
  const int64_t TG = d->T * (d->Hq / d->Hkv), most = 0xfffff000LL;
  const int64_t short_step = (d->B * d->Hq * d->T + d->B * d->Hkv * cdiv(d->S, kWeightKeys)) * 256;
  const int64_t long_step = cdiv(d->S, d->dtype == FBSA_F32 ? 128 : 256) * 512;
  if (pl.rows > lim || d->B * d->Hq * d->T > 0x3ff0000LL ||
      ((d->flags & FBSA_CACHE_WEIGHT) && (pl.scores ? short_step > most : TG > 128 && long_step > most)))
    return fail(FBSA_EUNSUPPORTED, "%s: grid too large", fn);
  return FBSA_OK;
}

}  // namespace fbsa

using namespace fbsa;

extern "C" {

size_t fbsa_cache_attn_workspace_bytes(const fbsa_cache_desc *d) { return check_cache(d) ? 0 : cache_plan(d).total; }

int fbsa_cache_attn(const fbsa_cache_desc *d, const void *q, const void *k, const void *v, const int32_t *lens,
                    const int32_t *count, const void *k_prefix, const void *v_prefix, const void *out_gate, void *o, float *lse,
                    const float *weight, float *out_weight, void *workspace, size_t workspace_bytes, void *stream) {
  int e = check_cache(d);
  if (e) return e;
  if (!q || !k || !v || !lens || !o || (d->P && (!k_prefix || !v_prefix)))
    return fail(FBSA_EINVAL, "fbsa_cache_attn: null tensor pointer");
  if (weight && !out_weight) return fail(FBSA_EINVAL, "fbsa_cache_attn: weight without out_weight");
  if (!out_weight != !(d->flags & FBSA_CACHE_WEIGHT))
    return fail(FBSA_EINVAL, "fbsa_cache_attn: out_weight and FBSA_CACHE_WEIGHT go together");
  const int64_t es = d->dtype == FBSA_F32 ? 4 : 2;
  if (!aligned_to(q, 16) || !aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(o, 16) ||
      (d->P && (!aligned_to(k_prefix, 16) || !aligned_to(v_prefix, 16))))
    return fail(FBSA_EINVAL, "fbsa_cache_attn: tensors must be 16-byte aligned");
  if (!aligned_to(lens, 4) || !aligned_to(count, 4) || !aligned_to(lse, 4) || !aligned_to(weight, 4) || !aligned_to(out_weight, 4) ||
      !aligned_to(out_gate, es))
    return fail(FBSA_EINVAL, "fbsa_cache_attn: lens/count/lse/weight/out_gate misaligned");
  const CachePlan pl = cache_plan(d);
  if (!workspace || workspace_bytes < pl.total)
    return fail(FBSA_EWORKSPACE, "fbsa_cache_attn: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, pl.total);
  if (!aligned_to(workspace, 256)) return fail(FBSA_EINVAL, "fbsa_cache_attn: workspace must be 256-byte aligned");
  CacheArgs a = {};
  a.q = q; a.k = k; a.v = v; a.kp = k_prefix; a.vp = v_prefix; a.og = out_gate; a.o = o; a.lse = lse; a.w = weight; a.wo = out_weight;
  a.lens = lens; a.count = count;
  for (int x = 0; x < 3; ++x) {
    a.sq[x] = d->sq[x]; a.sk[x] = d->sk[x]; a.sv[x] = d->sv[x]; a.so[x] = d->so[x]; a.sog[x] = d->sog[x];
    if (x < 2) { a.skp[x] = d->skp[x]; a.svp[x] = d->svp[x]; a.sw[x] = d->sw[x]; a.swo[x] = d->swo[x]; }
  }
  a.B = (int)d->B; a.Hq = (int)d->Hq; a.Hkv = (int)d->Hkv; a.T = (int)d->T; a.S = (int)d->S; a.P = (int)d->P; a.D = (int)d->D;
  a.G = (int)(d->Hq / d->Hkv); a.TG = a.T * a.G;
  a.tr_own = (int)pl.tr_own; a.tr_pre = (int)pl.tr_pre;
  a.rt_own = (int)pl.rt_own; a.rt_pre = (int)pl.rt_pre; a.np_own = (int)pl.np_own; a.np_pre = (int)pl.np_pre;
  a.few_own = pl.few_own; a.few_pre = pl.few_pre; a.direct = pl.direct;
  a.scale2 = d->scale == 0.f ? 1.f : fabsf(d->scale) * kLog2e;
  a.qand = d->scale == 0.f ? 0u : 0xffffffffu;
  a.qxor = d->scale < 0.f ? (d->dtype == FBSA_F32 ? 0x80000000u : 0x80008000u) : 0u;
  char *ws = (char *)workspace;
  a.stat = (float2 *)(ws + pl.stat); a.part = (float *)(ws + pl.part);
  if (out_weight && pl.scores) a.sc = (float *)(ws + pl.sc);
  else if (out_weight) { a.lse2 = (float *)(ws + pl.lse2); a.wpart = (float *)(ws + pl.wpart); }
  switch (d->dtype) {
    case FBSA_BF16: return dispatch_cache<bf16>(a, pl, (hipStream_t)stream);
    case FBSA_F16: return dispatch_cache<f16>(a, pl, (hipStream_t)stream);
    default: return dispatch_cache<float>(a, pl, (hipStream_t)stream);
  }
}

}  // extern "C"
