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
// the prefix those of every sequence) are stacked, 16 rows to an MFMA tile,
// ordered (token, head) so that a tile's rows see about the same keys.
//   part     a wave per (16-row tile, share of the keys): K and V stream
//            global -> LDS through a ring of the wave's own (no barrier), online
//            softmax in the log2 domain; leaves unnormalised fp32 O, row
//            maximum and row sum
//   combine  a row's parts joined in a fixed order; O, lse
//   weight   a wave per 32 keys over all rows, p recomputed from the final lse
// Lengths are read on the device; nothing depends on launch order.
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
  float scale2;              // scale * log2(e)
  float *part;               // [tile, share][row] unnormalised O (DP floats): prefix tiles, then own
  float2 *stat;              // [tile, share][row] row maximum (log2 domain), row sum
  float *lse2;               // [B][Hkv][TG] log2-domain lse, -inf for rows that see nothing
  float *sc;                 // [B][Hkv][TG][S rounded up to 32] log2-domain scores (few_own, with weights)
};

// keys per chunk: 32, 16 for fp32 at d >= 128 (registers)
template <typename T, int DP> struct CacheCfg {
  static constexpr int ES = sizeof(T);
  static constexpr int KC = ES == 4 && DP >= 128 ? 16 : 32;
  static constexpr int CPR = DP * ES / 16;
  static constexpr int TILE = KC * DP * ES;
  static constexpr int LPT = KC * CPR / 64;  // 16-byte loads per lane and tile
  static constexpr int NST = 2;
  static_assert(LPT * 64 == KC * CPR, "tile must be whole wave-loads");
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

template <typename T, int DP>
__device__ __forceinline__ void load_frag(RowFrag<T, DP> &fr, const T *row, int g, int D) {
  // (elements past the head dim are zeros: the tile's columns there hold copies of the row's last chunk)
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int ks = 0; ks < DP / 4; ++ks) fr.f[ks] = 4 * ks + g < D ? ((const float *)row)[4 * ks + g] : 0.f;
  } else {
#pragma unroll
    for (int ks = 0; ks < DP / 32; ++ks)
      fr.h[ks] = 32 * ks + 8 * g < D ? *(const s16x8 *)(row + 32 * ks + 8 * g) : s16x8{0, 0, 0, 0, 0, 0, 0, 0};
  }
}

// Per-lane byte offsets of a wave's copy of a KC-row tile (swizzled chunks);
// columns past the head dim read the row's last chunk.
template <typename T, int DP> struct TilePlan {
  using C = CacheCfg<T, DP>;
  uint32_t off[C::LPT];
  __device__ __forceinline__ void init(int64_t stride, int D, int lane) {
    const int last = D * C::ES / 16 - 1;
#pragma unroll
    for (int n = 0; n < C::LPT; ++n) {
      const int u = n * 64 + lane, row = u / C::CPR, c = (u % C::CPR) ^ swz(row, C::CPR);
      off[n] = (uint32_t)(((int64_t)row * stride) * C::ES + (c < last ? c : last) * 16);
    }
  }
  // rows [row0, ...) of a tensor of `rows` rows: rows past the end read its last one
  __device__ __forceinline__ void issue(unsigned st, const char *base, uint32_t row0, uint32_t rows, int64_t step, int rowbytes) const {
    const char *src = base + (int64_t)row0 * step;
    const uint32_t lim = tail_limit<C::KC>(row0, rows, (uint32_t)step, (uint32_t)rowbytes);
#pragma unroll
    for (int n = 0; n < C::LPT; ++n) g2lds16_s(src, off[n] > lim ? lim : off[n], st + n * 1024);
  }
};

// o[d .. d + 3] = acc * inv [* sigmoid(gate)] of a row
template <typename T> __device__ __forceinline__ void store_row(const CacheArgs &a, const RowInfo &ri, f32x4 acc, float inv, int d) {
  if (d >= a.D) return;
  T *orow = (T *)a.o + ri.b * a.so[0] + ri.hq * a.so[1] + ri.t * a.so[2] + d;
  float y[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = acc[r] * inv;
  if (a.og) {
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
__device__ __forceinline__ int64_t score_row(const CacheArgs &a, int b, int hk, int rho) {
  return (((int64_t)b * a.Hkv + hk) * a.TG + rho) * (((int64_t)a.S + 31) / 32 * 32);
}

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
  int split, np, keys;
  const char *kb, *vb;
  int64_t kstep, vstep;
  if (pre) {
    const int tile = id % a.rt_pre, hk = id / a.rt_pre / a.np_pre;
    split = id / a.rt_pre % a.np_pre;
    np = a.np_pre;
    const int64_t rho = (int64_t)tile * 16 + p, rows = (int64_t)a.B * a.TG;
    const int64_t x = rho < rows ? rho : 0;
    ri = row_info(a, (int)(x / a.TG), hk, (int)(x % a.TG));
    ri.valid = ri.valid && rho < rows;
    ri.lim = a.P;
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
    if (a.sc) score = a.sc + score_row(a, b, hk, ri.valid ? p : 0);
    slot = own_slot(a) + (((int64_t)b * a.Hkv + hk) * a.rt_own + tile) * np * 16 + split * 16;
    kstep = a.sk[2] * C::ES;
    vstep = a.sv[2] * C::ES;
    kb = (const char *)a.k + (b * a.sk[0] + hk * a.sk[1]) * C::ES;
    vb = (const char *)a.v + (b * a.sv[0] + hk * a.sv[1]) * C::ES;
  }
  // keys that any row sees; below `low` every row sees every key. A row that is
  // none (past the end, or past the sequence's new tokens) sees what the tile
  // sees, so that it asks for no masking, and is dropped by the combine.
  int low = ri.valid ? ri.lim : 0x7fffffff;
  keys = ri.valid ? ri.lim : 0;
#pragma unroll
  for (int x = 1; x < 16; x <<= 1) {
    low = min(low, __shfl_xor(low, x, 64));
    keys = max(keys, __shfl_xor(keys, x, 64));
  }
  keys = __builtin_amdgcn_readfirstlane(keys);
  low = __builtin_amdgcn_readfirstlane(low);
  const int lim = ri.valid ? ri.lim : keys;
  const int64_t nc = ((int64_t)keys + KC - 1) / KC;
  const int c0 = (int)(nc * split / np), c1 = (int)(nc * (split + 1) / np);

  RowFrag<T, DP> fr;
  load_frag<T, DP>(fr, (const T *)a.q + ri.b * a.sq[0] + ri.hq * a.sq[1] + ri.t * a.sq[2], g, a.D);
  TilePlan<T, DP> pk, pv;
  pk.init(kstep / C::ES, a.D, lane);
  pv.init(vstep / C::ES, a.D, lane);
  auto issue = [&](int c) {
    const unsigned st = (unsigned)(uintptr_t)smem + (c % C::NST) * 2 * C::TILE;
    pk.issue(st, kb, (uint32_t)c * KC, keys, kstep, a.D * C::ES);
    pv.issue(st + C::TILE, vb, (uint32_t)c * KC, keys, vstep, a.D * C::ES);
  };

  constexpr float TAU = 8.f;  // the running reference moves when a score passes it by 2^TAU
  float m_run = -INFINITY, l_run = 0.f;
  f32x4 oacc[DP / 16];
#pragma unroll
  for (int t = 0; t < DP / 16; ++t) oacc[t] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int c = c0; c < c0 + C::NST - 1 && c < c1; ++c) issue(c);
  wait_vmcnt<0>();  // the query rows too: the compiler then waits for nothing in the loop
  for (int c = c0; c < c1; ++c) {
    const int ahead = c1 - 1 - c;
    wait_ring<2 * C::LPT>(ahead < C::NST - 2 ? ahead : C::NST - 2);
    lds_wait_all();  // the previous chunk's reads, whose stage is written next
    if (c + C::NST - 1 < c1) issue(c + C::NST - 1);
    const char *Ks = smem + (c % C::NST) * 2 * C::TILE, *Vs = Ks + C::TILE;
    f32x4 s[NM];
    mm_rows_frag<T, DP, NM>(Ks, fr, s, g, p);
#pragma unroll
    for (int m = 0; m < NM; ++m) s[m] *= a.scale2;
    if ((c + 1) * (int64_t)KC > low) {
      const int lm = lim - c * KC - 4 * g;
#pragma unroll
      for (int m = 0; m < NM; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * m + r >= lm) s[m][r] = -INFINITY;
    }
    if (score && ri.valid) {
#pragma unroll
      for (int m = 0; m < NM; ++m) *(f32x4 *)(score + (int64_t)c * KC + 16 * m + 4 * g) = s[m];
    }
    float mx = -INFINITY;
#pragma unroll
    for (int m = 0; m < NM; ++m) mx = fmaxf(mx, fmaxf(fmaxf(s[m][0], s[m][1]), fmaxf(s[m][2], s[m][3])));
    if (__ballot(mx > m_run + TAU)) {
      float mc = fmaxf(mx, shfl_xor_f(mx, 16));
      mc = fmaxf(mc, shfl_xor_f(mc, 32));
      if (mc > m_run + TAU) {
        const float alpha = __builtin_amdgcn_exp2f(m_run - mc);
        l_run *= alpha;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) oacc[t] *= alpha;
        m_run = mc;
      }
    }
    const float ref = m_run == -INFINITY ? 0.f : m_run;
    float x[NM][4];
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[m][r] = __builtin_amdgcn_exp2f(s[m][r] - ref);
        l_run += x[m][r];
      }
    mm_tr_acc<T, DP, KC, 0, sizeof(T) == 2>(Vs, x, oacc, g, p);
  }

  float lt = l_run + shfl_xor_f(l_run, 16);
  lt += shfl_xor_f(lt, 32);
  if (g == 0) a.stat[slot + p] = float2{m_run, lt};
  if (ri.valid && lt != 0.f) {  // (a NaN sum is kept)
    float *dst = a.part + (slot + p) * DP;
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) *(f32x4 *)(dst + 16 * t + 4 * g) = oacc[t];
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
  const int64_t rp = (int64_t)b * a.TG + rho;
  r.npre = a.np_pre;
  r.n = a.np_pre + a.np_own;
  r.pre0 = a.np_pre ? ((int64_t)hk * a.rt_pre + rp / a.tr_pre) * a.np_pre * a.tr_pre + rp % a.tr_pre : 0;
  r.own0 = own_slot(a) + (((int64_t)b * a.Hkv + hk) * a.rt_own + rho / a.tr_own) * a.np_own * a.tr_own + rho % a.tr_own;
  return r;
}

constexpr int kMaxShares = 512;    // np_own + np_pre
constexpr int kWeightKeys = 1024;  // keys of a weight workgroup

// Workgroups [0, rows): a row each. Groups of DP / 4 threads take every NG-th
// part, a float4 a thread, and are added in order at the end.
// Workgroups past them (a.sc): kWeightKeys keys of a (sequence, KV head): each row's
// lse from its parts' statistics, then weight + sum over rows of exp2(score - lse).
template <typename T, int DP> __global__ __launch_bounds__(256) void cache_combine_kernel(CacheArgs a) {
  constexpr int LG = DP / 4, NG = 256 / LG;
  __shared__ float s_f[kMaxShares];
  __shared__ f32x4 s_acc[256];
  __shared__ float s_red[8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t rows = (int64_t)a.B * a.Hkv * a.TG;
  if (blockIdx.x >= rows) {
    const int per = (a.S + kWeightKeys - 1) / kWeightKeys;
    const int64_t u = blockIdx.x - rows;
    const int key0 = (int)(u % per) * kWeightKeys, hk = (int)(u / per % a.Hkv), b = (int)(u / per / a.Hkv);
    const int n = seq_len(a, b), c = seq_count(a, b);
    if (key0 >= n) return;
    __shared__ float s_lse[16];
    const int real = min(c * a.G, a.TG);  // rows of real queries
    for (int rho = wave; rho < real; rho += 4) {
      const RowParts rp = row_parts(a, b, hk, rho);
      float m = -INFINITY, l = 0.f;
      for (int i = lane; i < rp.n; i += 64) m = fmaxf(m, a.stat[rp.at(a, i)].x);
#pragma unroll
      for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, shfl_xor_f(m, x));
      const float ref = m == -INFINITY ? 0.f : m;
      for (int i = lane; i < rp.n; i += 64) {
        const float2 st = a.stat[rp.at(a, i)];
        if (st.y != 0.f) l += __builtin_amdgcn_exp2f(st.x - ref) * st.y;
      }
#pragma unroll
      for (int x = 1; x < 64; x <<= 1) l += shfl_xor_f(l, x);
      if (lane == 0) s_lse[rho] = l == 0.f ? -INFINITY : m + __log2f(l);
    }
    __syncthreads();
    const float *sc = a.sc + score_row(a, b, hk, 0);
    const int64_t step = score_row(a, 0, 0, 1);
    // four keys a thread, four rows' scores in flight (rows of scores are whole multiples of 32)
    static_assert(kWeightKeys == 4 * 256, "four keys to a thread");
    const int key = key0 + 4 * tid;
    if (key >= n) return;
    f32x4 w = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int r0 = 0; r0 < real; r0 += 4) {
      f32x4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = *(const f32x4 *)(sc + (r0 + j < real ? r0 + j : r0) * step + key);
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
      if (key + e < n) {
        const float w0 = a.w ? a.w[b * a.sw[0] + hk * a.sw[1] + key + e] : 0.f;
        a.wo[b * a.swo[0] + hk * a.swo[1] + key + e] = w0 + w[e];
      }
    return;
  }
  const int rho = (int)(blockIdx.x % a.TG), hk = (int)(blockIdx.x / a.TG % a.Hkv), b = (int)(blockIdx.x / a.TG / a.Hkv);
  const RowInfo ri = row_info(a, b, hk, rho);
  const RowParts rp = row_parts(a, b, hk, rho);
  const int n = ri.valid ? rp.n : 0;
  float m = -INFINITY;
  for (int i = tid; i < n; i += 256) m = fmaxf(m, a.stat[rp.at(a, i)].x);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, shfl_xor_f(m, x));
  if (lane == 0) s_red[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int i = tid; i < n; i += 256) {
    const float2 st = a.stat[rp.at(a, i)];
    const float f = st.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(st.x - ref);
    if (st.y != 0.f) l += f * st.y;
    s_f[i] = st.y == 0.f ? -1.f : f;  // (a part of no keys has no O)
  }
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) l += shfl_xor_f(l, x);
  if (lane == 0) s_red[4 + wave] = l;
  __syncthreads();
  l = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
  const int gi = tid / LG, e = tid % LG;
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int i = gi; i < n; i += NG) {
    const float f = s_f[i];
    if (f != -1.f) acc += f * *(const f32x4 *)(a.part + rp.at(a, i) * DP + 4 * e);
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
    if (a.lse2) a.lse2[blockIdx.x] = l2;
  }
}

// A wave per KC keys of a (sequence, KV head) over every row that sees them.
template <typename T, int DP> __global__ __launch_bounds__(64) void cache_weight_kernel(CacheArgs a) {
  using C = CacheCfg<T, DP>;
  constexpr int KC = C::KC, NM = KC / 16;
  extern __shared__ __attribute__((aligned(16))) char tile[];
  const int lane = threadIdx.x, g = lane >> 4, p = lane & 15;
  const int hk = blockIdx.y % a.Hkv, b = blockIdx.y / a.Hkv;
  const int n = seq_len(a, b);
  const int64_t key64 = (int64_t)blockIdx.x * KC;
  if (key64 >= n) return;
  const int key0 = (int)key64;
  TilePlan<T, DP> pk;
  pk.init(a.sk[2], a.D, lane);
  pk.issue((unsigned)(uintptr_t)tile, (const char *)a.k + (b * a.sk[0] + hk * a.sk[1]) * C::ES, (uint32_t)key0, n,
           a.sk[2] * C::ES, a.D * C::ES);
  wait_vmcnt<0>();
  lds_wait_all();  // (keeps the tile's reads behind the wait)
  float acc[NM][4];
#pragma unroll
  for (int m = 0; m < NM; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[m][r] = 0.f;
  for (int rt = 0; rt < a.rt_own; ++rt) {
    const RowInfo ri = row_info(a, b, hk, rt * 16 + p);
    if (!__ballot(ri.valid && ri.lim > key0)) continue;
    const float l2 = ri.valid ? a.lse2[((int64_t)b * a.Hkv + hk) * a.TG + rt * 16 + p] : -INFINITY;
    const int lm = l2 == -INFINITY ? 0 : ri.lim - key0 - 4 * g;  // (no row sees key 0 of a lane that has none)
    RowFrag<T, DP> fr;
    load_frag<T, DP>(fr, (const T *)a.q + b * a.sq[0] + ri.hq * a.sq[1] + ri.t * a.sq[2], g, a.D);
    f32x4 s[NM];
    mm_rows_frag<T, DP, NM>(tile, fr, s, g, p);
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (16 * m + r < lm) acc[m][r] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[m][r], a.scale2, -l2));
  }
#pragma unroll
  for (int m = 0; m < NM; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) acc[m][r] += shfl_xor_f(acc[m][r], x);
      const int key = key0 + 16 * m + 4 * g + r;
      if (p == 0 && key < n) {
        const float w0 = a.w ? a.w[b * a.sw[0] + hk * a.sw[1] + key] : 0.f;
        a.wo[b * a.swo[0] + hk * a.swo[1] + key] = w0 + acc[m][r];
      }
    }
}

static int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
static size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Tiles and shares of a call, from its sizes alone (lengths are on the device:
// the capacity stands for them).
struct CachePlan {
  int64_t tr_own, tr_pre, rt_own, rt_pre, np_own, np_pre, rows, DP;
  bool few_own, few_pre, direct;
  size_t stat, part, lse2, sc, total;
};
static CachePlan cache_plan(const fbsa_cache_desc *d) {
  CachePlan p;
  const int64_t G = d->Hq / d->Hkv, TG = d->T * G;
  p.DP = d->D <= 32 ? 32 : d->D <= 64 ? 64 : d->D <= 128 ? 128 : 256;
  const int64_t KC = d->dtype == FBSA_F32 && p.DP >= 128 ? 16 : 32;
  constexpr int64_t kWaves = 1024;  // four waves to a CU
  p.few_own = p.few_pre = true;
  p.direct = false;
  p.tr_own = p.tr_pre = 16;
  p.rt_own = cdiv(TG, p.tr_own);
  p.rt_pre = d->P ? cdiv(d->B * TG, p.tr_pre) : 0;
  auto shares = [&](int64_t tiles, int64_t keys) {
    const int64_t want = cdiv(kWaves, tiles), most = cdiv(keys, 4 * KC);
    const int64_t n = want < most ? want : most;
    return n < kMaxShares / 2 ? n : kMaxShares / 2;
  };
  p.np_own = shares(d->B * d->Hkv * p.rt_own, d->S);
  p.np_pre = d->P ? shares(d->Hkv * p.rt_pre, d->P) : 0;
  p.rows = d->B * d->Hkv * p.rt_own * p.np_own * p.tr_own + d->Hkv * p.rt_pre * p.np_pre * p.tr_pre;
  p.stat = 0;
  p.part = up256((size_t)p.rows * 8);
  p.lse2 = p.part + up256((size_t)p.rows * p.DP * 4);
  p.sc = p.lse2 + up256((size_t)(d->B * d->Hkv * TG) * 4);
  p.total = p.sc + (d->flags & FBSA_CACHE_WEIGHT && p.rt_own == 1 ? up256((size_t)(d->B * d->Hkv * TG) * cdiv(d->S, 32) * 128) : 0);
  return p;
}

template <typename T, int DP> static int launch_cache(const CacheArgs &a, hipStream_t s) {
  using C = CacheCfg<T, DP>;
  const size_t lds = (size_t)C::NST * 2 * C::TILE;
  int e = lds_optin((const void *)cache_part_kernel<T, DP>, lds, "hipFuncSetAttribute(cache_part)");
  if (e) return e;
  const int64_t rows = (int64_t)a.B * a.Hkv * a.TG;
  const int64_t parts = (int64_t)a.B * a.Hkv * a.rt_own * a.np_own + (int64_t)a.Hkv * a.rt_pre * a.np_pre;
  hipLaunchKernelGGL((cache_part_kernel<T, DP>), dim3((unsigned)parts), dim3(64), lds, s, a);
  if ((e = hip_check(hipGetLastError(), "cache_part_kernel launch"))) return e;
  const int64_t wgs = a.sc ? (int64_t)a.B * a.Hkv * cdiv(a.S, kWeightKeys) : 0;
  hipLaunchKernelGGL((cache_combine_kernel<T, DP>), dim3((unsigned)(rows + wgs)), dim3(256), 0, s, a);
  if ((e = hip_check(hipGetLastError(), "cache_combine_kernel launch"))) return e;
  if (a.wo && !a.sc) {
    hipLaunchKernelGGL((cache_weight_kernel<T, DP>), dim3((unsigned)cdiv(a.S, C::KC), (unsigned)(a.B * a.Hkv)), dim3(64), C::TILE, s, a);
    e = hip_check(hipGetLastError(), "cache_weight_kernel launch");
  }
  return e;
}

template <typename T> static int dispatch_cache(const CacheArgs &a, int64_t DP, hipStream_t s) {
  switch (DP) {
    case 32: return launch_cache<T, 32>(a, s);
    case 64: return launch_cache<T, 64>(a, s);
    case 128: return launch_cache<T, 128>(a, s);
    default: return launch_cache<T, 256>(a, s);
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
  if (!isfinite(d->scale)) return fail(FBSA_EINVAL, "%s: scale is not finite", fn);
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
  // the copies address the rows of a chunk (at most 32) with 32-bit offsets from its first
  const int64_t rs[4] = {d->sk[2], d->sv[2], d->P ? d->skp[1] : 0, d->P ? d->svp[1] : 0};
  for (int64_t r : rs)
    if (r * es >= 1LL << 26) return fail(FBSA_EUNSUPPORTED, "%s: a row stride of %lld elements is 64 MiB or more", fn, (long long)r);
  const CachePlan pl = cache_plan(d);
  if (pl.rows > lim || d->B * d->Hkv * (d->T * (d->Hq / d->Hkv) + cdiv(d->S, kWeightKeys)) > lim) return fail(FBSA_EUNSUPPORTED, "%s: grid too large", fn);
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
  a.scale2 = d->scale * kLog2e;
  char *ws = (char *)workspace;
  a.stat = (float2 *)(ws + pl.stat); a.part = (float *)(ws + pl.part);
  if (out_weight && pl.rt_own == 1) a.sc = (float *)(ws + pl.sc);
  else if (out_weight) a.lse2 = (float *)(ws + pl.lse2);
  switch (d->dtype) {
    case FBSA_BF16: return dispatch_cache<bf16>(a, pl.DP, (hipStream_t)stream);
    case FBSA_F16: return dispatch_cache<f16>(a, pl.DP, (hipStream_t)stream);
    default: return dispatch_cache<float>(a, pl.DP, (hipStream_t)stream);
  }
}

}  // extern "C"
