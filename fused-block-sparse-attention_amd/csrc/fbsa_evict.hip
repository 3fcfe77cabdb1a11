// What changes a cache of keys and values on gfx950: new rows written behind
// each sequence, and rows thrown away by the attention weight they gathered.
//
// Eviction keeps, of a (sequence, head) with n > budget rows, the first `sink`,
// the last `recent` and of those between the greatest weights that fill the
// budget. Weights become unsigned keys of the same order, and the rows that are
// kept anyway the greatest key of all, so that the kept rows are those above the
// budget-th greatest key and, of those that equal it, the first (ties go to the
// lower row). That key is found by a radix select in three digits; one ordered
// pass over the rows then writes the kept rows' numbers and weights. Another
// kernel moves the rows.
#include "fbsa_common.h"
#include "fbsa_internal.h"

namespace fbsa {

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct AppendArgs {
  char *k, *v;
  const char *kn, *vn;
  float *w;
  const int32_t *start, *count;
  int64_t sk[3], sv[3], skn[3], svn[3], sw[2];  // bytes (weight: elements)
  int32_t B, H, T, S, cpr;                      // cpr: 16-byte chunks per row
};

// A 16-byte chunk of a new key row and of its value row per thread: a copy, 5.9 us
// for 4 padded chunks of 2048 tokens, 8 heads, d 64 (27 MB), 3 us, a launch, for a step.
__global__ __launch_bounds__(256) void cache_append_kernel(AppendArgs a) {
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int c = (int)(u % a.cpr);
  const int64_t r = u / a.cpr;
  const int t = (int)(r % a.T), h = (int)(r / a.T % a.H);
  const int64_t b = r / a.T / a.H;
  if (b >= a.B || (a.count && t >= a.count[b])) return;
  const int64_t s = (int64_t)a.start[b] + t;
  if (s < 0 || s >= a.S) return;
  const i32x4 x = *(const i32x4 *)(a.kn + b * a.skn[0] + h * a.skn[1] + t * a.skn[2] + c * 16);
  const i32x4 y = *(const i32x4 *)(a.vn + b * a.svn[0] + h * a.svn[1] + t * a.svn[2] + c * 16);
  *(i32x4 *)(a.k + b * a.sk[0] + h * a.sk[1] + s * a.sk[2] + c * 16) = x;
  *(i32x4 *)(a.v + b * a.sv[0] + h * a.sv[1] + s * a.sv[2] + c * 16) = y;
  if (a.w && c == 0) a.w[b * a.sw[0] + h * a.sw[1] + s] = 0.f;
}

struct EvictArgs {
  const char *k, *v;
  char *ko, *vo;
  const float *w;
  float *wo;
  const int32_t *lens;
  int32_t *index, *new_lens;
  int64_t sk[3], sv[3], sko[3], svo[3], sw[2], swo[2];  // bytes (weights: elements)
  int32_t B, H, S, budget, recent, sink, ni, cpr;       // ni: entries of an index row
};

__device__ __forceinline__ int evict_len(const EvictArgs &a, int b) {
  const int n = a.lens[b];
  return n < 0 ? 0 : n > a.S ? a.S : n;
}

// Row i's key: the weight's bits in unsigned order (NaN as -inf, -0 as 0), which
// lie in [0x007fffff, 0xff800000]; the rows that are kept whatever they weigh have
// the greatest key of all, places past the length the least.
__device__ __forceinline__ uint32_t row_key(const EvictArgs &a, float w, int64_t i, int n) {
  if (!(w == w)) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f), k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return i >= n ? 0u : i < a.sink || i >= n - a.recent ? 0xffffffffu : k;
}

// The budget-th greatest key is found digit by digit: 11, 11 and 10 bits.
constexpr int kBins = 2048;
__device__ __forceinline__ constexpr int digit_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__device__ __forceinline__ constexpr int digit_bits(int pass) { return pass == 2 ? 10 : 11; }

// The bin of the need-th greatest key, and how many of that bin are needed, from
// a histogram in LDS; NT threads, each NB = kBins / NT bins in descending order.
struct Pick {
  uint32_t bin, need;
};
template <int NT> __device__ __forceinline__ Pick pick_bin(const uint32_t *hist, uint32_t need, uint32_t *s_wave, Pick *s_pick) {
  constexpr int NB = kBins / NT, NW = NT / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t c[NB], sum = 0;
#pragma unroll
  for (int j = 0; j < NB; ++j) sum += c[j] = hist[kBins - 1 - NB * tid - j];
  uint32_t before = sum;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    const uint32_t y = __shfl_up(before, x, 64);
    if (lane >= x) before += y;
  }
  if (lane == 63) s_wave[wave] = before;
  before -= sum;
  __syncthreads();
  for (int v = 0; v < NW; ++v)
    if (v < wave) before += s_wave[v];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    if (before < need && need <= before + c[j]) *s_pick = Pick{(uint32_t)(kBins - 1 - NB * tid - j), need - before};
    before += c[j];
  }
  __syncthreads();
  return *s_pick;
}

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;

// Whether the wave's 64 keys are one, which then counts in one addition: 64 to the
// same counter of LDS take turns (a call over 16 heads of 16384
// equal weights: 57 us, 20 so).
__device__ __forceinline__ bool wave_equal(uint32_t key) {
  return !__ballot(key != (uint32_t)__builtin_amdgcn_readfirstlane((int)key));
}

// Counts (of rows above the key, and << 16 of rows that equal it) to the sums
// before them, in row order; the first wave.
template <int N> __device__ __forceinline__ int counts_before(int *cnt, int lane) {
  constexpr int PL = (N + 63) / 64;
  int c[PL], sum = 0;
#pragma unroll
  for (int j = 0; j < PL; ++j) {
    const int u = lane * PL + j;
    c[j] = u < N ? cnt[u] : 0;
    sum += c[j];
  }
  int before = sum;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    const int y = __shfl_up(before, x, 64);
    if (lane >= x) before += y;
  }
  const int all = __shfl(before, 63, 64);
  before -= sum;
#pragma unroll
  for (int j = 0; j < PL; ++j) {
    const int u = lane * PL + j;
    if (u < N) cnt[u] = before;
    before += c[j];
  }
  return all;
}

// A workgroup per (sequence, head) whose weights stay in registers, R a thread:
// rows tid + 1024 r. One workgroup to a CU, so instructions per row are what it
// costs: keys are formed once (16 rows of up to 16301 weights: 18.2 us with the keys
// and bounds formed in every pass, 14.6 here; four copies of the first digit's
// counters, against lanes that count in one place, changed nothing).
template <int R> __global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.x % a.H, b = blockIdx.x / a.H;
  const int n = evict_len(a, b);
  const float *w = a.w + b * a.sw[0] + h * a.sw[1];
  float *wo = a.wo + b * a.swo[0] + h * a.swo[1];
  int32_t *index = a.index + (int64_t)blockIdx.x * a.ni;
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t s_wave[kSelWaves];
  __shared__ Pick s_pick;
  __shared__ int s_cnt[R][kSelWaves];
  float x[R];
  uint32_t key[R];
#pragma unroll
  for (int r = 0; r < R; ++r) x[r] = tid + r * kSelThreads < n ? w[tid + r * kSelThreads] : 0.f;
  const int kept = n < a.budget ? n : a.budget;
  if (h == 0 && tid == 0) a.new_lens[b] = kept;
  for (int i = kept + tid; i < a.ni; i += kSelThreads) index[i] = -1;
#pragma unroll
  for (int r = 0; r < R; ++r) key[r] = row_key(a, x[r], tid + r * kSelThreads, n);
  uint32_t same = 0;  // bit r: the wave's keys r are equal
#pragma unroll
  for (int r = 0; r < R; ++r) same |= (uint32_t)wave_equal(key[r]) << r;
  uint32_t need = 0, prefix = 0;  // (a length within the budget: every row is above key 0)
  if (n > a.budget) {
    need = (uint32_t)a.budget;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = digit_shift(pass), bits = digit_bits(pass);
      for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool all = same >> r & 1;
        if ((!all || lane == 0) && (pass == 0 ? r * kSelThreads < n : key[r] >> (shift + bits) == prefix))
          atomicAdd(&hist[key[r] >> shift & ((1u << bits) - 1)], all ? 64u : 1u);
      }
      __syncthreads();
      const Pick pk = pick_bin<kSelThreads>(hist, need, s_wave, &s_pick);
      prefix = prefix << bits | pk.bin;
      need = pk.need;
      __syncthreads();
    }
  }
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int d = __popcll(__ballot(key[r] > prefix)), e = __popcll(__ballot(key[r] == prefix));
    if (lane == 0) s_cnt[r][wave] = d | e << 16;
  }
  wait_vmcnt<0>();  // (in place: this wave's weights are here before any wave writes one)
  __syncthreads();
  if (wave == 0) counts_before<R * kSelWaves>(&s_cnt[0][0], lane);
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t c = (uint32_t)s_cnt[r][wave];
    const bool def = key[r] > prefix, eq = key[r] == prefix;
    const uint32_t d0 = (c & 0xffff) + __popcll(__ballot(def) & below), e0 = (c >> 16) + __popcll(__ballot(eq) & below);
    if (def || (eq && e0 < need)) {
      const uint32_t at = d0 + (e0 < need ? e0 : need);
      index[at] = tid + r * kSelThreads;
      wo[at] = x[r];
    }
  }
}

// Longer rows: chunks of kChunk weights, a workgroup each, in four steps over a
// workspace (262144 rows of 8 heads: 29 us in five launches, each a few microseconds of
// latency, against 470 with a workgroup per row). hist: the first digit's histogram of the row. cand: the chunk's keys
// that share the wanted key's first digit, in order, and how many lie above.
// rank (a workgroup per row): the other two digits among those, and each chunk's
// place in the output. place: kept rows' numbers and weights.
constexpr int kChunkR = 8, kChunk = kSelThreads * kChunkR;
struct EvictWs {
  uint32_t *hist;   // [row][kBins]
  uint32_t *cand;   // [row][chunk][kChunk]
  float *copy;      // [row][chunk][kChunk]: the weights, where they are moved in place
  uint2 *count;     // [row][chunk]: keys above the first digit, keys of it
  uint2 *start;     // [row][chunk]: keys above the wanted one before the chunk, equal to it before it
  uint2 *pick;      // [row]: the first digit and how many of it are kept; then the same of the whole key
  int nch;
};

__global__ __launch_bounds__(256) void evict_zero_kernel(uint32_t *x, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) x[i] = 0;
}

// a chunk's weights and keys
__device__ __forceinline__ void chunk_keys(const EvictArgs &a, const float *w, int64_t base, int n, float (&x)[kChunkR], uint32_t (&key)[kChunkR]) {
#pragma unroll
  for (int r = 0; r < kChunkR; ++r) {
    const int64_t i = base + threadIdx.x + r * kSelThreads;
    x[r] = i < n ? w[i] : 0.f;
  }
#pragma unroll
  for (int r = 0; r < kChunkR; ++r) key[r] = row_key(a, x[r], base + threadIdx.x + r * kSelThreads, n);
}

__global__ __launch_bounds__(kSelThreads) void evict_hist_kernel(EvictArgs a, EvictWs ws) {
  const int h = blockIdx.y % a.H, b = blockIdx.y / a.H, n = evict_len(a, b), kept = n < a.budget ? n : a.budget;
  const int64_t base = (int64_t)blockIdx.x * kChunk;
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) a.new_lens[b] = kept;
  for (int r = 0; r < kChunkR; ++r) {
    const int64_t i = base + threadIdx.x + r * kSelThreads;
    if (i >= kept && i < a.ni) a.index[(int64_t)blockIdx.y * a.ni + i] = -1;
  }
  if (base >= n) return;
  __shared__ uint32_t hist[kBins];
  for (int i = threadIdx.x; i < kBins; i += kSelThreads) hist[i] = 0;
  float x[kChunkR];
  uint32_t key[kChunkR];
  chunk_keys(a, a.w + b * a.sw[0] + h * a.sw[1], base, n, x, key);
  if (ws.copy) {
    float *to = ws.copy + (int64_t)blockIdx.y * ws.nch * kChunk + base;
#pragma unroll
    for (int r = 0; r < kChunkR; ++r) to[threadIdx.x + r * kSelThreads] = x[r];
  }
  if (n <= a.budget) return;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kChunkR; ++r) {
    const bool all = wave_equal(key[r]);
    if (!all || (threadIdx.x & 63) == 0) atomicAdd(&hist[key[r] >> digit_shift(0)], all ? 64u : 1u);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kSelThreads)
    if (hist[i]) atomicAdd(&ws.hist[(int64_t)blockIdx.y * kBins + i], hist[i]);  // (whole numbers: any order gives the same)
}

__global__ __launch_bounds__(kSelThreads) void evict_cand_kernel(EvictArgs a, EvictWs ws) {
  const int h = blockIdx.y % a.H, b = blockIdx.y / a.H, n = evict_len(a, b);
  const int64_t base = (int64_t)blockIdx.x * kChunk;
  if (n <= a.budget || base >= n) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ uint32_t hist[kBins], s_wave[kSelWaves];
  __shared__ Pick s_pick;
  __shared__ int s_cnt[kChunkR][kSelWaves];
  float x[kChunkR];
  uint32_t key[kChunkR];
  chunk_keys(a, a.w + b * a.sw[0] + h * a.sw[1], base, n, x, key);
  for (int i = tid; i < kBins; i += kSelThreads) hist[i] = ws.hist[(int64_t)blockIdx.y * kBins + i];
  __syncthreads();
  const Pick pk = pick_bin<kSelThreads>(hist, (uint32_t)a.budget, s_wave, &s_pick);
#pragma unroll
  for (int r = 0; r < kChunkR; ++r) {
    const uint32_t top = key[r] >> digit_shift(0);
    const int c = __popcll(__ballot(top == pk.bin)), above = __popcll(__ballot(top > pk.bin));
    if (lane == 0) s_cnt[r][wave] = c | above << 16;
  }
  __syncthreads();
  if (wave == 0) {
    const int all = counts_before<kChunkR * kSelWaves>(&s_cnt[0][0], lane);
    if (lane == 0) ws.count[(int64_t)blockIdx.y * ws.nch + blockIdx.x] = uint2{(uint32_t)all >> 16, (uint32_t)all & 0xffff};
    if (lane == 0 && blockIdx.x == 0) ws.pick[blockIdx.y] = uint2{pk.bin, pk.need};
  }
  __syncthreads();
  uint32_t *dst = ws.cand + ((int64_t)blockIdx.y * ws.nch + blockIdx.x) * kChunk;
#pragma unroll
  for (int r = 0; r < kChunkR; ++r) {
    const bool in = key[r] >> digit_shift(0) == pk.bin;
    const int at = (s_cnt[r][wave] & 0xffff) + __popcll(__ballot(in) & ((1ull << lane) - 1));
    if (in) dst[at] = key[r];
  }
}

__global__ __launch_bounds__(kSelThreads) void evict_rank_kernel(EvictArgs a, EvictWs ws) {
  const int n = evict_len(a, blockIdx.x / a.H);
  if (n <= a.budget) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nch = (int)(((int64_t)n + kChunk - 1) / kChunk);
  const uint2 *count = ws.count + (int64_t)blockIdx.x * ws.nch;
  uint2 *start = ws.start + (int64_t)blockIdx.x * ws.nch;
  const uint32_t *cand = ws.cand + (int64_t)blockIdx.x * ws.nch * kChunk;
  __shared__ uint32_t hist[kBins], s_wave[kSelWaves], s_above[64], s_equal[64];
  __shared__ Pick s_pick;
  uint32_t prefix = ws.pick[blockIdx.x].x, need = ws.pick[blockIdx.x].y;
  // 64 chunks at a time, whose counts the lanes hold: a wave takes slices of 512
  // candidates, eight loads under way, and a chunk's slices go to different waves:
  // rows kept before lie in the first chunks, all candidates again. A call over 262144
  // rows of 8 heads, d 64, in place, against a wave per chunk and 64 keys at a time: 140
  // -> 85 us where the kept rows lie first, 534 -> 125 with equal weights; spread over
  // all chunks the kernel takes 9.4 us against 8.3
  constexpr int R = 8, SL = kChunk / (64 * R);
  static_assert(SL <= kSelWaves && kSelWaves % SL == 0, "slices of a chunk");
  auto slices = [&](int c0, uint32_t cnt, auto f) {
    for (int j = 0; j < SL && __ballot((int)cnt > j * 64 * R); ++j)
      for (int q = 0; q < 64; q += kSelWaves) {
        const int at = q + (wave + j * (kSelWaves / SL)) % kSelWaves, m = __builtin_amdgcn_readlane((int)cnt, at);
        if (j * 64 * R >= m) continue;
        uint32_t key[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int i = (j * R + r) * 64 + lane;
          key[r] = i < m ? cand[(int64_t)(c0 + at) * kChunk + i] : 0;  // (no candidate's key is 0)
        }
        f(at, key, m - j * 64 * R);
      }
  };
#pragma unroll
  for (int pass = 1; pass < 3; ++pass) {
    const int shift = digit_shift(pass), bits = digit_bits(pass);
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int c0 = 0; c0 < nch; c0 += 64)
      slices(c0, c0 + lane < nch ? count[c0 + lane].y : 0, [&](int, const uint32_t (&key)[R], int m) {
        const uint32_t first = (uint32_t)__builtin_amdgcn_readfirstlane((int)key[0]);
        auto in = [&](uint32_t x) { return x && x >> (shift + bits) == prefix; };
        auto bin = [&](uint32_t x) { return x >> shift & ((1u << bits) - 1); };
        bool one = true;
#pragma unroll
        for (int r = 0; r < R && 64 * r < m; ++r) one = one && (key[r] == first || !key[r]);
        if (!__ballot(!one)) {  // (equal weights: one addition)
          if (lane == 0 && in(first)) atomicAdd(&hist[bin(first)], (uint32_t)(m < 64 * R ? m : 64 * R));
          return;
        }
#pragma unroll
        for (int r = 0; r < R && 64 * r < m; ++r)
          if (in(key[r])) atomicAdd(&hist[bin(key[r])], 1u);
      });
    __syncthreads();
    const Pick pk = pick_bin<kSelThreads>(hist, need, s_wave, &s_pick);
    prefix = prefix << bits | pk.bin;
    need = pk.need;
    __syncthreads();
  }
  // each chunk's keys above the wanted one and equal to it, and their sums before it
  uint32_t d0 = 0, e0 = 0;
  for (int c0 = 0; c0 < nch; c0 += 64) {
    if (tid < 64) s_above[tid] = s_equal[tid] = 0;
    __syncthreads();
    const uint2 x = c0 + lane < nch ? count[c0 + lane] : uint2{0, 0};
    slices(c0, x.y, [&](int at, const uint32_t (&key)[R], int m) {
      uint32_t d = 0, e = 0;
#pragma unroll
      for (int r = 0; r < R && 64 * r < m; ++r) {
        d += __popcll(__ballot(key[r] > prefix));
        e += __popcll(__ballot(key[r] == prefix));
      }
      if (lane == 0) {
        atomicAdd(&s_above[at], d);
        atomicAdd(&s_equal[at], e);
      }
    });
    __syncthreads();
    if (wave == 0) {
      const uint32_t dx = x.x + s_above[lane], ex = s_equal[lane];
      uint32_t d = dx, e = ex;
#pragma unroll
      for (int y = 1; y < 64; y <<= 1) {
        const uint32_t dd = __shfl_up(d, y, 64), ee = __shfl_up(e, y, 64);
        if (lane >= y) { d += dd; e += ee; }
      }
      if (c0 + lane < nch) start[c0 + lane] = uint2{d0 + d - dx, e0 + e - ex};
      d0 += __shfl(d, 63, 64);
      e0 += __shfl(e, 63, 64);
    }
    __syncthreads();
  }
  if (tid == 0) ws.pick[blockIdx.x] = uint2{prefix, need};
}

__global__ __launch_bounds__(kSelThreads) void evict_place_kernel(EvictArgs a, EvictWs ws) {
  const int h = blockIdx.y % a.H, b = blockIdx.y / a.H, n = evict_len(a, b);
  const int64_t base = (int64_t)blockIdx.x * kChunk;
  if (base >= n) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // (in place: another chunk's rows may already lie where this one's weights were)
  const float *w = ws.copy ? ws.copy + (int64_t)blockIdx.y * ws.nch * kChunk : a.w + b * a.sw[0] + h * a.sw[1];
  float *wo = a.wo + b * a.swo[0] + h * a.swo[1];
  int32_t *index = a.index + (int64_t)blockIdx.y * a.ni;
  float x[kChunkR];
  uint32_t key[kChunkR];
  chunk_keys(a, w, base, n, x, key);
  __shared__ int s_cnt[kChunkR][kSelWaves];
  uint2 st = uint2{(uint32_t)base, 0}, pk = uint2{0, 0};  // (a length within the budget: every row is above key 0)
  if (n > a.budget) {
    st = ws.start[(int64_t)blockIdx.y * ws.nch + blockIdx.x];
    pk = ws.pick[blockIdx.y];
  }
#pragma unroll
  for (int r = 0; r < kChunkR; ++r) {
    const int d = __popcll(__ballot(key[r] > pk.x)), e = __popcll(__ballot(key[r] == pk.x));
    if (lane == 0) s_cnt[r][wave] = d | e << 16;
  }
  __syncthreads();
  if (wave == 0) counts_before<kChunkR * kSelWaves>(&s_cnt[0][0], lane);
  __syncthreads();
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int r = 0; r < kChunkR; ++r) {
    const uint32_t c = (uint32_t)s_cnt[r][wave];
    const bool def = key[r] > pk.x, eq = key[r] == pk.x;
    const uint32_t d0 = st.x + (c & 0xffff) + __popcll(__ballot(def) & below), e0 = st.y + (c >> 16) + __popcll(__ballot(eq) & below);
    if (def || (eq && e0 < pk.y)) {
      const uint32_t at = d0 + (e0 < pk.y ? e0 : pk.y);
      index[at] = (int32_t)(base + tid + r * kSelThreads);
      wo[at] = x[r];
    }
  }
}

// Rows of up to this many weights: one workgroup, weights in registers. Longer
// ones: the steps above, whose five launches cost more than they save below it.
constexpr int64_t kOneGroup = 16 * kSelThreads;

// In place, many rows of few heads pass through the workspace, up to kStage bytes
// at a time: one more trip through memory, but at the whole card's rate, where the
// move kernel has a workgroup per (head, k or v, 64 bytes of a row) and goes through
// the rows kMove at a time. Calls, staged against moved: 16384 rows of 8 heads, d 64
// (32 workgroups) 77 and 211 us; 2048 of 8, d 128 (64) 17 and 24; 32768 of 8, d 256
// (128) 233 and 433; 4096 of 16, d 256 (256) 64 and 59; 4096 of 128, d 128 (1024) 224
// and 168; 512 of 8, d 64 (32) 10.4 and 10.1; 768 of 4 (16) 9.1 and 11.7.
constexpr int64_t kStage = 32 << 20, kStageWgs = 128;
constexpr int kMoveU = 8, kMove = 64 * kMoveU;

struct EvictPlan {
  int64_t nch, part;  // part: rows of a head that pass through the workspace at a time (0: none do)
  size_t hist, count, start, pick, cand, copy, stage, total;
};
static EvictPlan evict_plan(const fbsa_evict_desc *d) {
  EvictPlan p = {};
  const size_t rows = (size_t)(d->B * d->H);
  const int64_t cpr = d->D * (d->dtype == FBSA_F32 ? 4 : 2) / 16, ni = d->budget < d->S ? d->budget : d->S;
  size_t stage = 0;
  if (d->flags & FBSA_EVICT_IN_PLACE && d->budget < d->S && ni > kMove && 2 * (int64_t)rows * ((cpr + 3) / 4) <= kStageWgs) {
    const int64_t most = kStage / ((int64_t)rows * cpr * 32);
    p.part = ni < most ? ni : most;
    stage = (size_t)(p.part < ni ? 2 : 1) * rows * p.part * cpr * 32;
  }
  if (d->S <= kOneGroup) {
    p.total = stage;
    return p;
  }
  p.nch = (d->S + kChunk - 1) / kChunk;
  p.hist = 0;
  p.count = p.hist + rows * kBins * 4;
  p.start = p.count + rows * p.nch * 8;
  p.pick = p.start + rows * p.nch * 8;
  p.cand = (p.pick + rows * 8 + 255) / 256 * 256;
  p.copy = p.cand + rows * p.nch * kChunk * 4;
  p.stage = p.copy + (d->flags & FBSA_EVICT_IN_PLACE ? rows * p.nch * kChunk * 4 : 0);
  p.total = p.stage + stage;
  return p;
}

// Rows to other buffers: a 16-byte chunk of a key row and of its value row per
// thread; 16 caches of 4096 kept rows, d 256: 20 us, 6.4 TB/s read and written.
__global__ __launch_bounds__(256) void evict_copy_kernel(EvictArgs a) {
  const int h = blockIdx.y % a.H, b = blockIdx.y / a.H;
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int c = (int)(u % a.cpr);
  const int64_t i = u / a.cpr;
  const int n = evict_len(a, b);
  if (i >= n || i >= a.budget) return;
  const int64_t s = a.index[(int64_t)blockIdx.y * a.ni + i];
  const i32x4 x = *(const i32x4 *)(a.k + b * a.sk[0] + h * a.sk[1] + s * a.sk[2] + c * 16);
  const i32x4 y = *(const i32x4 *)(a.v + b * a.sv[0] + h * a.sv[1] + s * a.sv[2] + c * 16);
  *(i32x4 *)(a.ko + b * a.sko[0] + h * a.sko[1] + i * a.sko[2] + c * 16) = x;
  *(i32x4 *)(a.vo + b * a.svo[0] + h * a.svo[1] + i * a.svo[2] + c * 16) = y;
}

// Rows within their own buffer: a workgroup per (sequence, head, k or v, slice of
// 64 bytes of every row) walks the kept rows in order, kMove at a time. Row i
// comes from index[i] >= i, so a step writes only rows that no later step
// reads; within a step every read has ended before the first write.
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
  const int h = blockIdx.z % a.H, b = blockIdx.z / a.H;
  const int n = evict_len(a, b);
  if (n <= a.budget) return;
  const int c = blockIdx.x * 4 + (threadIdx.x & 3);
  const int64_t *st = blockIdx.y ? a.sv : a.sk;
  char *x = (blockIdx.y ? a.vo : a.ko) + b * st[0] + h * st[1] + c * 16;
  const int32_t *index = a.index + (int64_t)blockIdx.z * a.ni;
  for (int base = 0; base < a.budget; base += kMove) {
    i32x4 y[kMoveU];
    bool go[kMoveU];
#pragma unroll
    for (int j = 0; j < kMoveU; ++j) {
      const int i = base + j * 64 + (threadIdx.x >> 2);
      const int s = i < a.budget ? index[i] : i;
      go[j] = s != i && c < a.cpr;
      if (go[j]) y[j] = *(const i32x4 *)(x + s * st[2]);
    }
    wait_vmcnt<0>();
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kMoveU; ++j) {
      const int i = base + j * 64 + (threadIdx.x >> 2);
      if (go[j]) *(i32x4 *)(x + i * st[2]) = y[j];
    }
  }
}

// The same through the workspace, `part` rows of every head a launch: launch t
// takes part t in and part t - 1 out, which is written only after every row of it
// and of the parts before has been read, and below every row that part t reads.
__global__ __launch_bounds__(256) void evict_stage_kernel(EvictArgs a, char *stage, int part, int t, int nt) {
  const bool out = blockIdx.z;
  if (t - out < 0 || t - out >= nt) return;
  t -= out;
  const int h = blockIdx.y % a.H, b = blockIdx.y / a.H;
  const uint32_t u = blockIdx.x * 256 + threadIdx.x;
  const int c = (int)(u % (uint32_t)a.cpr), local = (int)(u / (uint32_t)a.cpr);
  const int64_t i = (int64_t)t * part + local;
  const int n = evict_len(a, b);
  if (n <= a.budget || local >= part || i >= a.budget) return;
  const int64_t s = a.index[(int64_t)blockIdx.y * a.ni + i];
  if (s == i) return;
  const int64_t size = (int64_t)part * a.cpr * 16;
  char *at = stage + ((int64_t)(t & 1) * gridDim.y + blockIdx.y) * 2 * size + (int64_t)u * 16;
  char *k = a.ko + b * a.sk[0] + h * a.sk[1] + (out ? i : s) * a.sk[2] + c * 16;
  char *v = a.vo + b * a.sv[0] + h * a.sv[1] + (out ? i : s) * a.sv[2] + c * 16;
  if (out) {
    const i32x4 x = *(const i32x4 *)at, y = *(const i32x4 *)(at + size);
    *(i32x4 *)k = x;
    *(i32x4 *)v = y;
  } else {
    const i32x4 x = *(const i32x4 *)k, y = *(const i32x4 *)v;
    *(i32x4 *)at = x;
    *(i32x4 *)(at + size) = y;
  }
}

static bool aligned_to(const void *p, int64_t n) { return (uintptr_t)p % (uintptr_t)n == 0; }

static int check_rows(const char *fn, int dtype, int64_t D, const int64_t (*const *st)[3], const char *const *name, int n) {
  if (dtype < FBSA_F32 || dtype > FBSA_F16) return fail(FBSA_EINVAL, "%s: bad dtype %d", fn, dtype);
  if (D < 8 || D > 256 || D % 8) return fail(FBSA_EUNSUPPORTED, "%s: head dim %lld is not a multiple of 8 up to 256", fn, (long long)D);
  const int64_t es = dtype == FBSA_F32 ? 4 : 2;
  for (int t = 0; t < n; ++t)
    for (int x = 0; x < 3; ++x)
      if ((*st[t])[x] < 0 || ((*st[t])[x] * es) % 16)
        return fail(FBSA_EINVAL, "%s: %s stride[%d]=%lld must be a non-negative multiple of 16 bytes", fn, name[t], x,
                    (long long)(*st[t])[x]);
  return FBSA_OK;
}

constexpr int64_t kMaxRows = 0x7fff0000LL, kMaxThreads = 0xfffff000LL;  // (a launch has fewer than 2^32 threads)

}  // namespace fbsa

using namespace fbsa;

extern "C" {

int fbsa_cache_append(const fbsa_append_desc *d, void *k, void *v, const void *k_new, const void *v_new, const int32_t *start,
                      const int32_t *count, float *weight, void *stream) {
  static const char *fn = "fbsa_cache_append";
  if (!d) return fail(FBSA_EINVAL, "%s: null descriptor", fn);
  const int64_t(*const st[])[3] = {&d->sk, &d->sv, &d->skn, &d->svn};
  static const char *const name[] = {"k", "v", "k_new", "v_new"};
  const int e = check_rows(fn, d->dtype, d->D, st, name, 4);
  if (e) return e;
  if (d->flags) return fail(FBSA_EINVAL, "%s: unknown flags 0x%x", fn, d->flags);
  if (d->B < 1 || d->H < 1 || d->T < 1 || d->S < 1)
    return fail(FBSA_EINVAL, "%s: sizes must be positive (B=%lld H=%lld T=%lld S=%lld)", fn, (long long)d->B, (long long)d->H,
                (long long)d->T, (long long)d->S);
  const int64_t es = d->dtype == FBSA_F32 ? 4 : 2, cpr = d->D * es / 16;
  if (d->B > kMaxRows || d->H > kMaxRows || d->T > kMaxRows || d->S > kMaxRows || d->B > kMaxRows / d->H ||
      d->B * d->H > kMaxRows / d->T || d->B * d->H * d->T * cpr > kMaxThreads)
    return fail(FBSA_EUNSUPPORTED, "%s: sizes exceed the grid or 32-bit row indices", fn);
  if (!k || !v || !k_new || !v_new || !start) return fail(FBSA_EINVAL, "%s: null tensor pointer", fn);
  if (!aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(k_new, 16) || !aligned_to(v_new, 16) || !aligned_to(start, 4) ||
      !aligned_to(count, 4) || !aligned_to(weight, 4))
    return fail(FBSA_EINVAL, "%s: misaligned pointer (rows: 16 bytes)", fn);
  AppendArgs a = {};
  a.k = (char *)k; a.v = (char *)v; a.kn = (const char *)k_new; a.vn = (const char *)v_new; a.w = weight;
  a.start = start; a.count = count;
  for (int x = 0; x < 3; ++x) {
    a.sk[x] = d->sk[x] * es; a.sv[x] = d->sv[x] * es; a.skn[x] = d->skn[x] * es; a.svn[x] = d->svn[x] * es;
    if (x < 2) a.sw[x] = d->sw[x];
  }
  a.B = (int)d->B; a.H = (int)d->H; a.T = (int)d->T; a.S = (int)d->S; a.cpr = (int)cpr;
  hipLaunchKernelGGL(cache_append_kernel, dim3((unsigned)((d->B * d->H * d->T * cpr + 255) / 256)), dim3(256), 0, (hipStream_t)stream, a);
  return hip_check(hipGetLastError(), "cache_append_kernel launch");
}

static int check_evict(const fbsa_evict_desc *d) {
  static const char *fn = "fbsa_cache_evict";
  if (!d) return fail(FBSA_EINVAL, "%s: null descriptor", fn);
  const int64_t(*const st[])[3] = {&d->sk, &d->sv, &d->sko, &d->svo};
  static const char *const name[] = {"k", "v", "k_out", "v_out"};
  const int e = check_rows(fn, d->dtype, d->D, st, name, 4);
  if (e) return e;
  if (d->flags & ~FBSA_EVICT_IN_PLACE) return fail(FBSA_EINVAL, "%s: unknown flags 0x%x", fn, d->flags);
  if (d->B < 1 || d->H < 1 || d->S < 1 || d->budget < 1)
    return fail(FBSA_EINVAL, "%s: sizes must be positive (B=%lld H=%lld S=%lld budget=%lld)", fn, (long long)d->B, (long long)d->H,
                (long long)d->S, (long long)d->budget);
  if (d->recent < 0 || d->sink < 0 || d->recent > d->budget || d->sink > d->budget - d->recent)
    return fail(FBSA_EINVAL, "%s: recent=%lld and sink=%lld must be non-negative and fit the budget of %lld", fn, (long long)d->recent,
                (long long)d->sink, (long long)d->budget);
  const int64_t ni = d->budget < d->S ? d->budget : d->S;
  if (d->SO < ni) return fail(FBSA_EINVAL, "%s: output capacity %lld is below %lld", fn, (long long)d->SO, (long long)ni);
  const int64_t cpr = d->D * (d->dtype == FBSA_F32 ? 4 : 2) / 16;
  if (d->S > kMaxRows || d->budget > kMaxRows || ni * cpr > kMaxThreads || d->B > 65535 || d->H > 65535 || d->B * d->H > 65535)
    return fail(FBSA_EUNSUPPORTED, "%s: sizes exceed the grid or 32-bit row indices", fn);
  return FBSA_OK;
}

size_t fbsa_cache_evict_workspace_bytes(const fbsa_evict_desc *d) { return check_evict(d) ? 0 : evict_plan(d).total; }

int fbsa_cache_evict(const fbsa_evict_desc *d, const void *k, const void *v, const float *weight, const int32_t *lens, void *k_out,
                     void *v_out, float *w_out, int32_t *index, int32_t *new_lens, void *workspace, size_t workspace_bytes,
                     void *stream) {
  static const char *fn = "fbsa_cache_evict";
  int e = check_evict(d);
  if (e) return e;
  const bool inplace = d->flags & FBSA_EVICT_IN_PLACE;
  const EvictPlan pl = evict_plan(d);
  const int64_t ni = d->budget < d->S ? d->budget : d->S;
  if (!k || !v || !weight || !lens || !k_out || !v_out || !w_out || !index || !new_lens)
    return fail(FBSA_EINVAL, "%s: null tensor pointer", fn);
  if (!aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(k_out, 16) || !aligned_to(v_out, 16) || !aligned_to(weight, 4) ||
      !aligned_to(lens, 4) || !aligned_to(w_out, 4) || !aligned_to(index, 4) || !aligned_to(new_lens, 4))
    return fail(FBSA_EINVAL, "%s: misaligned pointer (rows: 16 bytes)", fn);
  if (lens == new_lens) return fail(FBSA_EINVAL, "%s: new_lens is lens", fn);
  if (inplace) {
    bool same = k == k_out && v == v_out && weight == w_out && d->SO == d->S;
    for (int x = 0; x < 3; ++x) same = same && d->sk[x] == d->sko[x] && d->sv[x] == d->svo[x] && (x == 2 || d->sw[x] == d->swo[x]);
    if (!same) return fail(FBSA_EINVAL, "%s: FBSA_EVICT_IN_PLACE with outputs that are not the inputs", fn);
  } else if (k == k_out || v == v_out || weight == w_out) {
    return fail(FBSA_EINVAL, "%s: outputs overlap inputs (FBSA_EVICT_IN_PLACE evicts in place)", fn);
  }
  if (pl.total && (!workspace || workspace_bytes < pl.total))
    return fail(FBSA_EWORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, workspace ? workspace_bytes : 0, pl.total);
  if (pl.total && !aligned_to(workspace, 256)) return fail(FBSA_EINVAL, "%s: workspace must be 256-byte aligned", fn);
  const int64_t es = d->dtype == FBSA_F32 ? 4 : 2, cpr = d->D * es / 16;
  EvictArgs a = {};
  a.k = (const char *)k; a.v = (const char *)v; a.ko = (char *)k_out; a.vo = (char *)v_out; a.w = weight; a.wo = w_out;
  a.lens = lens; a.index = index; a.new_lens = new_lens;
  for (int x = 0; x < 3; ++x) {
    a.sk[x] = d->sk[x] * es; a.sv[x] = d->sv[x] * es; a.sko[x] = d->sko[x] * es; a.svo[x] = d->svo[x] * es;
    if (x < 2) { a.sw[x] = d->sw[x]; a.swo[x] = d->swo[x]; }
  }
  a.B = (int)d->B; a.H = (int)d->H; a.S = (int)d->S; a.budget = (int)d->budget; a.recent = (int)d->recent; a.sink = (int)d->sink;
  a.ni = (int)ni; a.cpr = (int)cpr;
  const hipStream_t s = (hipStream_t)stream;
  const unsigned rows = (unsigned)(d->B * d->H);
  if (d->S <= kOneGroup) {
    const dim3 grid(rows), wg(kSelThreads);
    if (d->S <= 2 * kSelThreads) hipLaunchKernelGGL(evict_select_kernel<2>, grid, wg, 0, s, a);
    else if (d->S <= 8 * kSelThreads) hipLaunchKernelGGL(evict_select_kernel<8>, grid, wg, 0, s, a);
    else hipLaunchKernelGGL(evict_select_kernel<16>, grid, wg, 0, s, a);
    if ((e = hip_check(hipGetLastError(), "evict_select_kernel launch"))) return e;
  } else {
    char *p = (char *)workspace;
    EvictWs ws = {(uint32_t *)(p + pl.hist), (uint32_t *)(p + pl.cand), inplace ? (float *)(p + pl.copy) : nullptr, (uint2 *)(p + pl.count),
                  (uint2 *)(p + pl.start), (uint2 *)(p + pl.pick), (int)pl.nch};
    const dim3 grid((unsigned)pl.nch, rows), wg(kSelThreads);
    const int64_t nz = (int64_t)rows * kBins;
    hipLaunchKernelGGL(evict_zero_kernel, dim3((unsigned)((nz + 255) / 256)), dim3(256), 0, s, ws.hist, nz);
    hipLaunchKernelGGL(evict_hist_kernel, grid, wg, 0, s, a, ws);
    hipLaunchKernelGGL(evict_cand_kernel, grid, wg, 0, s, a, ws);
    hipLaunchKernelGGL(evict_rank_kernel, dim3(rows), wg, 0, s, a, ws);
    hipLaunchKernelGGL(evict_place_kernel, grid, wg, 0, s, a, ws);
    if ((e = hip_check(hipGetLastError(), "evict kernels launch"))) return e;
  }
  if (pl.part) {
    const int nt = (int)((ni + pl.part - 1) / pl.part);
    for (int t = 0; t <= nt; ++t)
      hipLaunchKernelGGL(evict_stage_kernel, dim3((unsigned)((pl.part * cpr + 255) / 256), rows, 2), dim3(256), 0, s, a,
                         (char *)workspace + pl.stage, (int)pl.part, t, nt);
    return hip_check(hipGetLastError(), "evict_stage_kernel launch");
  }
  if (inplace)
    hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)((cpr + 3) / 4), 2, rows), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(evict_copy_kernel, dim3((unsigned)((ni * cpr + 255) / 256), rows), dim3(256), 0, s, a);
  return hip_check(hipGetLastError(), inplace ? "evict_move_kernel launch" : "evict_copy_kernel launch");
}

}  // extern "C"
