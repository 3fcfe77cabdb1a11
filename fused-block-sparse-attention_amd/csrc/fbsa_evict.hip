// What changes a cache of keys and values on gfx950: new rows written behind
// each sequence, and rows thrown away by the attention weight they gathered.
//
// Eviction keeps, of a (sequence, head) with n > budget rows, the first `sink`,
// the last `recent` and the K = budget - sink - recent greatest weights between.
// Weights become unsigned keys of the same order; the K-th greatest is found by
// a radix select, a byte a pass, and one ordered pass over the rows then writes
// the kept rows' numbers and weights (ties to the lower row: of the rows that
// equal the K-th greatest the first are kept). A second kernel moves the rows.
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

// a 16-byte chunk of a new key row and of its value row per thread
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

// unsigned key of the same order; NaN as -inf, -0 as 0
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (!(w == w)) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;

__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.x % a.H, b = blockIdx.x / a.H;
  const int n = evict_len(a, b);
  const float *w = a.w + b * a.sw[0] + h * a.sw[1];
  float *wo = a.wo + b * a.swo[0] + h * a.swo[1];
  int32_t *index = a.index + (int64_t)blockIdx.x * a.ni;
  const int kept = n < a.budget ? n : a.budget;
  if (h == 0 && tid == 0) a.new_lens[b] = kept;
  for (int i = kept + tid; i < a.ni; i += kSelThreads) index[i] = -1;

  __shared__ uint32_t hist[256];
  __shared__ uint32_t s_prefix, s_need;
  __shared__ int s_def[kSelWaves], s_eq[kSelWaves];
  const int lo = a.sink, hi = n - a.recent;       // rows that the weight decides about (n > budget)
  uint32_t need = n > a.budget ? (uint32_t)(a.budget - a.recent - a.sink) : 0, prefix = 0;
  if (need) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += kSelThreads) {
        const uint32_t key = weight_key(w[i]);
        if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&hist[key >> shift & 255], 1u);
      }
      __syncthreads();
      if (wave == 0) {
        // lane l holds bins 255 - 4l - j, j = 0..3: counts in descending key order
        uint32_t c[4], sum = 0;
        for (int j = 0; j < 4; ++j) sum += c[j] = hist[255 - 4 * lane - j];
        uint32_t before = sum;
        for (int x = 1; x < 64; x <<= 1) {
          const uint32_t y = __shfl_up(before, x, 64);
          if (lane >= x) before += y;
        }
        before -= sum;
        for (int j = 0; j < 4; ++j) {
          if (before < need && need <= before + c[j]) {
            s_prefix = prefix << 8 | (uint32_t)(255 - 4 * lane - j);
            s_need = need - before;
          }
          before += c[j];
        }
      }
      __syncthreads();
      prefix = s_prefix;
      need = s_need;
    }
  }
  // rows above the K-th greatest key are kept, and the first `need` that equal it
  int ndef = 0, neq = 0;  // of the rows before this step's
  const bool all = n <= a.budget, mid = !all && a.budget > a.recent + a.sink;
  for (int base = 0; base < n; base += kSelThreads) {
    const int i = base + tid;
    bool def = false, eq = false;
    float x = 0.f;
    if (i < n) {
      x = w[i];
      if (all || i < lo || i >= hi) def = true;
      else if (mid) {
        const uint32_t key = weight_key(x);
        def = key > prefix;
        eq = key == prefix;
      }
    }
    const uint64_t md = __ballot(def), me = __ballot(eq), below = (1ull << lane) - 1;
    if (lane == 0) { s_def[wave] = __popcll(md); s_eq[wave] = __popcll(me); }
    __syncthreads();
    int d0 = ndef + __popcll(md & below), e0 = neq + __popcll(me & below);
    for (int v = 0; v < kSelWaves; ++v) {
      if (v < wave) { d0 += s_def[v]; e0 += s_eq[v]; }
      ndef += s_def[v];
      neq += s_eq[v];
    }
    if (def || (eq && e0 < (int)need)) {
      const int at = d0 + (e0 < (int)need ? e0 : (int)need);
      index[at] = i;
      wo[at] = x;  // (in place: at <= i, and every row up to this step's last has been read)
    }
    __syncthreads();
  }
}

// rows to other buffers: a 16-byte chunk of a key row and of its value row per thread
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
constexpr int kMoveU = 8, kMove = 64 * kMoveU;
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

constexpr int64_t kMaxRows = 0x7fff0000LL;

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
      d->B * d->H > kMaxRows / d->T || (d->B * d->H * d->T * cpr + 255) / 256 > kMaxRows)
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

int fbsa_cache_evict(const fbsa_evict_desc *d, const void *k, const void *v, const float *weight, const int32_t *lens, void *k_out,
                     void *v_out, float *w_out, int32_t *index, int32_t *new_lens, void *stream) {
  static const char *fn = "fbsa_cache_evict";
  if (!d) return fail(FBSA_EINVAL, "%s: null descriptor", fn);
  const int64_t(*const st[])[3] = {&d->sk, &d->sv, &d->sko, &d->svo};
  static const char *const name[] = {"k", "v", "k_out", "v_out"};
  int e = check_rows(fn, d->dtype, d->D, st, name, 4);
  if (e) return e;
  const bool inplace = d->flags & FBSA_EVICT_IN_PLACE;
  if (d->flags & ~FBSA_EVICT_IN_PLACE) return fail(FBSA_EINVAL, "%s: unknown flags 0x%x", fn, d->flags);
  if (d->B < 1 || d->H < 1 || d->S < 1 || d->budget < 1)
    return fail(FBSA_EINVAL, "%s: sizes must be positive (B=%lld H=%lld S=%lld budget=%lld)", fn, (long long)d->B, (long long)d->H,
                (long long)d->S, (long long)d->budget);
  if (d->recent < 0 || d->sink < 0 || d->recent > d->budget || d->sink > d->budget - d->recent)
    return fail(FBSA_EINVAL, "%s: recent=%lld and sink=%lld must be non-negative and fit the budget of %lld", fn, (long long)d->recent,
                (long long)d->sink, (long long)d->budget);
  const int64_t ni = d->budget < d->S ? d->budget : d->S;
  if (d->SO < ni) return fail(FBSA_EINVAL, "%s: output capacity %lld is below %lld", fn, (long long)d->SO, (long long)ni);
  if (d->S > kMaxRows || d->budget > kMaxRows || d->B > 65535 || d->H > 65535 || d->B * d->H > 65535)
    return fail(FBSA_EUNSUPPORTED, "%s: sizes exceed the grid or 32-bit row indices", fn);
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
  hipLaunchKernelGGL(evict_select_kernel, dim3(rows), dim3(kSelThreads), 0, s, a);
  if ((e = hip_check(hipGetLastError(), "evict_select_kernel launch"))) return e;
  if (inplace)
    hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)((cpr + 3) / 4), 2, rows), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(evict_copy_kernel, dim3((unsigned)((ni * cpr + 255) / 256), rows), dim3(256), 0, s, a);
  return hip_check(hipGetLastError(), inplace ? "evict_move_kernel launch" : "evict_copy_kernel launch");
}

}  // extern "C"
