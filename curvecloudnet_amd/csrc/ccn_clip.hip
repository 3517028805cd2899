// The global norm of many gradients, their clipping, and the Adam update that clips as it goes.
//
//   norm = sqrt(sum g^2)  |  sum |g|  |  max |g|    over every value of every tensor,   scale = min(1, max_norm / (norm + 1e-6))
// Squares and sums are held in 64 bits: a square of any fp32 value is far inside their range, so no value is too large or too small
// for the norm.  Every workgroup writes one partial result and every reader adds the partial results in the same order: the norm has
// the same bits in every run.  The tensors' addresses and sizes travel in the kernel's arguments (CLIP_MAX tensors per launch), so a
// captured launch holds them by value.
#include <math.h>

#include <algorithm>
#include <vector>

#include "ccn_common.h"

namespace {

constexpr int CLIP_TPB = 256;
constexpr int CLIP_MAX = 320;                      // tensors of one launch: 12 bytes of arguments each
constexpr int CLIP_PART_MAX = 1024;                // workgroups of one launch of the norm, each with a partial result
constexpr int CLIP_CHUNK = 16384;                  // values that a workgroup takes at a time, at most (clip_chunk_of)
constexpr int CLIP_SHORT = 512;                    // chunks of less than CLIP_CHUNK, at most
constexpr int CLIP_GRID = 64 * 1024;               // workgroups of one launch of the clipping, and of the update

// Tensor i is chunks first[i] ... first[i + 1] - 1.  at[i]: its address (bits 0-47), the length of its last chunk less one (48-61),
// its type (62-63).
struct ClipTable {
  uint64_t at[CLIP_MAX];
  int first[CLIP_MAX + 1];
  int n, chunk;                                    // tensors; values of a chunk, a power of two
};
static_assert(sizeof(ClipTable) + 64 < 4096, "kernel arguments");
static_assert(CLIP_CHUNK <= 1 << 14 && CLIP_MAX % 64 == 0, "fields of ClipTable");

enum { NORM_SUM = 1, NORM_TWO = 2, NORM_MAX = 3 };

// The entry of `first` (ascending, n of them in use) whose run holds chunk c: all lanes look at once, the entries sit in memory that
// is slow to reach for the first time.
template <int N>
__device__ __forceinline__ int clip_find(const int (&first)[N], int n, int c) {
  const int lane = threadIdx.x & 63;
  int found = 0;
#pragma unroll
  for (int k = 0; k < N / 64; ++k) {
    const int i = k * 64 + lane;
    found += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < n && first[i] <= c));
  }
  return __builtin_amdgcn_readfirstlane(found - 1);
}

// ---- a thread's share of the norm: sums in 64 bits; the maximum as the largest pattern of bits without the sign (a NaN's is above
// every number's, so it stays)
template <int KIND> struct ClipAcc { double v = 0.0; };
template <> struct ClipAcc<NORM_MAX> { uint32_t v = 0; };

template <int KIND, int T>
__device__ __forceinline__ void clip_add(ClipAcc<KIND>& a, float x) {
  if constexpr (KIND == NORM_MAX) a.v = max(a.v, __float_as_uint(x) & 0x7fffffffu);
  else if constexpr (KIND == NORM_TWO) a.v = __builtin_fma((double)x, (double)x, a.v);
  else a.v += (double)fabsf(x);
}
template <int KIND>
__device__ __forceinline__ double clip_value(const ClipAcc<KIND>& a) {
  if constexpr (KIND == NORM_MAX) return (double)__uint_as_float(a.v);
  else return a.v;
}
// (a NaN stays: fmax would drop it)
template <int KIND>
__device__ __forceinline__ double clip_join(double a, double b) {
  if (KIND != NORM_MAX) return a + b;
  return a != a ? a : (b > a || b != b ? b : a);
}

template <int KIND>
__device__ __forceinline__ double clip_block(double v, double* red) {
  v = ccn_wave_join(v, [](double a, double b) { return clip_join<KIND>(a, b); });
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int k = 1; k < CLIP_TPB / 64; ++k) v = clip_join<KIND>(v, red[k]);
  __syncthreads();
  return v;
}

// n <= CLIP_CHUNK values at p: eight 16-byte loads of a thread in flight
template <int KIND, int T>
__device__ __forceinline__ void clip_sum(ClipAcc<KIND>& a, const char* p, int n) {
  constexpr int V = CcnVec16<T>::N, STEP = CLIP_TPB * V, U = 8;
  int i = threadIdx.x * V;
  for (; i - (int)threadIdx.x * V + U * STEP <= n; i += U * STEP) {
    ccn_u32x4 r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = ld16<T>(p, i + u * STEP);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < V; ++k) clip_add<KIND, T>(a, get16<T>(r[u], k));
  }
  ccn_u32x4 r[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    r[u] = ccn_u32x4{0, 0, 0, 0};
    if (i + u * STEP + V <= n) r[u] = ld16<T>(p, i + u * STEP);
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (i + u * STEP + V <= n)
#pragma unroll
      for (int k = 0; k < V; ++k) clip_add<KIND, T>(a, get16<T>(r[u], k));
  const int whole = n / V * V;
  if ((int)threadIdx.x < n - whole) clip_add<KIND, T>(a, ld_el<T>(p, whole + threadIdx.x));
}

// The first pass, bound by memory: 260M fp32 values 221 us (4.7 TB/s, while the lines that an update wrote before leave the cache), 400M bf16
// 197 us behind a clipping of them, 141 (5.7 TB/s) behind a pass that wrote nothing.  1024 workgroups take chunks in turn; 2048 or 4096 of
// them, 4 or 16 loads in flight are within 3 %.
template <int KIND>
__global__ __launch_bounds__(CLIP_TPB) void grad_norm_kernel(const ClipTable t, double* __restrict__ partial) {
  __shared__ double red[CLIP_TPB / 64];
  const int chunks = t.first[t.n];
  ClipAcc<KIND> a;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = clip_find(t.first, t.n, c);
    const uint64_t at = t.at[i];
    const int n = c + 1 == t.first[i + 1] ? (int)((at >> 48) & 0x3fff) + 1 : t.chunk, type = (int)(at >> 62);
    const char* const p = reinterpret_cast<const char*>(at & 0xffffffffffffull) + (int64_t)(c - t.first[i]) * t.chunk * (type ? 2 : 4);
    if (type == 0) clip_sum<KIND, 0>(a, p, n);
    else if (type == 1) clip_sum<KIND, 1>(a, p, n);
    else clip_sum<KIND, 2>(a, p, n);
  }
  const double v = clip_block<KIND>(clip_value<KIND>(a), red);
  if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

// Every thread of the workgroup gets the norm, from the partial results in a fixed order.
template <int KIND>
__device__ __forceinline__ double clip_total(const double* __restrict__ partial, int n, double* red) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += CLIP_TPB) v = clip_join<KIND>(v, partial[i]);
  v = clip_block<KIND>(v, red);
  return KIND == NORM_TWO ? sqrt(v) : v;
}
__device__ __forceinline__ float clip_scale(double norm, double max_norm) {
  const double s = max_norm / (norm + 1e-6);
  return s != s ? NAN : s < 1.0 ? (float)s : 1.f;       // (a NaN norm makes every gradient NaN; an infinite one 0, and NaN where infinite)
}

// The norm, and the factor of the kernels that follow where there are many of their workgroups.
template <int KIND>
__global__ __launch_bounds__(CLIP_TPB) void grad_norm_final_kernel(const double* __restrict__ partial, int n, double max_norm,
                                                                   float* __restrict__ norm, float* __restrict__ scale) {
  __shared__ double red[CLIP_TPB / 64];
  const double v = clip_total<KIND>(partial, n, red);
  if (threadIdx.x == 0) {
    *norm = (float)v;
    if (scale) *scale = clip_scale(v, max_norm);
  }
}

// The factor is rounded to the gradients' type first, as a torch tensor's product with a scalar tensor rounds it: the same bits come out,
// for half a step of the type more than with the factor in 32 bits.  That half step is common to all values, so the norm that is left is
// off by it too, 2^-8 of max_norm at most for bf16 (2^-11 for fp16) in either direction, and a bf16 factor above 1 - 2^-9 is 1.  Below the
// normal numbers of fp16, where half a step can be all of the factor (a norm of 10^7 and a bound of 0.1), it stays in 32 bits.
template <int T>
__device__ __forceinline__ float clip_factor_of(float scale) {
  if (T == 2 && scale < 0x1p-14f) return scale;
  ccn_u32x4 of_type = {0, 0, 0, 0};
  put16<T>(of_type, 0, scale);
  return get16<T>(of_type, 0);
}
template <int T>
__device__ __forceinline__ void clip_apply(char* p, int n, float scale) {
  scale = clip_factor_of<T>(scale);
  constexpr int V = CcnVec16<T>::N, STEP = CLIP_TPB * V, U = 4;
  for (int i = threadIdx.x * V; i - (int)threadIdx.x * V < n; i += U * STEP) {
    ccn_u32x4 r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      r[u] = ccn_u32x4{0, 0, 0, 0};
      if (i + u * STEP + V <= n) r[u] = ld16<T>(p, i + u * STEP);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ccn_u32x4 o;
#pragma unroll
      for (int k = 0; k < V; ++k) put16<T>(o, k, get16<T>(r[u], k) * scale);
      if (i + u * STEP + V <= n) st16<T>(p, i + u * STEP, o);
    }
  }
  const int whole = n / V * V;
  if ((int)threadIdx.x < n - whole) st_el<T>(p, whole + threadIdx.x, ld_el<T>(p, whole + threadIdx.x) * scale);
}

// The second pass, bound by memory: 400M bf16 values 257 us (6.2 TB/s of reads and writes); 310 tensors of 5.3M fp32 14 us (3 TB/s, in chunks
// of 2048 as of 16384), the waves waiting for 83 % of that: for the partial results, then for their values.
template <int KIND>
__global__ __launch_bounds__(CLIP_TPB) void grad_clip_kernel(const ClipTable t, const double* __restrict__ partial, int count,
                                                             double max_norm, float* __restrict__ norm,
                                                             const float* __restrict__ ready) {
  __shared__ double red[CLIP_TPB / 64];
  float scale;
  if (ready) {
    scale = *ready;
  } else {
    const double v = clip_total<KIND>(partial, count, red);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
    scale = clip_scale(v, max_norm);
  }
  if (scale == 1.f) return;
  // (from the last chunk to the first: what the norm read last is the likeliest to sit in a cache still)
  for (int c = t.first[t.n] - 1 - (int)blockIdx.x; c >= 0; c -= (int)gridDim.x) {
    const int i = clip_find(t.first, t.n, c);
    const uint64_t at = t.at[i];
    const int n = c + 1 == t.first[i + 1] ? (int)((at >> 48) & 0x3fff) + 1 : t.chunk, type = (int)(at >> 62);
    char* const p = reinterpret_cast<char*>(at & 0xffffffffffffull) + (int64_t)(c - t.first[i]) * t.chunk * (type ? 2 : 4);
    if (type == 0) clip_apply<0>(p, n, scale);
    else if (type == 1) clip_apply<1>(p, n, scale);
    else clip_apply<2>(p, n, scale);
  }
}

// ---- few values (pieces of SMALL_PIECE of a tensor, two to a wave at most): one workgroup keeps them in registers between the norm and
// the product, one launch does both: 6 tensors of 9001 fp32 values take 6.2 us with their call, 9.8 in two launches; 65536 values 9.6 and
// 9.8, of bf16 7.5 and 10.0.  max_norm < 0: the norm alone.  (1024 threads leave 128 registers each: four of them spill, but for the largest
// magnitude.)
constexpr int SMALL_TPB = 1024, SMALL_PIECE = 2048, SMALL_EACH = 2, SMALL_MAX = SMALL_EACH * SMALL_TPB / 64;
static_assert(SMALL_MAX <= 64, "found by one look of a wave");

struct SmallHeld {
  ccn_u32x4 whole[SMALL_PIECE / 256];
  float rest;                                      // (a lane's share of the values behind the last 16 whole bytes)
};
template <int KIND, int T>
__device__ __forceinline__ void small_read(ClipAcc<KIND>& a, SmallHeld& h, const char* p, int n) {
  constexpr int V = CcnVec16<T>::N, NJ = SMALL_PIECE / 64 / V;
  const int lane = threadIdx.x & 63, whole = n / V * V;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    h.whole[j] = ccn_u32x4{0, 0, 0, 0};
    if ((j * 64 + lane) * V < whole) h.whole[j] = ld16<T>(p, (j * 64 + lane) * V);
  }
  h.rest = lane < n - whole ? ld_el<T>(p, whole + lane) : 0.f;
#pragma unroll
  for (int j = 0; j < NJ; ++j)
    if (j * 64 * V < whole) {
#pragma unroll
      for (int k = 0; k < V; ++k) clip_add<KIND, T>(a, get16<T>(h.whole[j], k));
    }
  clip_add<KIND, T>(a, h.rest);
}
template <int T>
__device__ __forceinline__ void small_write(const SmallHeld& h, char* p, int n, float scale) {
  constexpr int V = CcnVec16<T>::N, NJ = SMALL_PIECE / 64 / V;
  const int lane = threadIdx.x & 63, whole = n / V * V;
  scale = clip_factor_of<T>(scale);
#pragma unroll
  for (int j = 0; j < NJ; ++j)
    if ((j * 64 + lane) * V < whole) {
      ccn_u32x4 o;
#pragma unroll
      for (int k = 0; k < V; ++k) put16<T>(o, k, get16<T>(h.whole[j], k) * scale);
      st16<T>(p, (j * 64 + lane) * V, o);
    }
  if (lane < n - whole) st_el<T>(p, whole + lane, h.rest * scale);
}

template <int KIND>
__global__ __launch_bounds__(SMALL_TPB) void grad_small_kernel(const ClipTable t, double max_norm, float* __restrict__ norm) {
  __shared__ double red[SMALL_TPB / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, pieces = t.first[t.n];
  SmallHeld held[SMALL_EACH];
  char* p[SMALL_EACH];
  int n[SMALL_EACH], type[SMALL_EACH];
  ClipAcc<KIND> a;
#pragma unroll
  for (int u = 0; u < SMALL_EACH; ++u) {
    const int c = wave + u * (SMALL_TPB / 64);
    n[u] = type[u] = 0;
    p[u] = nullptr;
    if (c < pieces) {
      const int i = __builtin_amdgcn_readfirstlane(__builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < t.n && t.first[lane] <= c))) - 1;
      const uint64_t at = t.at[i];
      n[u] = c + 1 == t.first[i + 1] ? (int)((at >> 48) & 0x3fff) + 1 : SMALL_PIECE;
      type[u] = (int)(at >> 62);
      p[u] = reinterpret_cast<char*>(at & 0xffffffffffffull) + (c - t.first[i]) * SMALL_PIECE * (type[u] ? 2 : 4);
      if (type[u] == 0) small_read<KIND, 0>(a, held[u], p[u], n[u]);
      else if (type[u] == 1) small_read<KIND, 1>(a, held[u], p[u], n[u]);
      else small_read<KIND, 2>(a, held[u], p[u], n[u]);
    }
  }
  double v = ccn_wave_join(clip_value<KIND>(a), [](double x, double y) { return clip_join<KIND>(x, y); });
  if (lane == 0) red[wave] = v;
  __syncthreads();
  v = red[0];
  for (int k = 1; k < SMALL_TPB / 64; ++k) v = clip_join<KIND>(v, red[k]);
  if (KIND == NORM_TWO) v = sqrt(v);
  if (threadIdx.x == 0) *norm = (float)v;
  if (max_norm < 0.0) return;
  const float scale = clip_scale(v, max_norm);
  if (scale == 1.f) return;
#pragma unroll
  for (int u = 0; u < SMALL_EACH; ++u)
    if (n[u]) {
      if (type[u] == 0) small_write<0>(held[u], p[u], n[u], scale);
      else if (type[u] == 1) small_write<1>(held[u], p[u], n[u], scale);
      else small_write<2>(held[u], p[u], n[u], scale);
    }
}

// ---- Adam over several runs of parameters with the gradients scaled on the way: 16 bytes read and 12 written for every value, bound by memory
// (260M values 1375 us, 5.3 TB/s; 19.7M 90 us, 6.1; without a bound the call takes 1359 and 84 us)
constexpr int ADAM_MAX = 64;
constexpr int ADAM_CHUNK = 4096;

struct AdamTable {
  float* p[ADAM_MAX];
  const float* g[ADAM_MAX];
  float* m[ADAM_MAX];
  float* v[ADAM_MAX];
  int64_t size[ADAM_MAX];
  int first[ADAM_MAX + 1];
  int n;
};
static_assert(sizeof(AdamTable) + 96 < 4096, "kernel arguments");

struct AdamCoef {
  float scale, beta1_rest, beta2, beta2_rest, step_size, inv_bc2_sqrt, eps, decay;
};
__device__ __forceinline__ void adam_one(float& p, float g, float& m, float& v, const AdamCoef& k) {
  const float grad = g * k.scale + k.decay * p;
  m = m + (grad - m) * k.beta1_rest;
  v = v * k.beta2 + k.beta2_rest * grad * grad;
  p = p - k.step_size * (m / (sqrtf(v) * k.inv_bc2_sqrt + k.eps));
}

__global__ __launch_bounds__(CLIP_TPB) void adam_clip_kernel(const AdamTable t, const double* __restrict__ partial, int count,
                                                             double max_norm, float* __restrict__ norm,
                                                             const float* __restrict__ ready, AdamCoef k) {
  __shared__ double red[CLIP_TPB / 64];
  if (ready) {
    k.scale = *ready;
  } else if (partial) {                                // (no partial results: no bound, and k.scale is 1)
    const double total = clip_total<NORM_TWO>(partial, count, red);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
    k.scale = clip_scale(total, max_norm);
  }
  for (int c = t.first[t.n] - 1 - (int)blockIdx.x; c >= 0; c -= (int)gridDim.x) {     // (as in grad_clip_kernel)
    const int lane = threadIdx.x & 63;
    const int i = __builtin_amdgcn_readfirstlane(__builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < t.n && t.first[lane] <= c))) - 1;
    const int64_t from = (int64_t)(c - t.first[i]) * ADAM_CHUNK;
    const int n = (int)min((int64_t)ADAM_CHUNK, t.size[i] - from);
    float* const p = t.p[i] + from;
    const float* const g = t.g[i] + from;
    float* const m = t.m[i] + from;
    float* const v = t.v[i] + from;
    for (int e = threadIdx.x * 4; e + 4 <= n; e += CLIP_TPB * 4) {
      float4 pp = *(const float4*)(p + e), mm = *(const float4*)(m + e), vv = *(const float4*)(v + e);
      const float4 gg = *(const float4*)(g + e);
      adam_one(pp.x, gg.x, mm.x, vv.x, k);
      adam_one(pp.y, gg.y, mm.y, vv.y, k);
      adam_one(pp.z, gg.z, mm.z, vv.z, k);
      adam_one(pp.w, gg.w, mm.w, vv.w, k);
      *(float4*)(p + e) = pp;
      *(float4*)(m + e) = mm;
      *(float4*)(v + e) = vv;
    }
    const int e = n / 4 * 4 + threadIdx.x;
    if (e < n) {
      float pp = p[e], mm = m[e], vv = v[e];
      adam_one(pp, g[e], mm, vv, k);
      p[e] = pp;
      m[e] = mm;
      v[e] = vv;
    }
  }
}

int clip_check(const void* const* ptr, const int64_t* size, const int32_t* dtype, int64_t n, bool writes, const char* who) {
  CCN_REQUIRE(n >= 0 && n < (1 << 24) && (n == 0 || (ptr && size)), "%s: n=%lld, or a null table", who, (long long)n);
  for (int64_t i = 0; i < n; ++i) {
    const int64_t el = dtype && dtype[i] ? 2 : 4;
    CCN_REQUIRE(!dtype || (dtype[i] >= 0 && dtype[i] <= 2), "%s: tensor %lld: dtype %d is not 0 (fp32), 1 (bf16) or 2 (fp16)", who,
                (long long)i, dtype ? dtype[i] : 0);
    CCN_REQUIRE(size[i] >= 0 && size[i] < ((int64_t)1 << 36), "%s: tensor %lld has %lld values", who, (long long)i, (long long)size[i]);
    CCN_REQUIRE(size[i] == 0 || (ptr[i] && ((uintptr_t)ptr[i] & (uintptr_t)(el - 1)) == 0 && (uintptr_t)ptr[i] < (uintptr_t)1 << 48),
                "%s: tensor %lld: null or not aligned to its type", who, (long long)i);
  }
  if (!writes) return CCN_OK;
  int runs = 0;                                      // tensors of one buffer mostly come in order: few ascending runs are merged
  size_t run[8];                                     // (where the second and later ones start)
  std::vector<std::pair<uintptr_t, uintptr_t>> span;
  try {
    span.reserve((size_t)n);
  } catch (...) {
    ccn_set_error("%s: out of host memory", who);
    return CCN_ERR_ARG;
  }
  for (int64_t i = 0; i < n; ++i) {
    if (size[i] == 0) continue;
    const uintptr_t a = (uintptr_t)ptr[i], b = a + (uintptr_t)size[i] * (dtype && dtype[i] ? 2 : 4);
    if (!span.empty() && a < span.back().first && runs++ < 8) run[runs - 1] = span.size();
    span.emplace_back(a, b);
  }
  if (runs > 8) std::sort(span.begin(), span.end());
  else
    for (int k = 0; k < runs; ++k)
      std::inplace_merge(span.begin(), span.begin() + run[k], k + 1 < runs ? span.begin() + run[k + 1] : span.end());
  for (size_t i = 1; i < span.size(); ++i)
    CCN_REQUIRE(span[i - 1].second <= span[i].first, "%s: two of the tensors share memory (the same one given twice?)", who);
  return CCN_OK;
}

int clip_chunks(int64_t size, int chunk) { return (int)((size + chunk - 1) / chunk); }

// The tables of the launches that a list of tensors takes: f(table) for each.
template <typename F>
int clip_tables(const void* const* ptr, const int64_t* size, const int32_t* dtype, int64_t n, int chunk, F f) {
  ClipTable t;
  t.chunk = chunk;
  t.n = 0;
  t.first[0] = 0;
  for (int64_t i = 0; i < n; ++i) {
    if (size[i] == 0) continue;
    t.at[t.n] = (uint64_t)(uintptr_t)ptr[i] | ((uint64_t)((size[i] - 1) & (chunk - 1)) << 48) | ((uint64_t)(dtype ? dtype[i] : 0) << 62);
    t.first[t.n + 1] = t.first[t.n] + clip_chunks(size[i], chunk);
    if (++t.n == CLIP_MAX) {
      if (int rc = f(t)) return rc;
      t.n = 0;
    }
  }
  return t.n ? f(t) : CCN_OK;
}

#define CLIP_KINDS(kind, KERNEL, ...)                                                              \
  do {                                                                                             \
    if ((kind) == NORM_TWO) hipLaunchKernelGGL(KERNEL<NORM_TWO>, __VA_ARGS__);                     \
    else if ((kind) == NORM_SUM) hipLaunchKernelGGL(KERNEL<NORM_SUM>, __VA_ARGS__);                \
    else hipLaunchKernelGGL(KERNEL<NORM_MAX>, __VA_ARGS__);                                        \
  } while (0)

// Short chunks where there are few, for more workgroups and more of a chunk in flight at once (clipping, events included, in chunks of 16384 /
// here: 0.2M fp32 values 14.0 / 11.4 us, 1M 15.6 / 12.4, 2.1M 16.8 / 15.1, 2M bf16 13.4 / 11.8; with up to 256 or 1024 chunks instead of 512 2.1M take
// 17.0 and 16.1).
int clip_chunk_of(const int64_t* size, int64_t n, int64_t* chunks) {
  for (int chunk = 2048;; chunk *= 2) {
    *chunks = 0;
    for (int64_t i = 0; i < n; ++i) *chunks += clip_chunks(size[i], chunk);
    if (chunk == CLIP_CHUNK || *chunks <= CLIP_SHORT) return chunk;
  }
}

int clip_grid(int chunks, int most) { return chunks < most ? chunks : most; }

// The partial results of the norm: *count of them, at `partial`.
int clip_norm_launches(const void* const* ptr, const int64_t* size, const int32_t* dtype, int64_t n, int chunk, int kind, double* partial,
                       int* count, hipStream_t s) {
  *count = 0;
  return clip_tables(ptr, size, dtype, n, chunk, [&](const ClipTable& t) {
    const int grid = clip_grid(t.first[t.n], CLIP_PART_MAX);
    CLIP_KINDS(kind, grad_norm_kernel, dim3(grid), dim3(CLIP_TPB), 0, s, t, partial + *count);
    *count += grid;
    return CCN_OK;
  });
}

// Whether grad_small_kernel does it all.
bool clip_is_small(const int64_t* size, int64_t n) {
  int64_t pieces = 0;
  for (int64_t i = 0; i < n && pieces <= SMALL_MAX; ++i) pieces += (size[i] + SMALL_PIECE - 1) / SMALL_PIECE;
  return pieces > 0 && pieces <= SMALL_MAX;
}
int clip_small(const void* const* ptr, const int64_t* size, const int32_t* dtype, int64_t n, int kind, double max_norm, float* norm,
               hipStream_t s) {
  return clip_tables(ptr, size, dtype, n, SMALL_PIECE, [&](const ClipTable& t) {
    CLIP_KINDS(kind, grad_small_kernel, dim3(1), dim3(SMALL_TPB), 0, s, t, max_norm, norm);
    return CCN_OK;
  });
}

int clip_outputs(const void* norm, const void* ws, size_t ws_bytes, int64_t n, const char* who) {
  CCN_REQUIRE(norm && ws && (uintptr_t)ws % 8 == 0, "%s: null norm or workspace", who);
  if (ws_bytes < ccn_grad_norm_workspace_bytes(n)) {
    ccn_set_error("%s: workspace %zu < %zu bytes", who, ws_bytes, ccn_grad_norm_workspace_bytes(n));
    return CCN_ERR_WORKSPACE;
  }
  return CCN_OK;
}

// Where the kernels that apply the factor have more workgroups than CLIP_PART_MAX, each of them adding up the partial results costs
// more than a launch that does it once.
float* clip_factor(int kind, const double* partial, int count, double max_norm, float* norm, int64_t chunks, hipStream_t s) {
  if (count > 0 && chunks <= CLIP_PART_MAX) return nullptr;
  float* const factor = (float*)const_cast<double*>(partial + count);
  CLIP_KINDS(kind, grad_norm_final_kernel, dim3(1), dim3(CLIP_TPB), 0, s, partial, count, max_norm, norm, factor);
  return factor;
}

}  // namespace

// (a partial result for every workgroup, and the factor behind them)
extern "C" size_t ccn_grad_norm_workspace_bytes(int64_t n) {
  if (n < 0) return 0;
  const int64_t launches = (n + CLIP_MAX - 1) / CLIP_MAX;
  return ccn_align256(((size_t)(launches < 1 ? 1 : launches) * CLIP_PART_MAX + 1) * sizeof(double));
}

extern "C" int ccn_grad_norm(const void* const* grads, const int64_t* sizes, const int32_t* dtypes, int64_t n, int kind, void* ws,
                             size_t ws_bytes, float* norm, void* stream) {
  if (int rc = clip_check(grads, sizes, dtypes, n, false, "grad_norm")) return rc;
  CCN_REQUIRE(kind >= NORM_SUM && kind <= NORM_MAX, "grad_norm: kind %d is not 1 (sum), 2 (two) or 3 (max)", kind);
  if (int rc = clip_outputs(norm, ws, ws_bytes, n, "grad_norm")) return rc;
  double* const partial = (double*)ws;
  int count = 0;
  int64_t chunks;
  const int chunk = clip_chunk_of(sizes, n, &chunks);
  hipStream_t s = (hipStream_t)stream;
  if (clip_is_small(sizes, n)) {
    if (int rc = clip_small(grads, sizes, dtypes, n, kind, -1.0, norm, s)) return rc;
    CCN_LAUNCH_OK("grad_norm");
    return CCN_OK;
  }
  if (int rc = clip_norm_launches(grads, sizes, dtypes, n, chunk, kind, partial, &count, s)) return rc;
  CLIP_KINDS(kind, grad_norm_final_kernel, dim3(1), dim3(CLIP_TPB), 0, s, partial, count, 0.0, norm, nullptr);
  CCN_LAUNCH_OK("grad_norm");
  return CCN_OK;
}

extern "C" int ccn_grad_clip(void* const* grads, const int64_t* sizes, const int32_t* dtypes, int64_t n, int kind, double max_norm,
                             void* ws, size_t ws_bytes, float* norm, void* stream) {
  if (int rc = clip_check(grads, sizes, dtypes, n, true, "grad_clip")) return rc;
  CCN_REQUIRE(kind >= NORM_SUM && kind <= NORM_MAX, "grad_clip: kind %d is not 1 (sum), 2 (two) or 3 (max)", kind);
  CCN_REQUIRE(max_norm >= 0.0, "grad_clip: max_norm %g", max_norm);
  if (int rc = clip_outputs(norm, ws, ws_bytes, n, "grad_clip")) return rc;
  double* const partial = (double*)ws;
  int count = 0;
  int64_t chunks;
  const int chunk = clip_chunk_of(sizes, n, &chunks);
  hipStream_t s = (hipStream_t)stream;
  if (clip_is_small(sizes, n)) {
    if (int rc = clip_small(grads, sizes, dtypes, n, kind, max_norm, norm, s)) return rc;
    CCN_LAUNCH_OK("grad_clip");
    return CCN_OK;
  }
  if (int rc = clip_norm_launches(grads, sizes, dtypes, n, chunk, kind, partial, &count, s)) return rc;
  const float* const factor = clip_factor(kind, partial, count, max_norm, norm, chunks, s);
  float* out = factor ? nullptr : norm;
  const int rc = clip_tables(grads, sizes, dtypes, n, chunk, [&](const ClipTable& t) {
    CLIP_KINDS(kind, grad_clip_kernel, dim3(clip_grid(t.first[t.n], CLIP_GRID)), dim3(CLIP_TPB), 0, s, t, partial, count, max_norm,
               out, factor);
    out = nullptr;
    return CCN_OK;
  });
  if (rc) return rc;
  CCN_LAUNCH_OK("grad_clip");
  return CCN_OK;
}

extern "C" int ccn_adam_clip(float* const* params, const float* const* grads, float* const* exp_avgs, float* const* exp_avg_sqs,
                             const int64_t* sizes, int64_t n, double lr, double beta1, double beta2, double eps,
                             double weight_decay, int64_t step, double max_norm, void* ws, size_t ws_bytes, float* norm, void* stream) {
  CCN_REQUIRE(step >= 1, "adam_clip: step=%lld", (long long)step);
  CCN_REQUIRE(n >= 0 && (n == 0 || (params && grads && exp_avgs && exp_avg_sqs && sizes)), "adam_clip: n=%lld, or a null table",
              (long long)n);
  CCN_REQUIRE(max_norm >= 0.0, "adam_clip: max_norm %g", max_norm);
  const bool bounded = norm || ws || isfinite(max_norm);
  if (int rc = clip_check((const void* const*)grads, sizes, nullptr, n, false, "adam_clip")) return rc;
  std::vector<const void*> all;
  std::vector<int64_t> every;
  int64_t chunks = 0, of_norm;
  try {                                              // nothing that is written may share memory with anything else that is used
    all.reserve((size_t)(4 * n));
    every.reserve((size_t)(4 * n));
    for (const void* const* list : {(const void* const*)params, (const void* const*)grads, (const void* const*)exp_avgs,
                                    (const void* const*)exp_avg_sqs})
      for (int64_t i = 0; i < n; ++i) {
        CCN_REQUIRE((uintptr_t)list[i] % 16 == 0, "adam_clip: buffers must be 16-byte aligned");
        all.push_back(list[i]);
        every.push_back(sizes[i]);
      }
    for (int64_t i = 0; i < n; ++i) chunks += clip_chunks(sizes[i], ADAM_CHUNK);
  } catch (...) {
    ccn_set_error("adam_clip: out of host memory");
    return CCN_ERR_ARG;
  }
  if (int rc = clip_check(all.data(), every.data(), nullptr, 4 * n, true, "adam_clip")) return rc;
  double* const partial = (double*)ws;
  int count = 0;
  hipStream_t s = (hipStream_t)stream;
  const float* factor = nullptr;
  if (bounded) {
    if (int rc = clip_outputs(norm, ws, ws_bytes, n, "adam_clip")) return rc;
    if (int rc = clip_norm_launches((const void* const*)grads, sizes, nullptr, n, clip_chunk_of(sizes, n, &of_norm), NORM_TWO, partial, &count, s)) return rc;
    factor = clip_factor(NORM_TWO, partial, count, max_norm, norm, chunks, s);
  }
  float* out = factor ? nullptr : norm;
  // bias corrections and 1 - beta in double on the host (1 - 0.999 from a beta in 32 bits is off by 1.3e-5 of itself)
  const double bc1 = 1.0 - pow(beta1, (double)step), bc2 = 1.0 - pow(beta2, (double)step);
  const AdamCoef coef = {1.f, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)(lr / bc1), (float)(1.0 / sqrt(bc2)),
                         (float)eps, (float)weight_decay};
  AdamTable t;
  t.n = 0;
  t.first[0] = 0;
  for (int64_t i = 0; i < n; ++i) {
    if (sizes[i] > 0) {
      t.p[t.n] = params[i];
      t.g[t.n] = grads[i];
      t.m[t.n] = exp_avgs[i];
      t.v[t.n] = exp_avg_sqs[i];
      t.size[t.n] = sizes[i];
      t.first[t.n + 1] = t.first[t.n] + clip_chunks(sizes[i], ADAM_CHUNK);
      ++t.n;
    }
    if (t.n == ADAM_MAX || (i == n - 1 && t.n > 0)) {
      hipLaunchKernelGGL(adam_clip_kernel, dim3(clip_grid(t.first[t.n], CLIP_GRID)), dim3(CLIP_TPB), 0, s, t, partial, count, max_norm,
                         out, factor, coef);
      out = nullptr;
      t.n = 0;
    }
  }
  CCN_LAUNCH_OK("adam_clip");
  return CCN_OK;
}
