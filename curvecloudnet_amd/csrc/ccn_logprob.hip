// Log-probabilities of given classes, the entropy of every row and its best alternatives, with their gradient.
//
// For a row x of C logits, m = max x, S = sum exp(x - m), W = sum exp(x - m) (x - m):
//   logprob = (x_t - m) - log S,   entropy = log S - W / S        (both terms of the entropy are >= 0)
//   alternatives: the `top` largest logits, equal ones by ascending class, and their log-probabilities.
// Backward, with l = (x - m) - log S, p = exp(l), G = g_logprob + sum_j g_top_j:
//   dx_i = -p_i (G + g_entropy (l_i + entropy)) + g_logprob [i = t] + sum_j g_top_j [i = top_j]
// (m and log S are kept for it apart: their sum, rounded at the size of the logits, would put that rounding on every p.)
// Sums and statistics are held in 32 bits; a 16-bit gradient is rounded once, when it is stored.
//
// Rows that no formula covers: every logit -inf -> logprob -inf, entropy 0, gradient 0 (but for the one-hot terms); a NaN or
// +inf anywhere -> NaN everywhere (a NaN counts as the largest logit among the alternatives).  target == ignore_index -> logprob 0
// and no gradient from it; any other target outside [0, C) -> NaN for both, and nothing is read there.
#include "ccn_common.h"

namespace {

constexpr int LP_TPB = 256;
constexpr int LP_TOP_MAX = 64;
constexpr float LP_LOG2E = 1.44269504088896340736f;

// e^d for d <= 0.  The product with log2(e) is off by at most |d| 2^-24 relative, which a weight of e^d turns into less than
// 2^-25 of the row's sum; results below 2^-126 are zero.
__device__ __forceinline__ float lp_exp(float d) { return __builtin_amdgcn_exp2f(d * LP_LOG2E); }

// Order of the alternatives as unsigned numbers: larger logit first, NaN above all, -0 equal to 0; then the lower class.
__device__ __forceinline__ uint64_t lp_key(float v, uint32_t c) {
  uint32_t b = __float_as_uint(v + 0.0f);
  if (v != v) b = 0x7f800001u;               // (right above infinity: no key is all ones)
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((uint64_t)b << 32) | (uint32_t)~c;
}
__device__ __forceinline__ float lp_key_value(uint64_t k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}
__device__ __forceinline__ int64_t lp_key_class(uint64_t k) { return (int64_t)(uint32_t)~(uint32_t)k; }

// The row's results from its statistics.
struct LpRow {
  float base, log_total, entropy;           // logprob of a logit v: (v - base) - log_total
};
__device__ __forceinline__ LpRow lp_finish(float m, float total, float weighted) {
  LpRow r;
  if (total == 0.f) {                       // every logit -inf
    r.base = 0.f;
    r.log_total = INFINITY;                 // (x - base) - log_total = -inf for every class
    r.entropy = 0.f;
  } else {
    r.base = m == -INFINITY ? 0.f : m;
    r.log_total = logf(total);
    r.entropy = r.log_total - weighted / total;
  }
  return r;
}

template <int T>
__global__ __launch_bounds__(LP_TPB) void logprob_fwd_kernel(const void* __restrict__ x, int64_t ld,
                                                             const int64_t* __restrict__ target, int C, int64_t ignore, int top,
                                                             float* __restrict__ logprob, float* __restrict__ entropy,
                                                             float2* __restrict__ stats, float* __restrict__ top_logprob,
                                                             int64_t* __restrict__ top_index) {
  __shared__ float red[2][LP_TPB / 64];
  __shared__ uint64_t kred[LP_TPB / 64];
  const int64_t row = blockIdx.x, at = row * ld;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  float m = -INFINITY;
  for (int c = threadIdx.x; c < C; c += LP_TPB) m = fmaxf(m, ld_el<T>(x, at + c));
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
  if (lane == 0) red[0][w] = m;
  __syncthreads();
  for (int k = 0; k < LP_TPB / 64; ++k) m = fmaxf(m, red[0][k]);
  __syncthreads();
  const float base = m == -INFINITY ? 0.f : m;
  float total = 0.f, weighted = 0.f;
  for (int c = threadIdx.x; c < C; c += LP_TPB) {
    const float d = ld_el<T>(x, at + c) - base, e = lp_exp(d);
    total += e;
    weighted += e > 0.f ? e * d : 0.f;
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    total += __shfl_xor(total, d, 64);
    weighted += __shfl_xor(weighted, d, 64);
  }
  if (lane == 0) {
    red[0][w] = total;
    red[1][w] = weighted;
  }
  __syncthreads();
  total = weighted = 0.f;
  for (int k = 0; k < LP_TPB / 64; ++k) {
    total += red[0][k];
    weighted += red[1][k];
  }
  const LpRow r = lp_finish(m, total, weighted);
  if (threadIdx.x == 0) {
    const int64_t t = target[row];
    float lp = 0.f;
    if (t != ignore) lp = t >= 0 && t < C ? (ld_el<T>(x, at + t) - r.base) - r.log_total : NAN;
    logprob[row] = lp;
    entropy[row] = r.entropy;
    if (stats) stats[row] = make_float2(r.base, r.log_total);
  }
  uint64_t last = ~(uint64_t)0;             // (above every key)
  for (int j = 0; j < top; ++j) {           // the largest key below the last one: keys are distinct
    uint64_t best = 0;
    for (int c = threadIdx.x; c < C; c += LP_TPB) {
      const uint64_t k = lp_key(ld_el<T>(x, at + c), (uint32_t)c);
      if (k < last && k > best) best = k;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      const uint64_t o = __shfl_xor((unsigned long long)best, d, 64);
      best = o > best ? o : best;
    }
    if (lane == 0) kred[w] = best;
    __syncthreads();
    for (int k = 0; k < LP_TPB / 64; ++k) best = kred[k] > best ? kred[k] : best;
    __syncthreads();
    if (threadIdx.x == 0) {
      top_logprob[row * top + j] = (lp_key_value(best) - r.base) - r.log_total;
      top_index[row * top + j] = lp_key_class(best);
    }
    last = best;
  }
}

template <int T>
__global__ __launch_bounds__(LP_TPB) void logprob_bwd_kernel(const void* __restrict__ x, int64_t ld,
                                                             const int64_t* __restrict__ target, int C, int64_t ignore, int top,
                                                             const int64_t* __restrict__ top_index, const float2* __restrict__ stats,
                                                             const float* __restrict__ entropy, const float* __restrict__ g_logprob,
                                                             int64_t g_logprob_stride, const float* __restrict__ g_entropy,
                                                             int64_t g_entropy_stride, const float* __restrict__ g_top,
                                                             void* __restrict__ dx, int64_t ldd) {
  const int64_t row = blockIdx.x, at = row * ld, to = row * ldd;
  const int64_t t = target[row];
  const bool scored = t != ignore, inside = t >= 0 && t < C;
  float g = 0.f;
  if (scored && g_logprob) g = inside ? g_logprob[row * g_logprob_stride] : NAN;
  float all = g;
  for (int j = 0; j < top; ++j) all += g_top[row * top + j];
  const float base = stats[row].x, log_total = stats[row].y, h = entropy[row], gh = g_entropy ? g_entropy[row * g_entropy_stride] : 0.f;
  for (int c = threadIdx.x; c < C; c += LP_TPB) {
    const float lp = (ld_el<T>(x, at + c) - base) - log_total, p = lp_exp(lp);
    float d = p == 0.f ? 0.f : -p * (all + gh * (lp + h));
    if (c == t && scored) d += g;
    for (int j = 0; j < top; ++j)
      if (top_index[row * top + j] == c) d += g_top[row * top + j];
    st_el<T>(dx, to + c, d);
  }
}

}  // namespace

extern "C" size_t ccn_logprob_workspace_bytes(int64_t rows, int64_t C, int top) {
  (void)rows; (void)C; (void)top;
  return 0;
}

extern "C" int ccn_logprob_fwd(const void* logits, int dtype, int64_t ld, const int64_t* target, int64_t rows, int64_t C,
                               int64_t ignore_index, int top, float* logprob, float* entropy, float* stats, float* top_logprob,
                               int64_t* top_index, void* ws, size_t ws_bytes, void* stream) {
  CCN_REQUIRE(logits && target && logprob && entropy, "logprob_fwd: null pointer");
  CCN_REQUIRE(dtype >= 0 && dtype <= 2, "logprob_fwd: dtype %d is not 0 (fp32), 1 (bf16) or 2 (fp16)", dtype);
  CCN_REQUIRE(rows > 0 && rows < ((int64_t)1 << 31) && C > 0 && C < ((int64_t)1 << 31) && (ld >= C || rows == 1),
              "logprob_fwd: rows=%lld C=%lld ld=%lld", (long long)rows, (long long)C, (long long)ld);
  CCN_REQUIRE(top >= 0 && top <= LP_TOP_MAX && top <= C, "logprob_fwd: top=%d (at most %d, and at most C)", top, LP_TOP_MAX);
  CCN_REQUIRE(top == 0 || (top_logprob && top_index), "logprob_fwd: top > 0 without its outputs");
  (void)ws; (void)ws_bytes;
  const dim3 grid((unsigned)rows), block(LP_TPB);
#define CCN_LP_FWD(T)                                                                                                             \
  hipLaunchKernelGGL(logprob_fwd_kernel<T>, grid, block, 0, (hipStream_t)stream, logits, ld, target, (int)C, ignore_index, top,    \
                     logprob, entropy, (float2*)stats, top_logprob, top_index)
  if (dtype == 0) CCN_LP_FWD(0);
  else if (dtype == 1) CCN_LP_FWD(1);
  else CCN_LP_FWD(2);
#undef CCN_LP_FWD
  CCN_LAUNCH_OK("logprob_fwd");
  return CCN_OK;
}

extern "C" int ccn_logprob_bwd(const void* logits, int dtype, int64_t ld, const int64_t* target, int64_t rows, int64_t C,
                               int64_t ignore_index, int top, const int64_t* top_index, const float* stats, const float* entropy,
                               const float* g_logprob, int64_t g_logprob_stride, const float* g_entropy, int64_t g_entropy_stride,
                               const float* g_top, void* dlogits, int64_t ldd, void* stream) {
  CCN_REQUIRE(logits && target && stats && entropy && dlogits, "logprob_bwd: null pointer");
  CCN_REQUIRE(dtype >= 0 && dtype <= 2, "logprob_bwd: dtype %d is not 0 (fp32), 1 (bf16) or 2 (fp16)", dtype);
  CCN_REQUIRE(rows > 0 && rows < ((int64_t)1 << 31) && C > 0 && C < ((int64_t)1 << 31) && (ld >= C || rows == 1) &&
              (ldd >= C || rows == 1), "logprob_bwd: rows=%lld C=%lld ld=%lld ldd=%lld", (long long)rows, (long long)C,
              (long long)ld, (long long)ldd);
  CCN_REQUIRE(top >= 0 && top <= LP_TOP_MAX && top <= C, "logprob_bwd: top=%d (at most %d, and at most C)", top, LP_TOP_MAX);
  CCN_REQUIRE(top == 0 || (g_top && top_index), "logprob_bwd: top > 0 without its gradient and classes");
  CCN_REQUIRE(g_logprob_stride >= 0 && g_entropy_stride >= 0, "logprob_bwd: negative gradient stride");
  const dim3 grid((unsigned)rows), block(LP_TPB);
#define CCN_LP_BWD(T)                                                                                                             \
  hipLaunchKernelGGL(logprob_bwd_kernel<T>, grid, block, 0, (hipStream_t)stream, logits, ld, target, (int)C, ignore_index, top,    \
                     top_index, (const float2*)stats, entropy, g_logprob, g_logprob_stride, g_entropy, g_entropy_stride, g_top, dlogits, ldd)
  if (dtype == 0) CCN_LP_BWD(0);
  else if (dtype == 1) CCN_LP_BWD(1);
  else CCN_LP_BWD(2);
#undef CCN_LP_BWD
  CCN_LAUNCH_OK("logprob_bwd");
  return CCN_OK;
}
