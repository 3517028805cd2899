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
#include <limits.h>

#include <type_traits>

#include "ccn_common.h"

namespace {

constexpr int LP_TPB = 256;
constexpr int LP_TOP_MAX = 64;

constexpr float LP_LOG2E = 1.44269504088896340736f;
constexpr float LP_FAR = -1000.f;           // differences below it weigh nothing; -inf, and -inf - -inf, become it

// e^d for LP_FAR <= d <= 0.  The product with log2(e) is off by at most |d| 2^-24 relative, which a weight of e^d turns into less
// than 2^-25 of the row's sum; results below 2^-126 are zero.
__device__ __forceinline__ float lp_exp(float d) { return __builtin_amdgcn_exp2f(d * LP_LOG2E); }
// v - base of a logit that may be -inf or NaN.  A NaN or +inf is not carried here: the row's maximum tells (lp_finish).
__device__ __forceinline__ float lp_diff(float v, float base) { return fmaxf(v - base, LP_FAR); }
// (of two values one of which is NaN: NaN)
__device__ __forceinline__ float lp_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

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
// The same order for the i-th 16-bit value of r, in 16 bits.
template <int T>
__device__ __forceinline__ uint32_t lp_key16(const ccn_u32x4& r, int i) {
  constexpr uint32_t INF = T == 1 ? 0x7f80 : 0x7c00;
  uint32_t h = (r[i >> 1] >> (16 * (i & 1))) & 0xffffu;
  if ((h & 0x7fffu) > INF) h = INF + 1;
  if (h == 0x8000u) h = 0;
  return h & 0x8000u ? h ^ 0xffffu : h | 0x8000u;
}
template <int T>
__device__ __forceinline__ float lp_key16_value(uint32_t k) {
  const uint32_t h = k & 0x8000u ? k & 0x7fffu : k ^ 0xffffu;
  return T == 1 ? __uint_as_float(h << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
__device__ __forceinline__ int64_t lp_key_class(uint64_t k) { return (int64_t)(uint32_t)~(uint32_t)k; }

// The row's results from its statistics.  m: the maximum, NaN where a logit is.
struct LpRow {
  float base, log_total, entropy;           // logprob of a logit v: (v - base) - log_total
};
__device__ __forceinline__ LpRow lp_finish(float m, float total, float weighted) {
  LpRow r;
  if (m == -INFINITY) {                     // every logit -inf
    r.base = 0.f;
    r.log_total = INFINITY;                 // (x - base) - log_total = -inf for every class
    r.entropy = 0.f;
  } else if (!(m < INFINITY)) {
    r.base = 0.f;
    r.log_total = r.entropy = NAN;
  } else {
    r.base = m;
    r.log_total = logf(total);
    r.entropy = r.log_total - weighted / total;
  }
  return r;
}

// -inf throughout, in 32 bits of the type
template <int T>
constexpr uint32_t LP_FILL = T == 0 ? 0xff800000u : T == 1 ? 0xff80ff80u : 0xfc00fc00u;

// 16 bytes of which only the first n values are the row's: the others are -inf and not read.
template <int T>
__device__ __forceinline__ ccn_u32x4 lp_load_part(const void* __restrict__ x, int64_t at, int n) {
  constexpr int V = CcnVec16<T>::N;
  ccn_u32x4 r = {LP_FILL<T>, LP_FILL<T>, LP_FILL<T>, LP_FILL<T>};
  if (n >= V) return ld16<T>(x, at);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n) {
      if (T == 0) {
        r[i] = reinterpret_cast<const uint32_t*>(x)[at + i];
      } else {
        const uint32_t v = reinterpret_cast<const uint16_t*>(x)[at + i];
        r[i >> 1] = (i & 1) ? ((r[i >> 1] & 0xffffu) | (v << 16)) : ((r[i >> 1] & 0xffff0000u) | v);
      }
    }
  return r;
}

// ---- sorted lists of 64 keys, one to a lane, descending

// One step of a bitonic sort: lanes D apart, in runs of SIZE of alternating direction (SIZE 64: descending throughout).
template <int SIZE, int D, typename K>
__device__ __forceinline__ K lp_step(K v) {
  const int lane = threadIdx.x & 63;
  const K o = ccn_lane_xor<D>(v);
  const bool larger = ((lane & SIZE) == 0) == ((lane & D) == 0);
  return (o > v) == larger ? o : v;
}
template <int SIZE, typename K>
__device__ __forceinline__ K lp_steps(K v) {
  if constexpr (SIZE >= 64) v = lp_step<SIZE, 32>(v);
  if constexpr (SIZE >= 32) v = lp_step<SIZE, 16>(v);
  if constexpr (SIZE >= 16) v = lp_step<SIZE, 8>(v);
  if constexpr (SIZE >= 8) v = lp_step<SIZE, 4>(v);
  if constexpr (SIZE >= 4) v = lp_step<SIZE, 2>(v);
  return lp_step<SIZE, 1>(v);
}
template <typename K>
__device__ __forceinline__ K lp_sort64(K v) {
  v = lp_steps<2>(v);
  v = lp_steps<4>(v);
  v = lp_steps<8>(v);
  v = lp_steps<16>(v);
  v = lp_steps<32>(v);
  return lp_steps<64>(v);
}
// The 64 largest of two lists: the larger of each pair (i, 63 - i) are they, and fall and rise; six steps put them in order.
__device__ __forceinline__ uint64_t lp_merge64(uint64_t a, uint64_t b) {
  const uint64_t o = __shfl((unsigned long long)b, 63 - (int)(threadIdx.x & 63), 64);
  return lp_steps<64>(a > o ? a : o);
}
// Lane k - 1 of the lane values in descending order (NaN first).
__device__ __forceinline__ uint32_t lp_kth_lane(uint32_t sorted, int k) { return (uint32_t)__builtin_amdgcn_readlane(sorted, k - 1); }

// ---- rows of more than 512 classes (or many alternatives of fewer): NW waves hold NW * 2048 logits of a row at a time in registers (32
// a thread), take their maximum, and add weights relative to the maximum so far: one pass over the row, one rescaling per 32 logits of a
// thread.  Bound by memory where rows are many (4000 x 65537 fp32 174 us, 6.0 TB/s; 4096 x 131072 bf16 225 us, 4.8), by the latency of its
// steps where they are few (1 x 50021 bf16 with 8 alternatives 7.6 us, and 3.1 to join the 7 parts).
//
// Alternatives: the threads' maxima give a lower bound of the top-th largest of the first logits held that few others reach
// (lp_limit).  Those that do wait in shared memory, and so do later ones that beat the bound, about `top` of 8192 random logits.  Wave 0
// puts them in order when another `top` would make them more than 64, and at the end; the last of the best is the new bound.
constexpr int LP_HOLD = 32;

template <int NW>
struct LpShared {
  static constexpr int ROOM = NW == 4 ? 1024 : 512;
  uint64_t cand[ROOM];                      // waiting
  uint64_t best[64];                        // in order, descending
  uint64_t last_key;                        // the top-th of them, 0 where there are fewer
  float last;
  int count[3];                             // those that came with this tile, the last one, the one before
  uint32_t limit[2][NW];
  float red[2][NW];
};

// (no alternatives, or the best class alone)
template <int NW>
struct LpSharedFew {
  uint64_t best[NW];
  float red[2][NW];
};

template <int NW>
__device__ __forceinline__ void lp_sync() {
  if (NW == 1) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}

// A value that at least `top` of the logits held reach, from the threads' maxima m: of every wave's 64 in order, the larger of the
// top-th of one wave and of the (top / NW)-th, the least over the waves.  (The least of the maxima of `top` or more groups of threads needs
// no order, but more logits reach it: 20000 x 1000 fp32 with 8 / 16 alternatives 33.4 / 39.1 us, in order 32.3 / 34.3.)
template <int NW>
__device__ __forceinline__ float lp_limit(float m, int top, LpShared<NW>& sh) {
  const int lane = threadIdx.x & 63, wave = NW == 4 ? threadIdx.x >> 6 : 0;
  uint32_t v = (uint32_t)(lp_key(m, 0) >> 32);
  v = lp_sort64(v);
  uint32_t bound = lp_kth_lane(v, top);
  if (NW > 1) {
    const uint32_t share = lp_kth_lane(v, (top + NW - 1) / NW);
    if (lane == 0) {
      sh.limit[0][wave] = bound;
      sh.limit[1][wave] = share;
    }
    lp_sync<NW>();
    bound = sh.limit[1][0];
#pragma unroll
    for (int k = 1; k < NW; ++k) bound = min(bound, sh.limit[1][k]);
#pragma unroll
    for (int k = 0; k < NW; ++k) bound = max(bound, sh.limit[0][k]);
  }
  return lp_key_value((uint64_t)bound << 32);
}

// Wave 0: the `got` that wait put among the `have` best.  64 in all: every key counts those above it, which is its place; more: sorted 64
// at a time and merged.
template <int NW>
__device__ __forceinline__ void lp_order(LpShared<NW>& sh, int top, int have, int got) {
  const int lane = threadIdx.x & 63;
  if (have + got <= 64) {
    const uint64_t k = lane < have ? sh.best[lane] : lane < have + got ? sh.cand[lane - have] : 0;
    int place = 0;
#pragma unroll 4
    for (int i = 0; i < have; ++i) place += sh.best[i] > k;
#pragma unroll 4
    for (int i = 0; i < got; ++i) place += sh.cand[i] > k;
    lp_sync<1>();
    if (lane < have + got && place < top) sh.best[place] = k;
  } else {
    uint64_t best = lane < have ? sh.best[lane] : 0;
    for (int b = 0; b < got; b += 64) best = lp_merge64(best, lp_sort64(b + lane < got ? sh.cand[b + lane] : 0));
    sh.best[lane] = best;
  }
  lp_sync<1>();
  if (lane == 0) {
    const uint64_t last = have + got >= top ? sh.best[top - 1] : 0;
    sh.last_key = last;
    sh.last = last ? lp_key_value(last) : -INFINITY;
  }
}

// The class of the e-th logit that a thread holds.
template <int T, int NT>
__device__ __forceinline__ int lp_class(int c0, int tid, int e) {
  constexpr int V = CcnVec16<T>::N;
  return c0 + ((e / V) * NT + tid) * V + e % V;
}

// TOP: 0 no alternatives, 1 the best class alone, 2 any number of them.  The best class needs no list: a wave looks for the class of its
// largest logit where a piece of the row holds a larger one than those before (20000 x 1000 bf16: 13.3 us without, 16.4 with the best class,
// 21.8 as a list of one; 600 x 20000 bf16 10.1, 12.2, 16.2).
template <int T, int NW, int TOP>
__global__ __launch_bounds__(LP_TPB, TOP < 2 ? 8 : NW == 1 || T == 0 ? 5 : 6) void logprob_wide_kernel(const void* __restrict__ x, int64_t ld,
                                                              const int64_t* __restrict__ target, int64_t rows, int C,
                                                              int64_t ignore, int top, int parts, int part_len,
                                                              float* __restrict__ logprob, float* __restrict__ entropy,
                                                              float2* __restrict__ stats, float* __restrict__ top_logprob,
                                                              int64_t* __restrict__ top_index, float4* __restrict__ part_stats,
                                                              uint64_t* __restrict__ part_keys) {
  constexpr int NT = NW * 64, V = CcnVec16<T>::N, NJ = LP_HOLD / V, TILE = NT * LP_HOLD;
  typedef std::conditional_t<TOP == 2, LpShared<NW>, LpSharedFew<NW>> Shared;
  __shared__ Shared shared[4 / NW];
  Shared& sh = shared[NW == 4 ? 0 : threadIdx.x >> 6];
  const int tid = NW == 4 ? threadIdx.x : threadIdx.x & 63, lane = threadIdx.x & 63, wave = NW == 4 ? threadIdx.x >> 6 : 0;
  const int64_t unit = NW == 4 ? blockIdx.x : (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t row = NW == 4 ? blockIdx.x / (unsigned)parts : unit;
  const int part = NW == 4 ? (int)(blockIdx.x % (unsigned)parts) : 0;
  if (NW == 1 && row >= rows) return;                // (a whole wave, and no barrier of the workgroup below)
  const int64_t at = row * ld;
  const int beg = part * part_len, end = min(C, beg + part_len);
  // the given class's logit, early: its latency passes beside the row
  const int64_t t = target[row];
  float given = 0.f;
  if (parts == 1 && t >= 0 && t < C) given = ld_el<T>(x, at + t);

  float m = -INFINITY, s = 0.f, w = 0.f;
  int turn = 0, have = 0, waiting = 0;               // (the same in every thread)
  float limit = -INFINITY;
  float first_value = -INFINITY;                     // (a row of -inf: its first class)
  uint32_t first_class = beg;
  if constexpr (TOP == 2) {
    if (tid < 3) sh.count[tid] = 0;
    lp_sync<NW>();
  }
  for (int c0 = beg; c0 < end; c0 += TILE) {
    const int n = end - c0;
    ccn_u32x4 raw[NJ];
    if (n >= TILE) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) raw[j] = ld16<T>(x, at + c0 + (j * NT + tid) * V);
    } else {
#pragma unroll
      for (int j = 0; j < NJ; ++j) raw[j] = lp_load_part<T>(x, at + c0 + (j * NT + tid) * V, n - (j * NT + tid) * V);
    }
    float tm = -INFINITY, vm[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      vm[j] = -INFINITY;
      if (j * NT * V < n) {
#pragma unroll
        for (int i = 0; i < V; i += 2) vm[j] = lp_max(lp_max(vm[j], get16<T>(raw[j], i)), get16<T>(raw[j], i + 1));
      }
      tm = lp_max(tm, vm[j]);
    }
    const float mn = lp_max(m, tm), dm = lp_diff(m, mn), f = lp_exp(dm);
    w = f * (w + dm * s);
    s *= f;
    m = mn;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      if (j * NT * V < n) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = lp_diff(get16<T>(raw[j], i), mn), e = lp_exp(d);
          s += e;
          w = __builtin_fmaf(e, d, w);
        }
      }
    if constexpr (TOP == 1) {
      const float of_wave = ccn_wave_join(tm, lp_max);
      if (!(of_wave <= first_value) && first_value == first_value) {
        uint32_t at = ~0u;
#pragma unroll
        for (int j = NJ - 1; j >= 0; --j)
          if (vm[j] == of_wave || vm[j] != vm[j]) {
#pragma unroll
            for (int i = V - 1; i >= 0; --i) {
              const float u = get16<T>(raw[j], i);
              if (u == of_wave || u != u) at = c0 + (j * NT + tid) * V + i;
            }
          }
        first_class = ccn_wave_join(at, [](uint32_t a, uint32_t b) { return min(a, b); });
        first_value = of_wave;
      }
    }
    if constexpr (TOP == 2) {
      const bool first = c0 == beg;
      if (first) limit = lp_limit<NW>(tm, top, sh);
      // the logits of this thread that are not below v, or that beat it (a NaN is and does, but for a v of NaN, which none beats)
      auto reach = [&](float v, bool beat) {
        uint32_t some = 0;
        if (beat && v != v) return some;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          if (beat ? !(vm[j] <= v) : !(vm[j] < v)) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float u = get16<T>(raw[j], i);
              if (beat ? !(u <= v) : !(u < v)) some |= 1u << (j * V + i);
            }
            const int left = n - (j * NT + tid) * V; // (of this row)
            if (left < V) some &= ~(~0u << (j * V + max(0, left)));
          }
        return some;
      };
      // (later ones have to beat the limit: an equal logit of a higher class comes behind)
      uint32_t pending = reach(limit, !first);
      const uint32_t all = pending;
      auto push = [&](uint32_t some) {               // (few: read again, from a cache, rather than picked out of registers)
        if (some) {
          const int want = __builtin_popcount(some), to = waiting + atomicAdd(&sh.count[turn], want);
          for (int k = to; k < min(to + want, LpShared<NW>::ROOM); ++k) {
            const int e = __builtin_ctz(some), c = lp_class<T, NT>(c0, tid, e);
            sh.cand[k] = lp_key(ld_el<T>(x, at + c), (uint32_t)c);
            some &= some - 1;
            pending &= ~(1u << e);
          }
        }
      };
      const bool flood = __builtin_amdgcn_ballot_w64(__builtin_popcount(pending) > LP_HOLD / 2) != 0;
      if (!flood) push(pending);
      else if (lane == 0) atomicAdd(&sh.count[turn], LpShared<NW>::ROOM + 1);
      lp_sync<NW>();
      const int came = sh.count[turn];
      if (waiting + came > LpShared<NW>::ROOM) {
        // equal logits or a rising row: over again, against what the logits held now promise by themselves; those of the first 64 classes
        // go first, which settles any number of equal ones; then as many at a time as there is room for
        // (one wave to a row has its logits at hand again in a cache, and no registers for two more looks at them)
        auto drop = [&](auto out) {
          for (uint32_t left = pending; left; left &= left - 1) {
            const int c = lp_class<T, NT>(c0, tid, __builtin_ctz(left));
            if (out(ld_el<T>(x, at + c), c)) pending &= ~(left & -left);
          }
        };
        pending = all;
        const float own = lp_limit<NW>(tm, top, sh);
        if (NW == 1) drop([&](float v, int) { return v < own; });
        else pending &= reach(own, false);
        for (bool opening = true;; opening = false) {
          if (tid == 0) sh.count[turn] = 0;          // (everyone has read it: a barrier ago)
          lp_sync<NW>();
          push(!opening ? pending : tid * V < 64 ? pending & ((1u << V) - 1) : 0);
          lp_sync<NW>();
          const int now = waiting + sh.count[turn], got = min(now, LpShared<NW>::ROOM);
          if (wave == 0) lp_order<NW>(sh, top, have, got);
          have = min(top, have + got);
          waiting = 0;
          lp_sync<NW>();
          limit = sh.last;
          if (!opening && now == got) break;
          if (NW > 1 && opening) pending &= reach(limit, true);
          else drop([&](float v, int c) { return lp_key(v, (uint32_t)c) < sh.last_key; });
        }
      } else {
        waiting += came;
        if (have + waiting + top > 64 && c0 + TILE < end) {
          if (wave == 0) lp_order<NW>(sh, top, have, waiting);
          have = min(top, have + waiting);
          waiting = 0;
          lp_sync<NW>();
          limit = sh.last;
        }
      }
      // (the count after next: read last before this tile's barrier, added to next behind the next one's)
      turn = turn == 2 ? 0 : turn + 1;
      if (tid == 0) sh.count[turn == 2 ? 0 : turn + 1] = 0;
    }
  }
  uint64_t best = 0;
  if constexpr (TOP == 2) {
    if (waiting && wave == 0) lp_order<NW>(sh, top, have, waiting);
    have = min(top, have + waiting);
  } else if (TOP == 1) {
    best = lp_key(first_value, first_class);
    if (NW > 1 && lane == 0) sh.best[wave] = best;
  }
  // the threads' statistics joined
  float all = m;
  all = ccn_wave_join(all, lp_max);
  if (NW > 1) {
    if (lane == 0) sh.red[0][wave] = all;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NW; ++k) all = lp_max(all, sh.red[0][k]);
    __syncthreads();
  }
  const float dm = lp_diff(m, all), f = lp_exp(dm);
  w = f * (w + dm * s);
  s *= f;
  s = ccn_wave_sum(s);
  w = ccn_wave_sum(w);
  if (NW > 1) {
    if (lane == 0) {
      sh.red[0][wave] = s;
      sh.red[1][wave] = w;
    }
    __syncthreads();
    s = w = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      s += sh.red[0][k];
      w += sh.red[1][k];
    }
  }
  if (wave != 0) return;
  if (TOP == 1 && NW > 1) {                          // (written two barriers ago)
#pragma unroll
    for (int k = 1; k < NW; ++k) best = best > sh.best[k] ? best : sh.best[k];
  }
  if (TOP == 2 && lane < have) best = sh.best[lane];
  if (parts > 1) {
    if (lane == 0) part_stats[unit] = make_float4(all, s, w, 0.f);
    if (TOP && lane < top) part_keys[unit * top + lane] = best;
    return;
  }
  const LpRow r = lp_finish(all, s, w);
  if (lane == 0) {
    logprob[row] = t == ignore ? 0.f : t >= 0 && t < C ? (given - r.base) - r.log_total : NAN;
    entropy[row] = r.entropy;
    if (stats) stats[row] = make_float2(r.base, r.log_total);
  }
  if (TOP && lane < top) {
    top_logprob[row * top + lane] = (lp_key_value(best) - r.base) - r.log_total;
    top_index[row * top + lane] = lp_key_class(best);
  }
}

// The parts of a row joined: four waves merge the lists of every fourth part each, wave 0 theirs.  All latency: 3.1 us for 7 parts of one
// row, 4.1 for 16 parts of 96 with 20 alternatives.
template <int T>
__global__ __launch_bounds__(LP_TPB) void logprob_join_kernel(const void* __restrict__ x, int64_t ld,
                                                              const int64_t* __restrict__ target, int C, int64_t ignore, int top,
                                                              int parts, const float4* __restrict__ part_stats,
                                                              const uint64_t* __restrict__ part_keys, float* __restrict__ logprob,
                                                              float* __restrict__ entropy, float2* __restrict__ stats,
                                                              float* __restrict__ top_logprob, int64_t* __restrict__ top_index) {
  __shared__ uint64_t lists[4][64];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // everything that is read, before anything waits: what depends on one another only
  const int64_t t = target[row];
  float4 q = make_float4(-INFINITY, 0.f, 0.f, 0.f);
  if (lane < parts) q = part_stats[row * parts + lane];
  uint64_t best = 0;
  if (top) {
    constexpr int U = 4;
    for (int p0 = wave; p0 < parts; p0 += 4 * U) {
      uint64_t k[U];
#pragma unroll
      for (int u = 0; u < U; ++u) k[u] = p0 + 4 * u < parts && lane < top ? part_keys[(row * parts + p0 + 4 * u) * top + lane] : 0;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (p0 + 4 * u < parts) best = p0 + 4 * u == wave ? k[u] : lp_merge64(best, k[u]);
    }
    lists[wave][lane] = best;
  }
  float given = 0.f;
  if (wave == 0 && t >= 0 && t < C) given = ld_el<T>(x, row * ld + t);
  if (top) {
    __syncthreads();
    if (wave < 2 && wave + 2 < parts) lists[wave][lane] = best = lp_merge64(best, lists[wave + 2][lane]);
    __syncthreads();
    if (wave == 0) best = lp_merge64(best, lists[1][lane]);
  }
  if (wave != 0) return;
  const float all = ccn_wave_join(q.x, lp_max);
  const float d = lp_diff(q.x, all), f = lp_exp(d);
  const float s = ccn_wave_sum(f * q.y), w = ccn_wave_sum(f * (q.z + d * q.y));
  const LpRow r = lp_finish(all, s, w);
  if (lane == 0) {
    logprob[row] = t == ignore ? 0.f : t >= 0 && t < C ? (given - r.base) - r.log_total : NAN;
    entropy[row] = r.entropy;
    if (stats) stats[row] = make_float2(r.base, r.log_total);
  }
  if (lane < top) {
    top_logprob[row * top + lane] = (lp_key_value(best) - r.base) - r.log_total;
    top_index[row * top + lane] = lp_key_class(best);
  }
}

// ---- the values of TEAM lanes next to one another, joined
template <int TEAM, typename V, typename F>
__device__ __forceinline__ V lp_team(V v, F f) {
  if constexpr (TEAM >= 2) v = f(v, ccn_lane_xor<1>(v));
  if constexpr (TEAM >= 4) v = f(v, ccn_lane_xor<2>(v));
  if constexpr (TEAM >= 8) v = f(v, ccn_lane_xor<4>(v));
  if constexpr (TEAM >= 16) v = f(v, ccn_lane_xor<8>(v));
  if constexpr (TEAM >= 32) v = f(v, ccn_lane_xor<16>(v));
  if constexpr (TEAM >= 64) v = f(v, ccn_lane_xor<32>(v));
  return v;
}

// ---- rows of 25 to 512 classes: TEAM lanes hold a row in registers, 16 logits each, and join their results by lane moves; a
// wave has 64 / TEAM rows.  Alternatives: `top` walks over the registers, each of which takes the largest logit that is left; TEAM of
// them are kept, a lane each, and stored side by side.  220011 x 55 fp32: 14.0 us, 3.8 TB/s, half of it the latency of one round of loads;
// with alternatives the walks' vector arithmetic bounds it (busy for 87 % of the time and more), each of them 1.2 us for 100000 x 50 fp32, 2.1 for
// 50000 x 256 fp32 and 1.1 in 16 bits.
template <int T, int TEAM, int TOP>
__global__ __launch_bounds__(LP_TPB) void logprob_team_kernel(const void* __restrict__ x, int64_t ld,
                                                              const int64_t* __restrict__ target, int64_t rows, int C,
                                                              int64_t ignore, int top, float* __restrict__ logprob,
                                                              float* __restrict__ entropy, float2* __restrict__ stats,
                                                              float* __restrict__ top_logprob, int64_t* __restrict__ top_index) {
  constexpr int V = CcnVec16<T>::N, HOLD = 16, NJ = HOLD / V;
  const int lane = threadIdx.x % TEAM;
  const int64_t mine = (int64_t)blockIdx.x * (LP_TPB / TEAM) + threadIdx.x / TEAM, row = min(mine, rows - 1);
  const bool live = mine < rows;                     // (every lane stays for the joins)
  ccn_u32x4 raw[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) raw[j] = lp_load_part<T>(x, row * ld + (j * TEAM + lane) * V, C - (j * TEAM + lane) * V);
  const int64_t t = target[row];
  const float given = t >= 0 && t < C ? ld_el<T>(x, row * ld + t) : 0.f;
  float m = -INFINITY, s = 0.f, w = 0.f;
#pragma unroll
  for (int j = 0; j < NJ; ++j)
    if (j * TEAM * V < C) {
#pragma unroll
      for (int i = 0; i < V; ++i) m = lp_max(m, get16<T>(raw[j], i));
    }
  m = lp_team<TEAM>(m, lp_max);
#pragma unroll
  for (int j = 0; j < NJ; ++j)
    if (j * TEAM * V < C) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = lp_diff(get16<T>(raw[j], i), m), e = lp_exp(d);
        s += e;
        w = __builtin_fmaf(e, d, w);
      }
    }
  s = lp_team<TEAM>(s, [](float a, float b) { return a + b; });
  w = lp_team<TEAM>(w, [](float a, float b) { return a + b; });
  const LpRow r = lp_finish(m, s, w);
  if (live && lane == 0) {
    logprob[row] = t == ignore ? 0.f : t >= 0 && t < C ? (given - r.base) - r.log_total : NAN;
    entropy[row] = r.entropy;
    if (stats) stats[row] = make_float2(r.base, r.log_total);
  }
  if (TOP == 0) return;
  if constexpr (TOP == 1) {                          // the lowest class of the largest logit (or of a NaN)
    int at = INT_MAX / 2;
#pragma unroll
    for (int j = NJ - 1; j >= 0; --j)
      if (j * TEAM * V < C) {
#pragma unroll
        for (int i = V - 1; i >= 0; --i) {
          const float v = get16<T>(raw[j], i);
          if (v == m || v != v) at = j * TEAM * V + i;
        }
      }
    const uint32_t c = lp_team<TEAM>((uint32_t)(at + lane * V), [](uint32_t x, uint32_t y) { return min(x, y); });
    if (live && lane == 0) {
      top_logprob[row] = (m - r.base) - r.log_total;
      top_index[row] = c;
    }
    return;
  }
  // the logits as whole numbers in the order of the alternatives; in 16 bits with the class below them, so that no two are equal
  uint32_t o[HOLD];
#pragma unroll
  for (int e = 0; e < HOLD; ++e) {
    const float v = get16<T>(raw[e / V], e % V);
    const int c = ((e / V) * TEAM + lane) * V + e % V;
    o[e] = c >= C ? 0 : T == 0 ? (uint32_t)(lp_key(v, 0) >> 32) : lp_key16<T>(raw[e / V], e % V) << 16 | (0xffffu - c);
  }
  uint32_t last = 0;
  float kept = 0.f;
  int kept_class = 0;
  for (int k = 0; k < top; ++k) {
    uint32_t best = 0;                               // (below every logit; taken ones become it)
    int c;
    float value;
    if constexpr (T == 0) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        if (j * TEAM * V < C) {
#pragma unroll
          for (int i = 0; i < V; ++i) best = max(best, o[j * V + i]);
        }
      best = lp_team<TEAM>(best, [](uint32_t x, uint32_t y) { return max(x, y); });
      int at = INT_MAX / 2;                          // the lowest class that has it
#pragma unroll
      for (int j = NJ - 1; j >= 0; --j)
        if (j * TEAM * V < C) {
#pragma unroll
          for (int i = V - 1; i >= 0; --i) at = o[j * V + i] == best ? j * TEAM * V + i : at;
        }
      c = (int)lp_team<TEAM>((uint32_t)(at + lane * V), [](uint32_t x, uint32_t y) { return min(x, y); });
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        if (j * TEAM * V < C) {
#pragma unroll
          for (int i = 0; i < V; ++i) o[j * V + i] = c - lane * V == j * TEAM * V + i ? 0 : o[j * V + i];
        }
      value = lp_key_value((uint64_t)best << 32);
    } else {
      // those below the last one wrap around when it is subtracted, and so are larger than those that are not: the largest difference is
      // the next one's
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        if (j * TEAM * V < C) {
#pragma unroll
          for (int i = 0; i < V; ++i) best = max(best, o[j * V + i] - last);
        }
      last += lp_team<TEAM>(best, [](uint32_t x, uint32_t y) { return max(x, y); });
      c = 0xffff - (int)(last & 0xffffu);
      value = lp_key16_value<T>(last >> 16);
    }
    if (k % TEAM == lane) {
      kept = (value - r.base) - r.log_total;
      kept_class = c;
    }
    if (k % TEAM == TEAM - 1 || k == top - 1) {
      const int from = k / TEAM * TEAM;
      if (live && from + lane <= k) {
        top_logprob[row * top + from + lane] = kept;
        top_index[row * top + from + lane] = kept_class;
      }
    }
  }
}

// ---- rows of up to 24 classes: 128 rows go through shared memory (16-byte loads) and a thread walks each of them there.  (Two threads to a
// row, or the registers of logprob_team_kernel, take 12.0 and 12.3 us for 400070 x 20 instead of 10.8.)  Bound by the latency from load to
// store of a workgroup's rows, its stores and, with alternatives, by vector arithmetic, which is busy for 71 % of the time (400000 x 20 fp32: 9.9 us,
// 3.9 TB/s; with 3 alternatives 15.1, 3.5).
// Up to LP_FEW_MAX alternatives come out of the two walks that the row takes anyway: the first keeps the K largest values in order, the second,
// from the last class to the first, notes where they are.  They leave through the row's own place in shared memory: a thread's own are K values
// wide, 64 such stores side by side cost more.  More of them: a walk for each, which takes the largest that is left (400000 x 20 fp32 with 3 / 5
// of them 16.1 / 22.3 us by walks and 15.1 / 18.3 so, x 12 12.4 / 16.6 and 12.2 / 14.1).
constexpr int LP_NARROW = 24;
constexpr int LP_NARROW_TPB = 128;

// TOP: 0 none, 1 the best class alone, LP_FEW + K: K of them, LP_WALK any number.
constexpr int LP_FEW = 100, LP_FEW_MAX = 5, LP_WALK = 2;
// A row's place in shared memory, which takes its few alternatives as well; odd, so that the lanes of a wave meet different banks.
__host__ __device__ inline int lp_pitch(int C, int few) { return (C > 2 * few ? C : 2 * few) | 1; }

template <int T, int TOP>
__global__ __launch_bounds__(LP_NARROW_TPB) void logprob_narrow_kernel(const void* __restrict__ x, int64_t ld,
                                                                       const int64_t* __restrict__ target, int64_t rows, int C,
                                                                       int vecs, uint32_t magic, int64_t ignore, int top,
                                                                       float* __restrict__ logprob, float* __restrict__ entropy,
                                                                       float2* __restrict__ stats,
                                                                       float* __restrict__ top_logprob,
                                                                       int64_t* __restrict__ top_index) {
  extern __shared__ float tile[];
  constexpr int V = CcnVec16<T>::N, ROWS = LP_NARROW_TPB, K = TOP > LP_FEW ? TOP - LP_FEW : 1;
  const int64_t r0 = (int64_t)blockIdx.x * ROWS;
  const int live = (int)min((int64_t)ROWS, rows - r0), pitch = lp_pitch(C, TOP > LP_FEW ? K : 0);
  // 16-byte pieces, `vecs` to a row (i / vecs as a product: exact for i < 2^16, the error of magic is below 2^-16)
  const int n = live * vecs;
  for (int i = threadIdx.x; i < n; i += LP_NARROW_TPB) {
    const int q = vecs == 1 ? i : (int)__umulhi((uint32_t)i, magic), c = (i - q * vecs) * V;
    const ccn_u32x4 raw = lp_load_part<T>(x, (r0 + q) * ld + c, C - c);
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (c + k < C) tile[q * pitch + c + k] = get16<T>(raw, k);
  }
  __syncthreads();
  float* const out = tile + ROWS * pitch;
  float* const out_class = out + ROWS * top;         // (classes and, below, keys: bits of whole numbers; this memory holds floats throughout)
  if ((int)threadIdx.x < live) {
    float* const mine = tile + threadIdx.x * pitch;
    const int64_t row = r0 + threadIdx.x, t = target[row];
    const float given = t >= 0 && t < C ? mine[t] : 0.f;
    // the K largest in order: a new one pushes those below it down by one
    float best[K];
#pragma unroll
    for (int k = 0; k < K; ++k) best[k] = -INFINITY;
#pragma unroll 4
    for (int c = 0; c < C; ++c) {
      const float v = mine[c];
#pragma unroll
      for (int k = K - 1; k > 0; --k) best[k] = __builtin_amdgcn_fmed3f(v, best[k - 1], best[k]);
      best[0] = lp_max(best[0], v);
    }
    const float m = best[0];
    float s = 0.f, w = 0.f;
    int at[K];                                       // their classes; from the last class to the first, equal ones by ascending class
#pragma unroll
    for (int k = 0; k < K; ++k) at[k] = 0;
#pragma unroll 4
    for (int c = C - 1; c >= 0; --c) {
      const float v = mine[c], d = lp_diff(v, m), e = lp_exp(d);
      s += e;
      w = __builtin_fmaf(e, d, w);
      if (TOP == 1) at[0] = v == m || v != v ? c : at[0];
      if (TOP > LP_FEW) {
#pragma unroll
        for (int k = K - 1; k > 0; --k) at[k] = v == best[k] ? (best[k] == best[k - 1] ? at[k - 1] : c) : at[k];
        at[0] = v == m ? c : at[0];
      }
    }
    const LpRow r = lp_finish(m, s, w);
    logprob[row] = t == ignore ? 0.f : t >= 0 && t < C ? (given - r.base) - r.log_total : NAN;
    entropy[row] = r.entropy;
    if (stats) stats[row] = make_float2(r.base, r.log_total);
    if (TOP == 1) {
      top_logprob[row] = (m - r.base) - r.log_total;
      top_index[row] = at[0];
    }
    // (the K largest are not found among NaN: the few waves that have any walk)
    if (TOP == LP_WALK || (TOP > LP_FEW && __builtin_amdgcn_ballot_w64(m != m) != 0)) {
#pragma unroll 4
      for (int c = 0; c < C; ++c) {                      // whole numbers in the order of the alternatives
        const float v = mine[c];
        int o = __float_as_int(v + 0.0f);
        if (v != v) o = 0x7f800001;
        mine[c] = __int_as_float(o ^ ((o >> 31) & 0x7fffffff));
      }
      auto walk = [&](float& value, int& c) {
        int v = INT_MIN;                             // (below every value; taken ones become it)
        c = 0;
#pragma unroll 4
        for (int i = 0; i < C; ++i) {
          const int o = __float_as_int(mine[i]);
          c = o > v ? i : c;
          v = max(v, o);
        }
        mine[c] = __int_as_float(INT_MIN);
        value = __int_as_float(v ^ ((v >> 31) & 0x7fffffff));
      };
      if constexpr (TOP == LP_WALK) {
        for (int j = 0; j < top; ++j) {
          float v;
          int c;
          walk(v, c);
          out[threadIdx.x * top + j] = (v - r.base) - r.log_total;
          out_class[threadIdx.x * top + j] = __int_as_float(c);
        }
      } else {
#pragma unroll
        for (int k = 0; k < K; ++k) walk(best[k], at[k]);
      }
    }
    if (TOP > LP_FEW) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        mine[k] = (best[k] - r.base) - r.log_total;  // (the row itself is not needed any more)
        mine[K + k] = __int_as_float(at[k]);
      }
    }
  }
  if (TOP < 2) return;
  __syncthreads();
  if constexpr (TOP > LP_FEW) {
    for (int i = threadIdx.x; i < live * K; i += LP_NARROW_TPB) {
      const float* const from = tile + i / K * pitch + i % K;
      top_logprob[r0 * K + i] = from[0];
      top_index[r0 * K + i] = __float_as_int(from[K]);
    }
  } else {
    for (int i = threadIdx.x; i < live * top; i += LP_NARROW_TPB) {
      top_logprob[r0 * top + i] = out[i];
      top_index[r0 * top + i] = __float_as_int(out_class[i]);
    }
  }
}

// ---- the gradient: dx = -p (G + g_entropy (l + entropy)) + one-hot terms, 16 bytes of a row at a time.  What belongs to the row alone:
struct LpGrad {
  float base, log_total, flat, slope;       // dx = p (flat + slope l)
  int t;                                    // the given class, -1 where it is not scored
  float g;
};
__device__ __forceinline__ LpGrad lp_grad(int64_t row, const int64_t* __restrict__ target, int C, int64_t ignore,
                                          const float2* __restrict__ stats, const float* __restrict__ entropy,
                                          const float* __restrict__ g_logprob, int64_t g_logprob_stride,
                                          const float* __restrict__ g_entropy, int64_t g_entropy_stride, float of_top) {
  LpGrad q;
  const int64_t t = target[row];
  const float2 st = stats[row];
  const float gh = g_entropy ? g_entropy[row * g_entropy_stride] : 0.f;
  q.t = -1;
  q.g = 0.f;
  if (t != ignore && g_logprob) {
    if (t >= 0 && t < C) q.t = (int)t;
    q.g = q.t >= 0 ? g_logprob[row * g_logprob_stride] : NAN;
  }
  const float all = q.g + of_top;           // (of_top: the sum of the row's g_top)
  q.base = st.x;
  q.log_total = st.y;
  q.slope = -gh;
  // (a row with a NaN or an infinity in it: NaN, though every p below is taken as 0)
  q.flat = st.y != st.y ? NAN : -(all + gh * entropy[row]);
  return q;
}
__device__ __forceinline__ float lp_smooth(const LpGrad& q, float v) {
  const float l = fmaxf((v - q.base) - q.log_total, LP_FAR);
  return lp_exp(l) * __builtin_fmaf(q.slope, l, q.flat);
}
template <int T>
__device__ __forceinline__ void lp_store_part(void* __restrict__ x, int64_t at, int n, const ccn_u32x4& r) {
  constexpr int V = CcnVec16<T>::N;
  if (n >= V) {
    st16<T>(x, at, r);
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n) {
      if (T == 0) reinterpret_cast<uint32_t*>(x)[at + i] = r[i];
      else reinterpret_cast<uint16_t*>(x)[at + i] = (uint16_t)(r[i >> 1] >> (16 * (i & 1)));
    }
}
// 16 bytes of the gradient from 16 bytes of the row, c the class of the first.
template <int T>
__device__ __forceinline__ ccn_u32x4 lp_grad16(const LpGrad& q, const ccn_u32x4& raw, int c) {
  constexpr int V = CcnVec16<T>::N;
  ccn_u32x4 out;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float d = lp_smooth(q, get16<T>(raw, i));
    if (c + i == q.t) d += q.g;
    put16<T>(out, i, d);
  }
  return out;
}
// The value of an alternative: written again, with its one-hot term (a row's alternatives are distinct).
template <int T>
__device__ __forceinline__ void lp_grad_top(const LpGrad& q, const void* __restrict__ x, int64_t at, void* __restrict__ dx,
                                            int64_t to, int64_t c, float g) {
  st_el<T>(dx, to + c, lp_smooth(q, ld_el<T>(x, at + c)) + (c == q.t ? q.g : 0.f) + g);
}

// A workgroup takes `group` rows of up to LP_GROUP_MAX classes, whose own values it computes once into shared memory; `vecs`: 16-byte
// pieces of a row.  220011 x 55 fp32: 21.3 us, 4.7 TB/s read and written.
constexpr int LP_GROUP = 4096;              // logits of a group of rows, about
constexpr int LP_GROUP_MAX = 4096;
constexpr int LP_GROUPS = 1024;             // groups, about, where rows are few (1500 x 20 fp32 with 20 alternatives: 14.8 us in 8 groups, 7.7)

template <int T>
__global__ __launch_bounds__(LP_TPB) void logprob_bwd_rows_kernel(
    const void* __restrict__ x, int64_t ld, const int64_t* __restrict__ target, int64_t rows, int C, int64_t ignore, int top, int group,
    int vecs, uint32_t magic, const int64_t* __restrict__ top_index, const float2* __restrict__ stats,
    const float* __restrict__ entropy, const float* __restrict__ g_logprob, int64_t g_logprob_stride,
    const float* __restrict__ g_entropy, int64_t g_entropy_stride, const float* __restrict__ g_top, void* __restrict__ dx, int64_t ldd) {
  constexpr int V = CcnVec16<T>::N;
  __shared__ LpGrad mine[LP_TPB];
  extern __shared__ float gt[];                      // the group's g_top
  const int64_t r0 = (int64_t)blockIdx.x * group;
  const int live = (int)min((int64_t)group, rows - r0), n = live * vecs;
  if (top) {
    for (int i = threadIdx.x; i < live * top; i += LP_TPB) gt[i] = g_top[r0 * top + i];
    __syncthreads();
  }
  if ((int)threadIdx.x < live) {
    float of_top = 0.f;
    for (int j = 0; j < top; ++j) of_top += gt[threadIdx.x * top + j];
    mine[threadIdx.x] = lp_grad(r0 + threadIdx.x, target, C, ignore, stats, entropy, g_logprob, g_logprob_stride, g_entropy,
                                g_entropy_stride, of_top);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += LP_TPB) {
    const int r = vecs == 1 ? i : (int)__umulhi((uint32_t)i, magic), c = (i - r * vecs) * V;
    const ccn_u32x4 raw = lp_load_part<T>(x, (r0 + r) * ld + c, C - c);
    lp_store_part<T>(dx, (r0 + r) * ldd + c, C - c, lp_grad16<T>(mine[r], raw, c));
  }
  if (top == 0) return;
  __syncthreads();
  for (int i = threadIdx.x; i < live * top; i += LP_TPB) {
    const int r = i / top;
    const int64_t row = r0 + r, c = top_index[r0 * top + i];
    if (c >= 0 && c < C) lp_grad_top<T>(mine[r], x, row * ld, dx, row * ldd, c, gt[i]);
  }
}

// Longer rows: a workgroup takes LP_TPB * LP_HOLD logits of one, all loads in flight before the first is used.  Memory bounds it: 4096 x
// 131072 bf16 386 us, 5.6 TB/s read and written.
template <int T>
__global__ __launch_bounds__(LP_TPB) void logprob_bwd_wide_kernel(
    const void* __restrict__ x, int64_t ld, const int64_t* __restrict__ target, int C, int64_t ignore, int top, int tiles,
    const int64_t* __restrict__ top_index, const float2* __restrict__ stats, const float* __restrict__ entropy,
    const float* __restrict__ g_logprob, int64_t g_logprob_stride, const float* __restrict__ g_entropy, int64_t g_entropy_stride,
    const float* __restrict__ g_top, void* __restrict__ dx, int64_t ldd) {
  constexpr int V = CcnVec16<T>::N, NJ = LP_HOLD / V, TILE = LP_TPB * LP_HOLD;
  const int64_t row = blockIdx.x / (unsigned)tiles, at = row * ld, to = row * ldd;
  const int c0 = (int)(blockIdx.x % (unsigned)tiles) * TILE, n = min(C - c0, TILE), tid = threadIdx.x;
  ccn_u32x4 raw[NJ];
  if (n == TILE) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) raw[j] = ld16<T>(x, at + c0 + (j * LP_TPB + tid) * V);
  } else {
#pragma unroll
    for (int j = 0; j < NJ; ++j) raw[j] = lp_load_part<T>(x, at + c0 + (j * LP_TPB + tid) * V, n - (j * LP_TPB + tid) * V);
  }
  float of_top = 0.f;
  for (int j = 0; j < top; ++j) of_top += g_top[row * top + j];
  const LpGrad q = lp_grad(row, target, C, ignore, stats, entropy, g_logprob, g_logprob_stride, g_entropy, g_entropy_stride, of_top);
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int c = (j * LP_TPB + tid) * V;
    if (j * LP_TPB * V < n) lp_store_part<T>(dx, to + c0 + c, n - c, lp_grad16<T>(q, raw[j], c0 + c));
  }
  if (top == 0) return;
  __syncthreads();
  if (tid < top) {
    const int64_t c = top_index[row * top + tid];
    if (c >= c0 && c < c0 + n) lp_grad_top<T>(q, x, at, dx, to, c, g_top[row * top + tid]);
  }
}

// Whether the row is logprob_narrow_kernel's.  Its walks wait for shared memory: where rows are few the team's registers are faster from three
// alternatives on (us, narrow / team, 1500 x 20 with 3 / 10 / 20 of them: fp32 7.7 / 6.7, 12.0 / 9.3, 17.6 / 12.3, bf16 8.6 / 6.4, 13.1 / 7.5,
// 19.0 / 8.9), and where they are many in 16 bits with many alternatives (400000 x 20 with 5 / 10: bf16 19.1 / 24.2, 35 / 30, fp32 18.3 / 29, 33 / 42).
bool lp_is_narrow(int64_t rows, int64_t C, int top, bool wide_type) {
  if (C > LP_NARROW) return false;
  if (C < 12 || top < 3) return true;
  return rows > 65536 && (wide_type || C < 20 || top < 8);
}

// Lanes to a row of logprob_team_kernel, 0 where the row is logprob_wide_kernel's: that one's way to the alternatives costs the same for
// many of them, and a walk here costs less in 16 bits (us, 50000 rows, here / there: 500 bf16 with 12 of them 44 / 57, with 20 58 / 60; 256 fp16
// with 32 44 / 66; 500 fp32 with 8 53 / 58, with 12 70 / 61; 256 fp32 with 20 55 / 61).
int lp_team_of(int64_t C, int top, bool wide_type) {
  if (C <= 64) return 4;
  if (C <= 128) return 8;
  if (C > 512 || C * top > (wide_type ? 5120 : 10240)) return 0;
  return C <= 256 ? 16 : 32;
}

// Waves to a row of logprob_wide_kernel.  One is enough up to 2048 classes; where rows are many it goes on longer alone, since four spend more
// on joining what they found (us, four / one, 20000 rows of 2050: bf16 with 0 / 5 alternatives 40 / 23, 86 / 38, fp32 40 / 29, 98 / 43; of 4100: 48 /
// 34, 96 / 55, fp32 52 / 56, 117 / 70; of 8192: 55 / 60, 125 / 93, fp32 107 / 118, 131 / 124; 4000 rows of 2050 bf16 with 5 22 / 13, of 8192 26.5 /
// 25.2; 1000 of 2050 11.1 / 10.8, of 4100 11.3 / 13.1).
int lp_waves(int64_t rows, int64_t C, int top, bool wide_type) {
  if (C <= 64 * LP_HOLD) return 1;
  if (rows < (C <= 4096 ? 2048 : 4096)) return 4;
  return (top > 1 ? C <= 8192 : C * (wide_type ? 4 : 2) <= 12000) ? 1 : 4;
}

// How rows are cut into parts of about one length, a workgroup each, where there are too few rows to fill the card: 512 x 131072 bf16
// with 8 alternatives takes 58 us in one part to a row and 45 in three, 512 x 50000 31 and 27, but 1000 x 50000 38 and 44 in two (each
// part orders its own); without alternatives 256 x 50000 12.2 and 13.0, 512 x 20000 fp32 11.3 and 13.6 (the joining launch).  Parts of less
// than a piece cost more than they gain (96 x 131072 fp16 with 20: 23.9, with parts of half that 34.6).  Rows of a few pieces stay
// whole, since the joining launch costs more than the workgroup's next turns (us, in parts / whole, 1 or 30 rows of bf16: 32000 classes 9.2 / 7.6,
// 20000 and the best class 9.1 / 8.0, of 32000 9.4 / 9.4, 12000 with 5 alternatives 12.4 / 12.1, 20000 12.8 / 14.4); with alternatives also those of
// 600 rows and up to 32768 classes (24000 with 5 19.6 / 18.4, of 300 14.5 / 16.2).
// Parts of one piece where a quarter more workgroups than fit at once do that; else as many as fit, and no more than take as many pieces each
// (bf16 with 5: 266 x 51831 in 4 / 5 / 6 / 7 parts 18.8 / 19.8 / 22.5 / 20.1 us, 180 x 131072 in 7 / 8 / 9 23.5 / 21.5 / 25.8, 100 x 131072 in 15 / 16
// 19.6 / 18.2; fp32, of which fewer fit, 400 x 51831 in 3 / 4 25.2 / 26.6).
constexpr int64_t LP_FULL = 256, LP_FULL_TOP = 768, LP_FULL_SHORT = 512, LP_PIECE = LP_TPB * LP_HOLD, LP_PARTS_MAX = 64;
int64_t lp_pieces(int64_t C) { return (C + LP_PIECE - 1) / LP_PIECE; }
struct LpPlan {
  int nw, parts, part_len;
};
LpPlan lp_plan(int64_t rows, int64_t C, int top, bool wide_type) {
  LpPlan p = {lp_waves(rows, C, top, wide_type), 1, (int)C};
  if (p.nw == 1 || C <= LP_PIECE * (top > 1 ? 2 : top ? 3 : 4)) return p;
  if (rows >= (top <= 1 ? LP_FULL : C <= 4 * LP_PIECE ? LP_FULL_SHORT : LP_FULL_TOP)) return p;
  const int64_t fit = 256 * (top <= 1 ? 8 : wide_type ? 5 : 6);       // (the launch bounds of logprob_wide_kernel)
  int64_t parts = lp_pieces(C);
  if (rows * parts > fit + fit / 4) parts = fit / rows < 1 ? 1 : fit / rows;
  if (parts > LP_PARTS_MAX) parts = LP_PARTS_MAX;
  parts = (lp_pieces(C) + lp_pieces((C + parts - 1) / parts) - 1) / lp_pieces((C + parts - 1) / parts);
  p.part_len = (int)(((C + parts - 1) / parts + 7) / 8 * 8);
  p.parts = (int)((C + p.part_len - 1) / p.part_len);
  return p;
}

// A launch holds fewer than 2^32 threads: rows go in pieces (a workgroup of the widest takes one).
constexpr int64_t LP_LAUNCH_ROWS = (int64_t)1 << 22;
const void* lp_row(const void* x, int dtype, int64_t at) { return (const char*)x + at * (dtype == 0 ? 4 : 2); }

// The launches of one piece of the rows (p: of all of them).
int lp_fwd(const void* logits, int dtype, int64_t ld, const int64_t* target, int64_t rows, int64_t C, int64_t ignore_index, int top,
           const LpPlan& p, float* logprob, float* entropy, float* stats, float* top_logprob, int64_t* top_index, void* ws,
           hipStream_t s) {
  if (lp_is_narrow(rows, C, top, dtype == 0)) {
    const int per = dtype == 0 ? 4 : 8, vecs = (int)((C + per - 1) / per);
    const uint32_t magic = vecs == 1 ? 0 : (uint32_t)((((uint64_t)1 << 32) + vecs - 1) / vecs);
    const dim3 grid((unsigned)((rows + LP_NARROW_TPB - 1) / LP_NARROW_TPB)), block(LP_NARROW_TPB);
    const size_t lds = (size_t)LP_NARROW_TPB * (lp_pitch((int)C, top > 1 && top <= LP_FEW_MAX ? top : 0) + (top > LP_FEW_MAX ? 2 * top : 0)) * sizeof(float);
#define CCN_LP_NARROW(T, TOP)                                                                                                     \
  hipLaunchKernelGGL((logprob_narrow_kernel<T, TOP>), grid, block, lds, s, logits, ld, target, rows, (int)C, vecs, magic,          \
                     ignore_index, top, logprob, entropy, (float2*)stats, top_logprob, top_index)
#define CCN_LP_NARROWS(T)                                 \
  do {                                                    \
    if (top == 0) CCN_LP_NARROW(T, 0);                    \
    else if (top == 1) CCN_LP_NARROW(T, 1);               \
    else if (top == 2) CCN_LP_NARROW(T, LP_FEW + 2);      \
    else if (top == 3) CCN_LP_NARROW(T, LP_FEW + 3);      \
    else if (top == 4) CCN_LP_NARROW(T, LP_FEW + 4);      \
    else if (top == 5) CCN_LP_NARROW(T, LP_FEW + 5);      \
    else CCN_LP_NARROW(T, LP_WALK);                       \
  } while (0)
    static_assert(LP_FEW_MAX == 5, "the launches below");
    if (dtype == 0) CCN_LP_NARROWS(0);
    else if (dtype == 1) CCN_LP_NARROWS(1);
    else CCN_LP_NARROWS(2);
#undef CCN_LP_NARROWS
#undef CCN_LP_NARROW
    CCN_LAUNCH_OK("logprob_fwd");
    return CCN_OK;
  }
  if (const int team = lp_team_of(C, top, dtype == 0)) {
#define CCN_LP_TEAM_TOP(T, TEAM, TOP)                                                                                             \
  hipLaunchKernelGGL((logprob_team_kernel<T, TEAM, TOP>), grid, block, 0, s, logits, ld, target, rows, (int)C, ignore_index, top, \
                     logprob, entropy, (float2*)stats, top_logprob, top_index)
#define CCN_LP_TEAM(T, TEAM)                                                                                                      \
  do {                                                                                                                            \
    const dim3 grid((unsigned)((rows + LP_TPB / TEAM - 1) / (LP_TPB / TEAM))), block(LP_TPB);                                     \
    if (top > 1) CCN_LP_TEAM_TOP(T, TEAM, 2);                                                                                     \
    else if (top) CCN_LP_TEAM_TOP(T, TEAM, 1);                                                                                    \
    else CCN_LP_TEAM_TOP(T, TEAM, 0);                                                                                             \
  } while (0)
#define CCN_LP_TEAMS(T)                                                                                                           \
  do {                                                                                                                            \
    if (team == 4) CCN_LP_TEAM(T, 4);                                                                                    \
    else if (team == 8) CCN_LP_TEAM(T, 8);                                                                                    \
    else if (team == 16) CCN_LP_TEAM(T, 16);                                                                                  \
    else CCN_LP_TEAM(T, 32);                                                                                                  \
  } while (0)
    if (dtype == 0) CCN_LP_TEAMS(0);
    else if (dtype == 1) CCN_LP_TEAMS(1);
    else CCN_LP_TEAMS(2);
#undef CCN_LP_TEAMS
#undef CCN_LP_TEAM
#undef CCN_LP_TEAM_TOP
    CCN_LAUNCH_OK("logprob_fwd");
    return CCN_OK;
  }
  float4* const part_stats = (float4*)ws;
  uint64_t* const part_keys = ws ? (uint64_t*)((char*)ws + ccn_align256((size_t)rows * p.parts * sizeof(float4))) : nullptr;
  const int64_t blocks = p.nw == 1 ? (rows + 3) / 4 : rows * p.parts;
#define CCN_LP_WIDE(T, NW, TOP)                                                                                                   \
  hipLaunchKernelGGL((logprob_wide_kernel<T, NW, TOP>), dim3((unsigned)blocks), dim3(LP_TPB), 0, s, logits, ld, target, rows,      \
                     (int)C, ignore_index, top, p.parts, p.part_len, logprob, entropy, (float2*)stats, top_logprob, top_index,   \
                     part_stats, part_keys)
#define CCN_LP_FWD(T)                                                                                                             \
  do {                                                                                                                            \
    if (p.nw == 1 && top > 1) CCN_LP_WIDE(T, 1, 2);                                                                               \
    else if (p.nw == 1 && top) CCN_LP_WIDE(T, 1, 1);                                                                              \
    else if (p.nw == 1) CCN_LP_WIDE(T, 1, 0);                                                                                     \
    else if (top > 1) CCN_LP_WIDE(T, 4, 2);                                                                                       \
    else if (top) CCN_LP_WIDE(T, 4, 1);                                                                                           \
    else CCN_LP_WIDE(T, 4, 0);                                                                                                    \
    if (p.parts > 1)                                                                                                              \
      hipLaunchKernelGGL(logprob_join_kernel<T>, dim3((unsigned)rows), dim3(LP_TPB), 0, s, logits, ld, target, (int)C,             \
                         ignore_index, top, p.parts, part_stats, part_keys, logprob, entropy, (float2*)stats, top_logprob,        \
                         top_index);                                                                                              \
  } while (0)
  if (dtype == 0) CCN_LP_FWD(0);
  else if (dtype == 1) CCN_LP_FWD(1);
  else CCN_LP_FWD(2);
#undef CCN_LP_FWD
#undef CCN_LP_WIDE
  CCN_LAUNCH_OK("logprob_fwd");
  return CCN_OK;
}

int lp_bwd(const void* logits, int dtype, int64_t ld, const int64_t* target, int64_t rows, int64_t C, int64_t ignore_index, int top,
           const int64_t* top_index, const float* stats, const float* entropy, const float* g_logprob, int64_t g_logprob_stride,
           const float* g_entropy, int64_t g_entropy_stride, const float* g_top, void* dlogits, int64_t ldd, hipStream_t s) {
  if (C <= LP_GROUP_MAX) {
    const int per = dtype == 0 ? 4 : 8, vecs = (int)((C + per - 1) / per);
    const int64_t share = rows / LP_GROUPS, most = LP_GROUP / C > LP_TPB ? LP_TPB : LP_GROUP / C;
    const int group = (int)(share < 1 || most < 1 ? 1 : share < most ? share : most);
    const uint32_t magic = vecs == 1 ? 0 : (uint32_t)((((uint64_t)1 << 32) + vecs - 1) / vecs);
    const dim3 grid((unsigned)((rows + group - 1) / group)), block(LP_TPB);
#define CCN_LP_BWD(T)                                                                                                             \
  hipLaunchKernelGGL(logprob_bwd_rows_kernel<T>, grid, block, (size_t)group * top * sizeof(float), s, logits, ld, target, rows,   \
                     (int)C, ignore_index, top, group, vecs, magic, top_index, (const float2*)stats, entropy, g_logprob,          \
                     g_logprob_stride, g_entropy, g_entropy_stride, g_top, dlogits, ldd)
    if (dtype == 0) CCN_LP_BWD(0);
    else if (dtype == 1) CCN_LP_BWD(1);
    else CCN_LP_BWD(2);
#undef CCN_LP_BWD
  } else {
    const int64_t tiles = lp_pieces(C);
    const dim3 grid((unsigned)(rows * tiles)), block(LP_TPB);
#define CCN_LP_BWD(T)                                                                                                             \
  hipLaunchKernelGGL(logprob_bwd_wide_kernel<T>, grid, block, 0, s, logits, ld, target, (int)C, ignore_index, top, (int)tiles,     \
                     top_index, (const float2*)stats, entropy, g_logprob, g_logprob_stride, g_entropy, g_entropy_stride, g_top,   \
                     dlogits, ldd)
    if (dtype == 0) CCN_LP_BWD(0);
    else if (dtype == 1) CCN_LP_BWD(1);
    else CCN_LP_BWD(2);
#undef CCN_LP_BWD
  }
  CCN_LAUNCH_OK("logprob_bwd");
  return CCN_OK;
}

}  // namespace

extern "C" size_t ccn_logprob_workspace_bytes(int64_t rows, int64_t C, int top) {
  if (rows <= 0 || C <= LP_NARROW || top < 0) return 0;
  const int a = lp_plan(rows, C, top, false).parts, b = lp_plan(rows, C, top, true).parts, parts = a > b ? a : b;      // (for any type)
  if (parts == 1) return 0;
  return ccn_align256((size_t)rows * parts * sizeof(float4)) + ccn_align256((size_t)rows * parts * top * sizeof(uint64_t));
}

extern "C" int ccn_logprob_fwd(const void* logits, int dtype, int64_t ld, const int64_t* target, int64_t rows, int64_t C,
                               int64_t ignore_index, int top, float* logprob, float* entropy, float* stats, float* top_logprob,
                               int64_t* top_index, void* ws, size_t ws_bytes, void* stream) {
  CCN_REQUIRE(logits && target && logprob && entropy, "logprob_fwd: null pointer");
  CCN_REQUIRE((uintptr_t)stats % 8 == 0, "logprob_fwd: stats are not 8-byte aligned");
  CCN_REQUIRE(dtype >= 0 && dtype <= 2, "logprob_fwd: dtype %d is not 0 (fp32), 1 (bf16) or 2 (fp16)", dtype);
  CCN_REQUIRE(rows > 0 && rows < ((int64_t)1 << 31) && C > 0 && C < ((int64_t)1 << 30) && (ld >= C || rows == 1),
              "logprob_fwd: rows=%lld C=%lld ld=%lld", (long long)rows, (long long)C, (long long)ld);
  CCN_REQUIRE(top >= 0 && top <= LP_TOP_MAX && top <= C, "logprob_fwd: top=%d (at most %d, and at most C)", top, LP_TOP_MAX);
  CCN_REQUIRE(top == 0 || (top_logprob && top_index), "logprob_fwd: top > 0 without its outputs");
  const LpPlan p = lp_plan(rows, C, top, dtype == 0);
  const size_t need = ccn_logprob_workspace_bytes(rows, C, top);
  if (need && (ws == nullptr || (uintptr_t)ws % 16 || ws_bytes < need)) {
    ccn_set_error("logprob_fwd: workspace of %zu bytes, %zu are needed (16-byte aligned)", ws ? ws_bytes : (size_t)0, need);
    return CCN_ERR_WORKSPACE;
  }
  for (int64_t r = 0; r < rows; r += LP_LAUNCH_ROWS) {
    const int rc = lp_fwd(lp_row(logits, dtype, r * ld), dtype, ld, target + r, rows - r < LP_LAUNCH_ROWS ? rows - r : LP_LAUNCH_ROWS, C,
                          ignore_index, top, p, logprob + r, entropy + r, stats ? stats + 2 * r : nullptr,
                          top ? top_logprob + r * top : nullptr, top ? top_index + r * top : nullptr, need ? ws : nullptr,
                          (hipStream_t)stream);
    if (rc) return rc;
  }
  return CCN_OK;
}

extern "C" int ccn_logprob_bwd(const void* logits, int dtype, int64_t ld, const int64_t* target, int64_t rows, int64_t C,
                               int64_t ignore_index, int top, const int64_t* top_index, const float* stats, const float* entropy,
                               const float* g_logprob, int64_t g_logprob_stride, const float* g_entropy, int64_t g_entropy_stride,
                               const float* g_top, void* dlogits, int64_t ldd, void* stream) {
  CCN_REQUIRE(logits && target && stats && entropy && dlogits, "logprob_bwd: null pointer");
  CCN_REQUIRE((uintptr_t)stats % 8 == 0, "logprob_bwd: stats are not 8-byte aligned");
  CCN_REQUIRE(dtype >= 0 && dtype <= 2, "logprob_bwd: dtype %d is not 0 (fp32), 1 (bf16) or 2 (fp16)", dtype);
  CCN_REQUIRE(rows > 0 && rows < ((int64_t)1 << 31) && C > 0 && C < ((int64_t)1 << 30) && (ld >= C || rows == 1) &&
              (ldd >= C || rows == 1), "logprob_bwd: rows=%lld C=%lld ld=%lld ldd=%lld", (long long)rows, (long long)C,
              (long long)ld, (long long)ldd);
  CCN_REQUIRE(top >= 0 && top <= LP_TOP_MAX && top <= C, "logprob_bwd: top=%d (at most %d, and at most C)", top, LP_TOP_MAX);
  CCN_REQUIRE(top == 0 || (g_top && top_index), "logprob_bwd: top > 0 without its gradient and classes");
  CCN_REQUIRE(g_logprob_stride >= 0 && g_entropy_stride >= 0, "logprob_bwd: negative gradient stride");
  const int64_t most = C <= LP_GROUP_MAX ? LP_LAUNCH_ROWS : (LP_LAUNCH_ROWS + lp_pieces(C) - 1) / lp_pieces(C);
  for (int64_t r = 0; r < rows; r += most) {
    const int rc = lp_bwd(lp_row(logits, dtype, r * ld), dtype, ld, target + r, rows - r < most ? rows - r : most, C, ignore_index, top,
                          top ? top_index + r * top : nullptr, stats + 2 * r, entropy + r,
                          g_logprob ? g_logprob + r * g_logprob_stride : nullptr, g_logprob_stride,
                          g_entropy ? g_entropy + r * g_entropy_stride : nullptr, g_entropy_stride, top ? g_top + r * top : nullptr,
                          const_cast<void*>(lp_row(dlogits, dtype, r * ldd)), ldd, (hipStream_t)stream);
    if (rc) return rc;
  }
  return CCN_OK;
}
