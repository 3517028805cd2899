// Shared helpers for libccn_hip.so (gfx950 only).
#pragma once
#include <hip/hip_runtime.h>

#include <atomic>
#include <stdint.h>
#include <stddef.h>

#include "../../include/ccn_hip.h"
#include "../../include/ccn_hip_debug.h"   // (included so that a drift between a hook's prototype and its definition is a compile error)

// ---- error reporting (never throws; negative return + ccn_last_error()) ----
void ccn_set_error(const char* fmt, ...);

#define CCN_REQUIRE(cond, ...)          \
  do {                                  \
    if (!(cond)) {                      \
      ccn_set_error(__VA_ARGS__);       \
      return CCN_ERR_ARG;               \
    }                                   \
  } while (0)

#define CCN_LAUNCH_OK(name)                                               \
  do {                                                                    \
    hipError_t e__ = hipGetLastError();                                   \
    if (e__ != hipSuccess) {                                              \
      ccn_set_error("%s: launch failed: %s", name, hipGetErrorString(e__)); \
      return CCN_ERR_LAUNCH;                                              \
    }                                                                     \
  } while (0)

#define CCN_HIP(call, name)                                             \
  do {                                                                  \
    hipError_t e__ = (call);                                            \
    if (e__ != hipSuccess) {                                            \
      ccn_set_error("%s: %s", name, hipGetErrorString(e__));            \
      return CCN_ERR_LAUNCH;                                            \
    }                                                                   \
  } while (0)

// ---- workspace carving: 256-byte aligned bump allocator over a caller-owned buffer ----
struct CcnArena {
  char* base;
  size_t cap;
  size_t used;
  __host__ CcnArena(void* p, size_t n) : base((char*)p), cap(n), used(0) {}
  template <typename T>
  __host__ T* take(size_t count) {
    size_t bytes = (count * sizeof(T) + 255) & ~(size_t)255;
    if (base == nullptr || used + bytes > cap) {
      used = cap + 1;  // poison
      return nullptr;
    }
    T* r = (T*)(base + used);
    used += bytes;
    return r;
  }
  __host__ bool ok() const { return used <= cap; }
};
static inline size_t ccn_align256(size_t b) { return (b + 255) & ~(size_t)255; }

static inline int ccn_blocks(int64_t n, int per_block) { return (int)((n + per_block - 1) / per_block); }

// Per-device one-time setup (function attributes are per device): `slot` = a zero-initialised static array of CCN_MAX_DEVICES
// atomics; returns the current device's entry, nullptr when the device cannot be named.  A race between two threads only repeats
// an idempotent call.  (Round 6: the `static bool` latches of rounds 3-5 were per process.)
constexpr int CCN_MAX_DEVICES = 64;
static inline std::atomic<int>* ccn_device_slot(std::atomic<int>* slots) {
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= CCN_MAX_DEVICES) return nullptr;
  return slots + dev;
}

// ---- device-wide scans (ccn_scan.hip) ----
// exclusive/inclusive prefix sums over n elements; `scratch` needs ccn_scan_scratch_bytes(n) bytes.
size_t ccn_scan_scratch_bytes(int64_t n);
int ccn_scan_i32(const int32_t* in, int32_t* out, int64_t n, bool inclusive, int32_t* total_out, void* scratch,
                 hipStream_t s);
int ccn_scan_f64(const double* in, double* out, int64_t n, bool inclusive, void* scratch, hipStream_t s);

// ---- stable LSD radix sort with payload (ccn_sort.hip) ----
// n non-negative int64 keys sorted on the 8-bit digits named by digit_mask (bit b = digit b); *vout = the original positions
// in sorted order, equal keys in ascending position (it points into `ws`, ccn_rank_keys_workspace_bytes(n) bytes).
int ccn_sort_payload(const int64_t* key, int64_t n, int digit_mask, void* ws, size_t ws_bytes, hipStream_t s,
                     const int32_t** vout);

// exact distance arithmetic shared by every index kernel and by oracle/frnn_bruteforce.c
// XCD-aware work order for one-dimensional grids of row-gathering kernels (round 5).  Workgroup ids are dealt round-robin over
// the eight XCDs (ids b and b + 8 share an XCD and its 4 MiB L2 -- observed placement, used for speed only: any placement
// gives the same result): with the work taken in id order, eight consecutive pieces -- 32 neighbouring points whose
// neighbour lists overlap almost completely -- go to eight different L2s and every gathered row is fetched eight times.
// ccn_xcd_block() renumbers the ids so that the workgroups with id % 8 == x take ONE contiguous eighth of the work: the
// workgroups in flight on an XCD then sit next to each other in the point order and share their gathered rows in its L2.
// A bijection of [0, gridDim.x) for any grid size.  -DCCN_XCD_ORDER=0 builds the id-order form (A/B).
#ifndef CCN_XCD_ORDER
#define CCN_XCD_ORDER 1
#endif
__device__ __forceinline__ unsigned ccn_xcd_block() {
#if CCN_XCD_ORDER
  const unsigned n = gridDim.x, b = blockIdx.x, x = b & 7u, k = b >> 3, per = n >> 3, rem = n & 7u;
  return x * per + (x < rem ? x : rem) + k;
#else
  return blockIdx.x;
#endif
}

__device__ __forceinline__ float ccn_sqdist3(float dx, float dy, float dz) {
  return __builtin_fmaf(dz, dz, __builtin_fmaf(dy, dy, dx * dx));
}

// ---- 16-bit rows at the MLP boundary of the 16-bit storage modes (ccn_gemm_h.hip): the first-layer edge kernels (ccn_edge.hip) and the shifted-row matrix (ccn_curve.hip) can write
// their activation as bf16 / fp16 rows (ZT) and read the gradient of such an activation as bf16 rows (DZ16) -- the fp32 round
// trip through ccn_cast_rows_h is 8 bytes per element of an E x C tensor.  T: 0 = fp32, 1 = bf16, 2 = fp16.
template <int T>
__device__ __forceinline__ float ld_el(const void* __restrict__ p, int64_t i) {
  if (T == 0) return reinterpret_cast<const float*>(p)[i];
  const uint16_t v = reinterpret_cast<const uint16_t*>(p)[i];
  if (T == 2) return (float)__builtin_bit_cast(_Float16, v);
  return __builtin_bit_cast(float, (uint32_t)v << 16);
}
template <int T>
__device__ __forceinline__ void st_el(void* __restrict__ p, int64_t i, float v) {
  if (T == 0) {
    reinterpret_cast<float*>(p)[i] = v;
  } else if (T == 2) {
    const _Float16 x = (_Float16)v;
    reinterpret_cast<uint16_t*>(p)[i] = __builtin_bit_cast(uint16_t, x);
  } else {
    const __bf16 x = (__bf16)v;        // round to nearest even (the rounding of ccn_cast_rows_h)
    reinterpret_cast<uint16_t*>(p)[i] = __builtin_bit_cast(uint16_t, x);
  }
}

// ---- 16 bytes of fp32 / bf16 / fp16 values (T as above) at any alignment of the type
typedef uint32_t ccn_u32x4 __attribute__((ext_vector_type(4)));
template <int T> struct CcnVec16 {
  static constexpr int N = 8;
  typedef ccn_u32x4 mem __attribute__((aligned(2)));
};
template <> struct CcnVec16<0> {
  static constexpr int N = 4;
  typedef ccn_u32x4 mem __attribute__((aligned(4)));
};
template <int T>
__device__ __forceinline__ float get16(const ccn_u32x4& r, int i) {
  if (T == 0) return __builtin_bit_cast(float, (uint32_t)r[i]);
  if (T == 1) return __builtin_bit_cast(float, (uint32_t)((i & 1) ? (r[i >> 1] & 0xffff0000u) : (r[i >> 1] << 16)));
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(r[i >> 1] >> (16 * (i & 1))));
}
// (values are put in ascending order: an even one clears its neighbour)
template <int T>
__device__ __forceinline__ void put16(ccn_u32x4& r, int i, float v) {
  if (T == 0) {
    r[i] = __builtin_bit_cast(uint32_t, v);
  } else {
    uint32_t b;
    if (T == 1) b = __builtin_bit_cast(uint16_t, (__bf16)v);
    else b = __builtin_bit_cast(uint16_t, (_Float16)v);
    r[i >> 1] = (i & 1) ? (r[i >> 1] | (b << 16)) : b;
  }
}
template <int T>
__device__ __forceinline__ ccn_u32x4 ld16(const void* p, int64_t i) {
  return *reinterpret_cast<const typename CcnVec16<T>::mem*>(reinterpret_cast<const char*>(p) + i * (T == 0 ? 4 : 2));
}
template <int T>
__device__ __forceinline__ void st16(void* p, int64_t i, const ccn_u32x4& r) {
  *reinterpret_cast<typename CcnVec16<T>::mem*>(reinterpret_cast<char*>(p) + i * (T == 0 ? 4 : 2)) = r;
}

// ---- the value of lane (lane ^ D), by data-parallel moves instead of the LDS crossbar (4 to 16 cycles instead of about 100); every lane
// of the wave has to be active
template <int D>
__device__ __forceinline__ uint32_t ccn_lane_xor(uint32_t v) {
  static_assert(D == 1 || D == 2 || D == 4 || D == 8 || D == 16 || D == 32, "a power of two below 64");
  if constexpr (D == 1) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true);         // quad_perm [1,0,3,2]
  else if constexpr (D == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true);    // quad_perm [2,3,0,1]
  else if constexpr (D == 4)                                                                    // ^ 7 by row_half_mirror, then ^ 3
    return __builtin_amdgcn_update_dpp(0, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true), 0x1B, 0xf, 0xf, true);
  else if constexpr (D == 8) return __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, true);   // row_ror:8
  else if constexpr (D == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return (threadIdx.x & 16) ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (threadIdx.x & 32) ? r[0] : r[1];
  }
}
template <int D>
__device__ __forceinline__ float ccn_lane_xor(float v) {
  return __builtin_bit_cast(float, ccn_lane_xor<D>(__builtin_bit_cast(uint32_t, v)));
}
template <int D>
__device__ __forceinline__ uint64_t ccn_lane_xor(uint64_t v) {
  return ((uint64_t)ccn_lane_xor<D>((uint32_t)(v >> 32)) << 32) | ccn_lane_xor<D>((uint32_t)v);
}
template <int D>
__device__ __forceinline__ double ccn_lane_xor(double v) {
  return __builtin_bit_cast(double, ccn_lane_xor<D>(__builtin_bit_cast(uint64_t, v)));
}
// v of all 64 lanes joined by f, in the same order in every lane's tree
template <typename V, typename F>
__device__ __forceinline__ V ccn_wave_join(V v, F f) {
  v = f(v, ccn_lane_xor<1>(v));
  v = f(v, ccn_lane_xor<2>(v));
  v = f(v, ccn_lane_xor<4>(v));
  v = f(v, ccn_lane_xor<8>(v));
  v = f(v, ccn_lane_xor<16>(v));
  return f(v, ccn_lane_xor<32>(v));
}
template <typename V>
__device__ __forceinline__ V ccn_wave_sum(V v) {
  return ccn_wave_join(v, [](V a, V b) { return a + b; });
}
