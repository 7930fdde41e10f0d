// Shared by the operators of residual blocks with experts (nn_dropout.cu,
// nn_norm.cu, nn_grouped.cu): element types, the counter-based generator,
// argument checks and launch helpers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <exception>
#include <string>
#include <type_traits>

#include "../../include/ccb.h"

namespace ccb {
void set_error(const std::string& msg);  // the library's thread-local message (runtime.cpp)
}

namespace ccb_nn {

typedef unsigned long long u64;
typedef long long i64;

// ------------------------------------------------------------- host helpers
inline int fail(int code, const char* entry, const std::string& m) {
  ccb::set_error(std::string(entry) + ": " + m);
  return code;
}
inline int launched(const char* entry) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? CCB_OK : fail(CCB_ERR_DRIVER, entry, std::string("launch: ") + cudaGetErrorString(e));
}
inline bool float_type(int d) { return d == CCB_F32 || d == CCB_BF16 || d == CCB_F16; }
inline int type_bytes(int d) { return d == CCB_F32 ? 4 : 2; }
inline bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
// rows x cols x stride stays inside the 63-bit byte range
inline bool sane(i64 rows, i64 cols, i64 stride) {
  return rows >= 0 && cols >= 0 && rows < (1ll << 40) && cols < (1ll << 40) && stride >= 0 && stride < (1ll << 40) &&
         (rows <= 1 || stride == 0 || rows < (1ll << 58) / (stride + 1));
}
// SMs of the current device (a fixed property of the device).
inline int sm_count(const char* entry, int* sms) {
  static int known[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return fail(CCB_ERR_NO_DEVICE, entry, std::string("cudaGetDevice: ") + cudaGetErrorString(e));
  int n = dev >= 0 && dev < 64 ? __atomic_load_n(&known[dev], __ATOMIC_RELAXED) : 0;
  if (n == 0) {
    e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess || n < 1)
      return fail(CCB_ERR_DRIVER, entry, std::string("cudaDeviceGetAttribute: ") + cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) __atomic_store_n(&known[dev], n, __ATOMIC_RELAXED);
  }
  *sms = n;
  return CCB_OK;
}

// No C++ exception leaves a C entry point.
#define CCB_NN_GUARD(entry, ...)                                         \
  try {                                                                  \
    __VA_ARGS__                                                          \
  } catch (const std::exception& ex) {                                   \
    return ccb_nn::fail(CCB_ERR_DRIVER, entry, ex.what());               \
  } catch (...) {                                                        \
    return ccb_nn::fail(CCB_ERR_DRIVER, entry, "unknown C++ exception"); \
  }

// ------------------------------------------------------------ element types
// Arithmetic is in F32; a result is rounded to its storage type once, to
// nearest even, when it is stored.
template <class T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }

template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// Two results in one 32-bit word of a 16-bit type.
template <class T>
__device__ __forceinline__ unsigned pack2(float lo, float hi) {
  unsigned r;
  if constexpr (std::is_same<T, __half>::value)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Element i of a vector whose type is known at run time (weights, biases).
__device__ __forceinline__ float load_as(const void* p, int dtype, i64 i) {
  if (dtype == CCB_F32) return static_cast<const float*>(p)[i];
  if (dtype == CCB_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// ---------------------------------------------------------------- dropout
// Element e of a tensor is word e % 4 of Philox-4x32-10 (Salmon, Moraes, Dror,
// Shaw 2011; the generator of Rng) at the counter (q lo, q hi, offset lo,
// offset hi), q = e / 4, under the 64-bit key `seed`: one block of ten rounds
// serves four elements. It is dropped when its word is below
// round(p * 2^32). The ten round keys depend on the seed alone and are laid
// out by the host, so a round is two 32x32 -> 64 products and two
// three-operand XORs. The products bound the generator (one of them takes the
// multiplier for four cycles a warp): where all of a tensor's counters share
// q's high word, the second product of round one and the first of round two
// are constants, so the host computes them and 18 products are left of 20.
struct Drop {
  unsigned key[20];
  u64 offset, base;
  unsigned last;   // words <= last are dropped
  float factor;    // 1 / (1 - p); 0 for p = 1
  int on;          // 0: no element is dropped
  int same;        // one high word for all: round two's constants hold
  unsigned c2, c0, hi, c3;
};

// p is in [0, 1]; n elements from `base` on.
inline Drop make_drop(double p, u64 seed, u64 offset, u64 base, u64 n) {
  Drop d = {};
  unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
  for (int i = 0; i < 10; ++i) {
    d.key[2 * i] = k0;
    d.key[2 * i + 1] = k1;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  d.offset = offset;
  d.base = base;
  const double t = std::nearbyint(p * 4294967296.0);
  d.on = t >= 1.0;
  d.last = d.on ? (unsigned)(u64)(t - 1.0) : 0u;
  d.factor = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
  // the last block that a vector of 8 touches lies up to 11 elements on
  const u64 end = base + n + 11 < base ? ~0ull : base + n + 11;
  d.same = (base >> 34) == (end >> 34);
  const u64 b = (u64)0xCD9E8D57u * (unsigned)offset;
  const unsigned r1c0 = (unsigned)(b >> 32) ^ (unsigned)(base >> 34) ^ d.key[0];
  const u64 a = (u64)0xD2511F53u * r1c0;
  d.c2 = (unsigned)(offset >> 32) ^ d.key[1];
  d.c0 = (unsigned)b ^ d.key[2];
  d.hi = (unsigned)(a >> 32) ^ d.key[3];
  d.c3 = (unsigned)a;
  return d;
}

__device__ __forceinline__ void philox_round(const Drop& d, int i, unsigned& c0, unsigned& c1, unsigned& c2, unsigned& c3) {
  const u64 a = (u64)0xD2511F53u * c0, b = (u64)0xCD9E8D57u * c2;
  c0 = (unsigned)(b >> 32) ^ c1 ^ d.key[2 * i];
  c1 = (unsigned)b;
  c2 = (unsigned)(a >> 32) ^ c3 ^ d.key[2 * i + 1];
  c3 = (unsigned)a;
}
// N blocks from q on, round by round: their products do not wait for one another.
// SAME: d.same is known to hold.
template <int N, bool SAME>
__device__ __forceinline__ void philox(const Drop& d, u64 q, unsigned* w) {
  unsigned c[N][4];
  if (SAME || d.same) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const u64 a = (u64)0xD2511F53u * (unsigned)(q + n);
      const u64 b = (u64)0xCD9E8D57u * ((unsigned)(a >> 32) ^ d.c2);
      c[n][0] = (unsigned)(b >> 32) ^ d.c0;
      c[n][1] = (unsigned)b;
      c[n][2] = (unsigned)a ^ d.hi;
      c[n][3] = d.c3;
    }
  } else {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      c[n][0] = (unsigned)(q + n);
      c[n][1] = (unsigned)((q + n) >> 32);
      c[n][2] = (unsigned)d.offset;
      c[n][3] = (unsigned)(d.offset >> 32);
      philox_round(d, 0, c[n][0], c[n][1], c[n][2], c[n][3]);
      philox_round(d, 1, c[n][0], c[n][1], c[n][2], c[n][3]);
    }
  }
#pragma unroll
  for (int i = 2; i < 10; ++i)
#pragma unroll
    for (int n = 0; n < N; ++n) philox_round(d, i, c[n][0], c[n][1], c[n][2], c[n][3]);
#pragma unroll
  for (int i = 0; i < 4 * N; ++i) w[i] = c[i >> 2][i & 3];
}
__device__ __forceinline__ void philox4(const Drop& d, u64 q, unsigned* w) { philox<1, false>(d, q, w); }
// The words of the 8 elements from e0 on, d.same: two blocks, or three where
// the index is no multiple of 4.
__device__ __forceinline__ void philox8(const Drop& d, u64 e0, unsigned* w) {
  const u64 q = e0 >> 2;
  philox<2, true>(d, q, w);
  const int shift = (int)(e0 & 3);
  if (shift) {
    unsigned x[4];
    philox<1, true>(d, q + 2, x);
    for (int k = 0; k < shift; ++k) {
#pragma unroll
      for (int i = 0; i < 7; ++i) w[i] = w[i + 1];
      w[7] = x[0];
      x[0] = x[1], x[1] = x[2], x[2] = x[3];
    }
  }
}
// v / (1 - p), or 0 (whatever v holds) where the word says so.
__device__ __forceinline__ float dropped(const Drop& d, unsigned word, float v) { return word > d.last ? v * d.factor : 0.0f; }
// The same for one element by its index, at a whole block's cost.
__device__ __forceinline__ float dropped_at(const Drop& d, u64 e, float v) {
  if (!d.on) return v * d.factor;
  unsigned w[4];
  philox4(d, e >> 2, w);
  const unsigned j = (unsigned)e & 3u;
  return dropped(d, j == 0 ? w[0] : j == 1 ? w[1] : j == 2 ? w[2] : w[3], v);
}

}  // namespace ccb_nn
