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
// three-operand XORs.
struct Drop {
  unsigned key[20];
  u64 offset, base;
  unsigned last;   // words <= last are dropped
  float factor;    // 1 / (1 - p); 0 for p = 1
  int on;          // 0: no element is dropped
};

// p is in [0, 1].
inline Drop make_drop(double p, u64 seed, u64 offset, u64 base) {
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
  return d;
}

__device__ __forceinline__ void philox4(const Drop& d, u64 q, unsigned w[4]) {
  unsigned c0 = (unsigned)q, c1 = (unsigned)(q >> 32), c2 = (unsigned)d.offset, c3 = (unsigned)(d.offset >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const u64 a = (u64)0xD2511F53u * c0, b = (u64)0xCD9E8D57u * c2;
    c0 = (unsigned)(b >> 32) ^ c1 ^ d.key[2 * i];
    c1 = (unsigned)b;
    c2 = (unsigned)(a >> 32) ^ c3 ^ d.key[2 * i + 1];
    c3 = (unsigned)a;
  }
  w[0] = c0;
  w[1] = c1;
  w[2] = c2;
  w[3] = c3;
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
