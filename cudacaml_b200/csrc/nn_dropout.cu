// ccb_nn_dropout: out = residual + keep(e) * x / (1 - p), the mask a pure
// function of (seed, offset, element index) that is never stored; the
// gradient is the same call on dy without the residual.
//
// Bytes: x and the residual read once, out written once.
#include "nn_common.cuh"

namespace ccb_nn {
namespace {

struct DropoutP {
  const void* x;
  const void* res;
  void* out;
  i64 rows, cols, xs, rs, os;
  Drop d;
};

// Element i of 8, in one 16-byte word or two.
template <class T>
__device__ __forceinline__ float element(const uint4* u, int i) {
  const uint4 q = u[sizeof(T) == 4 ? i >> 2 : 0];
  const int j = sizeof(T) == 4 ? i & 3 : i >> 1;
  const unsigned w = j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w;
  if constexpr (sizeof(T) == 4)
    return __uint_as_float(w);
  else if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
  else
    return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w >> 16 : w)));
}

// Any alignment, stride and base: a thread takes one block of the generator,
// the up to four elements of the tensor that lie in it, by single loads and
// stores (16384 x 4096 bf16 with a residual: 119 us, against 78 by pieces of 8).
template <class T>
__global__ void __launch_bounds__(256) dropout_any(const __grid_constant__ DropoutP p) {
  const u64 n = (u64)p.rows * (u64)p.cols;
  const u64 q0 = p.d.base >> 2, q1 = (p.d.base + n - 1) >> 2;
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.res);
  T* out = static_cast<T*>(p.out);
  const u64 step = (u64)gridDim.x * blockDim.x;
  for (u64 q = q0 + (u64)blockIdx.x * blockDim.x + threadIdx.x; q <= q1; q += step) {
    unsigned w[4] = {};
    if (p.d.on) philox4(p.d, q, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u64 e = 4 * q + j;
      if (e < p.d.base || e - p.d.base >= n) continue;
      const i64 i = (i64)(e - p.d.base);
      const i64 r = p.rows == 1 ? 0 : i / p.cols, c = i - r * p.cols;
      const float v = to_f<T>(x[r * p.xs + c]);
      float y = p.d.on ? dropped(p.d, w[j], v) : v * p.d.factor;
      if (res) y += to_f<T>(res[r * p.rs + c]);
      out[r * p.os + c] = from_f<T>(y);
    }
  }
}

// 8 consecutive elements of a row by 16-byte accesses: pointers and strides of
// 16 bytes, and rows of whole pieces of 8 (dense rows are one long row, whose
// last elements the first threads take). The generator takes half as long as
// the memory, so they have to overlap: a thread has 32 bytes (64 with a
// residual) on their way whatever the type, two pieces of a 16-bit one (with one
// alone 16384 x 4096 of them took 1 us more).
// 16384 x 4096 bf16 with a residual takes 80 us (5.0 TB/s), without 74 (3.6
// TB/s): no unit is saturated (the generator's products and the ALU at half their
// rates); some 21 KB an SM on their way are too few for the memory's latency.
// 8192 x 4096 f32 with a residual takes 62 us (6.5 TB/s, HBM).
template <class T>
__global__ void __launch_bounds__(256) dropout_wide(const __grid_constant__ DropoutP p, unsigned pieces, u64 total) {
  constexpr int kWords = sizeof(T) / 2, kOnce = 4 / (int)sizeof(T);  // 16-byte words of a piece, pieces at once
  const u64 step = (u64)gridDim.x * blockDim.x, first = (u64)blockIdx.x * blockDim.x + threadIdx.x;
  for (u64 v0 = first; v0 < total; v0 += kOnce * step) {
    uint4 a[kOnce][kWords], b[kOnce][kWords];
    u64 row[kOnce], col[kOnce];
#pragma unroll
    for (int k = 0; k < kOnce; ++k) {
      const u64 v = v0 + k * step;
      row[k] = 0;
      col[k] = v;
      if (p.rows > 1) {  // total is below 2^32
        row[k] = (unsigned)v / pieces;
        col[k] = (unsigned)v - (unsigned)row[k] * pieces;
      }
      col[k] *= 8;
      if (v >= total) continue;
      const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + row[k] * p.xs + col[k]);
      const uint4* res = reinterpret_cast<const uint4*>(static_cast<const T*>(p.res) + row[k] * p.rs + col[k]);
#pragma unroll
      for (int i = 0; i < kWords; ++i) a[k][i] = x[i];
      if (p.res)
#pragma unroll
        for (int i = 0; i < kWords; ++i) b[k][i] = res[i];
    }
#pragma unroll
    for (int k = 0; k < kOnce; ++k) {
      if (v0 + k * step >= total) break;
      unsigned w[8];
      if (p.d.on) philox8(p.d, p.d.base + row[k] * (u64)p.cols + col[k], w);
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = element<T>(a[k], i) * p.d.factor;
        if (p.d.on && w[i] <= p.d.last) y[i] = 0.0f;
        if (p.res) y[i] += element<T>(b[k], i);
      }
      uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + row[k] * p.os + col[k]);
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if constexpr (sizeof(T) == 4)
          out[i] = make_uint4(__float_as_uint(y[4 * i]), __float_as_uint(y[4 * i + 1]), __float_as_uint(y[4 * i + 2]), __float_as_uint(y[4 * i + 3]));
        else
          out[i] = make_uint4(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7]));
      }
    }
  }
  if (p.rows == 1) {
    const u64 e = (u64)p.cols / 8 * 8 + first;
    if (e < (u64)p.cols) {
      float y = dropped_at(p.d, p.d.base + e, to_f<T>(static_cast<const T*>(p.x)[e]));
      if (p.res) y += to_f<T>(static_cast<const T*>(p.res)[e]);
      static_cast<T*>(p.out)[e] = from_f<T>(y);
    }
  }
}

template <class T>
void go(const DropoutP& p, int sms, cudaStream_t st) {
  const u64 n = (u64)p.rows * (u64)p.cols;
  const bool lines = p.rows == 1 || (p.cols % 8 == 0 && p.xs % 8 == 0 && p.os % 8 == 0 && (!p.res || p.rs % 8 == 0) && n / 8 < (1ull << 32));
  if (lines && (p.d.same || !p.d.on) && aligned(p.x, 16) && aligned(p.out, 16) && aligned(p.res, 16)) {
    const u64 total = n / 8, want = total / 256 + 1, most = (u64)sms * 16;
    dropout_wide<T><<<(unsigned)(want < most ? want : most), 256, 0, st>>>(p, (unsigned)(p.cols / 8), total);
    return;
  }
  const u64 blocks = n / 4 + 2;
  const u64 want = (blocks + 255) / 256, most = (u64)sms * 32;
  dropout_any<T><<<(unsigned)(want < most ? want : most), 256, 0, st>>>(p);
}

}  // namespace
}  // namespace ccb_nn

using namespace ccb_nn;

extern "C" int ccb_nn_dropout(const ccb_nn_dropout_t* a, void* stream) {
  static const char* const me = "ccb_nn_dropout";
  CCB_NN_GUARD(me, {
    if (!a) return fail(CCB_ERR_INVALID, me, "null argument block");
    if (!float_type(a->dtype)) return fail(CCB_ERR_INVALID, me, "dtype code " + std::to_string(a->dtype) + " (0 f32, 4 bf16, 5 f16)");
    if (!(a->p >= 0.0 && a->p <= 1.0)) return fail(CCB_ERR_INVALID, me, "p = " + std::to_string(a->p) + " is outside [0, 1]");
    if (!sane(a->rows, a->cols, a->x_stride) || !sane(a->rows, a->cols, a->out_stride) ||
        (a->residual && !sane(a->rows, a->cols, a->residual_stride)) || (a->cols > 0 && a->rows > (1ll << 60) / a->cols))
      return fail(CCB_ERR_INVALID, me, "rows, cols or a stride is out of range");
    if (a->rows > 1 && (a->x_stride < a->cols || a->out_stride < a->cols || (a->residual && a->residual_stride < a->cols)))
      return fail(CCB_ERR_INVALID, me, "a row stride is shorter than a row");
    const i64 n = a->rows * a->cols;
    if (n == 0) return CCB_OK;
    if (a->base > ~0ull - (u64)n) return fail(CCB_ERR_INVALID, me, "base + rows * cols passes 2^64");
    if (!a->x || !a->out) return fail(CCB_ERR_INVALID, me, "null pointer");
    const int b = type_bytes(a->dtype);
    if (!aligned(a->x, b) || !aligned(a->out, b) || !aligned(a->residual, b))
      return fail(CCB_ERR_INVALID, me, "a pointer is not aligned to its element type");
    int sms = 0;
    if (const int rc = sm_count(me, &sms)) return rc;
    DropoutP p = {a->x, a->residual, a->out, a->rows, a->cols, a->x_stride, a->residual_stride, a->out_stride,
                  make_drop(a->p, a->seed, a->offset, a->base, (u64)n)};
    // dense rows are one long row
    if (p.rows > 1 && p.xs == p.cols && p.os == p.cols && (!p.res || p.rs == p.cols)) {
      p.cols = n;
      p.rows = 1;
    }
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->dtype == CCB_F32)
      go<float>(p, sms, st);
    else if (a->dtype == CCB_BF16)
      go<__nv_bfloat16>(p, sms, st);
    else
      go<__half>(p, sms, st);
    return launched(me);
  })
}
