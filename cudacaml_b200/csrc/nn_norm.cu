// ccb_nn_block_norm and its gradient: the norm after a block, its gate,
// dropout and residual scale, the residual sum, and the next block's norm.
//
//   u = norm(b) * w2 + c2,  y = x + s * m * act(g) * u,  h = norm(y) * w1 + c1
//
// With hat(v) = norm(v) and r its 1/deviation, the gradient is
//   g1 = dh * w1,  dY = dy + r1 * (g1 - yhat * mean(g1 * yhat) [- mean(g1)])
//   dx = dY,  du = s * m * act(g) * dY,  dgate = s * m * dY * u * act'(g)
//   g2 = du * w2,  db = r2 * (g2 - bhat * mean(g2 * bhat) [- mean(g2)])
//   dw1 = sum dh * yhat, dc1 = sum dh, dw2 = sum du * bhat, dc2 = sum du
// with the terms in brackets for the layer norm only. Statistics and sums are
// F32; the layer norm's variance is of the centred row (a second pass), since
// mean(v^2) - mean(v)^2 cancels where the mean is large.
#include "nn_common.cuh"

namespace ccb_nn {
namespace {

constexpr int kBlock = 256;
constexpr int kVecs = 5;  // dpre_weight, dpre_bias, dpost_weight, dpost_bias, dgate of a channel

struct NormP {
  const void *x, *b, *gate, *w1, *c1, *w2, *c2;
  void *y, *h;
  i64 rows, cols, xs, bs, gs, ys, hs;
  float eps, scale;
  int gdt, wdt, act, post;
  Drop d;
};

struct BackP {
  const void *y, *dy, *dh, *b, *gate, *w1, *w2, *c2;
  void *dx, *db, *dgate;
  float* vec[kVecs];
  float* part;  // [grid][kVecs][cols]
  i64 rows, cols, ys, dys, dhs, bs, gs, dxs, dbs, dgs;
  float eps, scale;
  int gdt, wdt, act, post;
  Drop d;
};

__device__ __forceinline__ float act_of(int act, float g) {
  return act == 1 ? 1.0f / (1.0f + expf(-g)) : act == 2 ? tanhf(g) : g;
}
// act'(g), from a = act(g)
__device__ __forceinline__ float slope_of(int act, float a) { return act == 1 ? a * (1.0f - a) : act == 2 ? 1.0f - a * a : 1.0f; }

// Sum of v over the block, the same in every thread.
__device__ __forceinline__ float block_sum(float v, float* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.0f;
#pragma unroll
  for (int i = 0; i < kBlock / 32; ++i) t += s[i];
  __syncthreads();
  return t;
}

// Mean (0 for kind 0) and 1/deviation of f(c), c < cols.
template <int KIND, class F>
__device__ __forceinline__ void stats(i64 cols, float eps, float* s, float& mean, float& r, F f) {
  mean = 0.0f;
  if (KIND == 1) {
    float t = 0.0f;
    for (i64 c = threadIdx.x; c < cols; c += kBlock) t += f(c);
    mean = block_sum(t, s) / (float)cols;
  }
  float t = 0.0f;
  for (i64 c = threadIdx.x; c < cols; c += kBlock) {
    const float v = f(c) - mean;
    t += v * v;
  }
  r = rsqrtf(block_sum(t, s) / (float)cols + eps);
}

// Rows of any length and alignment: a block walks a row once for each
// statistic and once for the results, reading it again each time.
template <class T, class TX, int KIND>
__global__ void __launch_bounds__(kBlock) norm_any(const __grid_constant__ NormP p) {
  __shared__ float s[kBlock / 32];
  for (i64 r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const TX* x = static_cast<const TX*>(p.x) + r * p.xs;
    const T* b = static_cast<const T*>(p.b) + r * p.bs;
    TX* yo = static_cast<TX*>(p.y) + r * p.ys;
    T* ho = static_cast<T*>(p.h) + r * p.hs;
    float m2 = 0.0f, r2 = 1.0f, m1, r1;
    if (p.b && p.post) stats<KIND>(p.cols, p.eps, s, m2, r2, [&](i64 c) { return to_f<T>(b[c]); });
    auto y_at = [&](i64 c) {
      float v = to_f<TX>(x[c]);
      if (p.b) {
        float u = (to_f<T>(b[c]) - m2) * r2;
        if (p.w2) u *= load_as(p.w2, p.wdt, c);
        if (p.c2) u += load_as(p.c2, p.wdt, c);
        if (p.gate) u *= act_of(p.act, load_as(p.gate, p.gdt, r * p.gs + c));
        v += p.scale * dropped_at(p.d, p.d.base + (u64)(r * p.cols + c), u);
      }
      return v;
    };
    if (p.h) stats<KIND>(p.cols, p.eps, s, m1, r1, y_at);
    for (i64 c = threadIdx.x; c < p.cols; c += kBlock) {
      const float v = y_at(c);
      if (p.h) {
        float h = (v - m1) * r1;
        if (p.w1) h *= load_as(p.w1, p.wdt, c);
        if (p.c1) h += load_as(p.c1, p.wdt, c);
        ho[c] = from_f<T>(h);
      }
      if (p.y) yo[c] = from_f<TX>(v);
    }
  }
}

// The gradient for any length and alignment. A block takes every grid-th row
// and keeps its own partial sums over rows in the workspace; a thread always
// handles the same columns of it.
template <class T, class TX, int KIND>
__global__ void __launch_bounds__(kBlock) norm_back_any(const __grid_constant__ BackP p) {
  __shared__ float s[kBlock / 32];
  float* part = p.part + (i64)blockIdx.x * kVecs * p.cols;
  for (int v = 0; v < kVecs; ++v)
    if (p.vec[v])
      for (i64 c = threadIdx.x; c < p.cols; c += kBlock) part[v * p.cols + c] = 0.0f;
  for (i64 r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const TX* y = static_cast<const TX*>(p.y) + r * p.ys;
    const TX* dy = static_cast<const TX*>(p.dy) + r * p.dys;
    const T* dh = static_cast<const T*>(p.dh) + r * p.dhs;
    const T* b = static_cast<const T*>(p.b) + r * p.bs;
    float m1 = 0.0f, r1 = 0.0f, a1 = 0.0f, f1 = 0.0f, m2 = 0.0f, r2 = 1.0f, a2 = 0.0f, f2 = 0.0f;
    auto g1_at = [&](i64 c) { return to_f<T>(dh[c]) * (p.w1 ? load_as(p.w1, p.wdt, c) : 1.0f); };
    if (p.dh) {
      stats<KIND>(p.cols, p.eps, s, m1, r1, [&](i64 c) { return to_f<TX>(y[c]); });
      float ta = 0.0f, tf = 0.0f;
      for (i64 c = threadIdx.x; c < p.cols; c += kBlock) {
        const float g = g1_at(c);
        ta += g * ((to_f<TX>(y[c]) - m1) * r1);
        tf += g;
      }
      a1 = block_sum(ta, s) / (float)p.cols;
      if (KIND == 1) f1 = block_sum(tf, s) / (float)p.cols;
    }
    auto dy_at = [&](i64 c) {
      float v = p.dy ? to_f<TX>(dy[c]) : 0.0f;
      if (p.dh) v += r1 * (g1_at(c) - (to_f<TX>(y[c]) - m1) * r1 * a1 - f1);
      return v;
    };
    auto act_at = [&](i64 c) { return p.gate ? act_of(p.act, load_as(p.gate, p.gdt, r * p.gs + c)) : 1.0f; };
    auto dz_at = [&](i64 c, float d) { return p.scale * dropped_at(p.d, p.d.base + (u64)(r * p.cols + c), d); };
    auto w2_at = [&](i64 c) { return p.w2 ? load_as(p.w2, p.wdt, c) : 1.0f; };
    if (p.b && p.post) {
      stats<KIND>(p.cols, p.eps, s, m2, r2, [&](i64 c) { return to_f<T>(b[c]); });
      float ta = 0.0f, tf = 0.0f;
      for (i64 c = threadIdx.x; c < p.cols; c += kBlock) {
        const float g = dz_at(c, dy_at(c)) * act_at(c) * w2_at(c);
        ta += g * ((to_f<T>(b[c]) - m2) * r2);
        tf += g;
      }
      a2 = block_sum(ta, s) / (float)p.cols;
      if (KIND == 1) f2 = block_sum(tf, s) / (float)p.cols;
    }
    // each element is read before the thread that owns it writes over it
    for (i64 c = threadIdx.x; c < p.cols; c += kBlock) {
      const float d = dy_at(c);
      if (p.dh) {
        const float h = to_f<T>(dh[c]);
        if (p.vec[0]) part[c] += h * ((to_f<TX>(y[c]) - m1) * r1);
        if (p.vec[1]) part[p.cols + c] += h;
      }
      if (p.b) {
        const float a = act_at(c), dz = dz_at(c, d), du = dz * a, w2 = w2_at(c);
        const float hat = (to_f<T>(b[c]) - m2) * r2;
        if (p.gate && (p.dgate || p.vec[4])) {
          const float u = hat * w2 + (p.c2 ? load_as(p.c2, p.wdt, c) : 0.0f);
          const float dg = dz * u * slope_of(p.act, a);
          if (p.vec[4])
            part[4 * p.cols + c] += dg;
          else if (p.gdt == CCB_F32)
            static_cast<float*>(p.dgate)[r * p.dgs + c] = dg;
          else
            static_cast<T*>(p.dgate)[r * p.dgs + c] = from_f<T>(dg);
        }
        if (p.vec[2]) part[2 * p.cols + c] += du * hat;
        if (p.vec[3]) part[3 * p.cols + c] += du;
        if (p.db) static_cast<T*>(p.db)[r * p.dbs + c] = from_f<T>(p.post ? r2 * (du * w2 - hat * a2 - f2) : du);
      }
      if (p.dx) static_cast<TX*>(p.dx)[r * p.dxs + c] = from_f<TX>(d);
    }
  }
}

// Column sums of the blocks' partials, in block order.
__global__ void __launch_bounds__(kBlock) norm_back_sum(const __grid_constant__ BackP p, int blocks) {
  float* out = p.vec[blockIdx.y];
  const i64 c = (i64)blockIdx.x * kBlock + threadIdx.x;
  if (!out || c >= p.cols) return;
  float t = 0.0f;
  for (int i = 0; i < blocks; ++i) t += p.part[((i64)i * kVecs + blockIdx.y) * p.cols + c];
  out[c] = t;
}

constexpr i64 kBackBlocks = 296;  // most blocks (and partial sums) of the gradient

size_t back_bytes(i64 rows, i64 cols) { return (size_t)(rows < kBackBlocks ? rows : kBackBlocks) * kVecs * (size_t)cols * sizeof(float); }

// The element types a call may have: dtype, and the residual stream in it or in f32.
template <template <class, class, int> class Go, class... A>
void by_type(int dtype, int x_dtype, int kind, A... a) {
#define CCB_NN_CASE(dt, xdt, T, TX)         \
  if (dtype == dt && x_dtype == xdt) {      \
    if (kind == 0)                          \
      Go<T, TX, 0>::run(a...);              \
    else                                    \
      Go<T, TX, 1>::run(a...);              \
    return;                                 \
  }
  CCB_NN_CASE(CCB_F32, CCB_F32, float, float)
  CCB_NN_CASE(CCB_BF16, CCB_BF16, __nv_bfloat16, __nv_bfloat16)
  CCB_NN_CASE(CCB_BF16, CCB_F32, __nv_bfloat16, float)
  CCB_NN_CASE(CCB_F16, CCB_F16, __half, __half)
  CCB_NN_CASE(CCB_F16, CCB_F32, __half, float)
#undef CCB_NN_CASE
}

template <class T, class TX, int KIND>
struct Forward {
  static void run(const NormP& p, int sms, cudaStream_t st) {
    const i64 most = (i64)sms * 8;
    norm_any<T, TX, KIND><<<(unsigned)(p.rows < most ? p.rows : most), kBlock, 0, st>>>(p);
  }
};

template <class T, class TX, int KIND>
struct Backward {
  static void run(const BackP& p, int sms, cudaStream_t st) {
    const i64 grid = p.rows < kBackBlocks ? p.rows : kBackBlocks;
    norm_back_any<T, TX, KIND><<<(unsigned)grid, kBlock, 0, st>>>(p);
    if (p.vec[0] || p.vec[1] || p.vec[2] || p.vec[3] || p.vec[4])
      norm_back_sum<<<dim3((unsigned)((p.cols + kBlock - 1) / kBlock), kVecs), kBlock, 0, st>>>(p, (int)grid);
  }
};

// Checks that both directions share; "" when fine.
std::string check_common(i64 rows, i64 cols, int dtype, int x_dtype, int gate_dtype, int weight_dtype, int kind, int act, double p,
                         double eps, double scale, bool gate, bool weights) {
  if (rows < 0 || cols < 0 || rows > INT_MAX || cols > (1 << 24)) return "rows must be in [0, 2^31), cols in [0, 2^24]";
  if (!float_type(dtype)) return "dtype code " + std::to_string(dtype) + " (0 f32, 4 bf16, 5 f16)";
  if (x_dtype != dtype && x_dtype != CCB_F32) return "x_dtype must be dtype or f32";
  if (gate && gate_dtype != dtype && gate_dtype != CCB_F32) return "gate_dtype must be dtype or f32";
  if (weights && !float_type(weight_dtype)) return "weight_dtype code " + std::to_string(weight_dtype) + " (0 f32, 4 bf16, 5 f16)";
  if (kind != 0 && kind != 1) return "kind must be 0 (rms) or 1 (layer)";
  if (act < 0 || act > 2) return "act must be 0 (none), 1 (sigmoid) or 2 (tanh)";
  if (!(p >= 0.0 && p <= 1.0)) return "p = " + std::to_string(p) + " is outside [0, 1]";
  if (!(eps >= 0.0) || !std::isfinite(eps)) return "eps must be finite and not negative";
  if (!std::isfinite(scale)) return "scale must be finite";
  return "";
}

// One matrix of a call: its pointer (may be NULL), row stride and element bytes.
struct Mat {
  const void* p;
  i64 stride;
  int bytes;
  const char* name;
};
std::string check_mats(i64 rows, i64 cols, std::initializer_list<Mat> mats) {
  for (const Mat& m : mats) {
    if (!m.p) continue;
    if (!sane(rows, cols, m.stride) || (rows > 1 && m.stride < cols)) return std::string(m.name) + "'s row stride is shorter than a row or out of range";
    if (!aligned(m.p, m.bytes)) return std::string(m.name) + " is not aligned to its element type";
  }
  return "";
}

}  // namespace
}  // namespace ccb_nn

using namespace ccb_nn;

extern "C" int ccb_nn_block_norm(const ccb_nn_block_norm_t* a, void* stream) {
  static const char* const me = "ccb_nn_block_norm";
  CCB_NN_GUARD(me, {
    if (!a) return fail(CCB_ERR_INVALID, me, "null argument block");
    std::string bad = check_common(a->rows, a->cols, a->dtype, a->x_dtype, a->gate_dtype, a->weight_dtype, a->kind, a->act, a->p, a->eps,
                                   a->scale, a->gate != nullptr, a->pre_weight || a->pre_bias || a->post_weight || a->post_bias);
    if (!bad.empty()) return fail(CCB_ERR_INVALID, me, bad);
    const int tb = type_bytes(a->dtype), xb = type_bytes(a->x_dtype), wb = type_bytes(a->weight_dtype);
    bad = check_mats(a->rows, a->cols, {{a->x, a->x_stride, xb, "x"}, {a->branch, a->branch_stride, tb, "branch"}, {a->y, a->y_stride, xb, "y"},
                                        {a->h, a->h_stride, tb, "h"}, {a->pre_weight, a->cols, wb, "pre_weight"}, {a->pre_bias, a->cols, wb, "pre_bias"},
                                        {a->post_weight, a->cols, wb, "post_weight"}, {a->post_bias, a->cols, wb, "post_bias"}});
    if (bad.empty() && a->gate && a->gate_stride != 0) bad = check_mats(a->rows, a->cols, {{a->gate, a->gate_stride, type_bytes(a->gate_dtype), "gate"}});
    if (bad.empty() && a->gate && !aligned(a->gate, type_bytes(a->gate_dtype))) bad = "gate is not aligned to its element type";
    if (bad.empty() && (a->rows == 0 || a->cols == 0)) return CCB_OK;
    if (bad.empty() && !a->branch && (a->y || a->gate || a->post_weight || a->post_bias))
      bad = "without a branch there is no y, gate, post_weight or post_bias";
    if (bad.empty() && !a->post_norm && (a->post_weight || a->post_bias)) bad = "post_weight and post_bias need post_norm";
    if (bad.empty() && !a->h && (a->pre_weight || a->pre_bias)) bad = "pre_weight and pre_bias need h";
    if (bad.empty() && !a->y && !a->h) bad = "neither y nor h is asked for";
    if (!bad.empty()) return fail(CCB_ERR_INVALID, me, bad);
    if (!a->x) return fail(CCB_ERR_INVALID, me, "null pointer");
    if (a->base > ~0ull - (u64)a->rows * (u64)a->cols) return fail(CCB_ERR_INVALID, me, "base + rows * cols passes 2^64");
    int sms = 0;
    if (const int rc = sm_count(me, &sms)) return rc;
    const NormP p = {a->x, a->branch, a->gate, a->pre_weight, a->pre_bias, a->post_weight, a->post_bias, a->y, a->h, a->rows, a->cols,
                     a->x_stride, a->branch_stride, a->gate_stride, a->y_stride, a->h_stride, (float)a->eps, (float)a->scale, a->gate_dtype,
                     a->weight_dtype, a->act, a->post_norm, make_drop(a->p, a->seed, a->offset, a->base)};
    by_type<Forward>(a->dtype, a->x_dtype, a->kind, p, sms, static_cast<cudaStream_t>(stream));
    return launched(me);
  })
}

extern "C" int ccb_nn_block_norm_backward_workspace(long long rows, long long cols, size_t* bytes) {
  static const char* const me = "ccb_nn_block_norm_backward_workspace";
  CCB_NN_GUARD(me, {
    if (!bytes) return fail(CCB_ERR_INVALID, me, "null pointer");
    if (rows < 0 || cols < 0 || rows > INT_MAX || cols > (1 << 24)) return fail(CCB_ERR_INVALID, me, "rows must be in [0, 2^31), cols in [0, 2^24]");
    *bytes = back_bytes(rows, cols);
    return CCB_OK;
  })
}

extern "C" int ccb_nn_block_norm_backward(const ccb_nn_block_norm_backward_t* a, void* stream) {
  static const char* const me = "ccb_nn_block_norm_backward";
  CCB_NN_GUARD(me, {
    if (!a) return fail(CCB_ERR_INVALID, me, "null argument block");
    std::string bad = check_common(a->rows, a->cols, a->dtype, a->x_dtype, a->gate_dtype, a->weight_dtype, a->kind, a->act, a->p, a->eps,
                                   a->scale, a->gate != nullptr, a->pre_weight || a->post_weight || a->post_bias);
    if (!bad.empty()) return fail(CCB_ERR_INVALID, me, bad);
    const int tb = type_bytes(a->dtype), xb = type_bytes(a->x_dtype), wb = type_bytes(a->weight_dtype), gb = a->gate ? type_bytes(a->gate_dtype) : 4;
    const bool channel = a->gate && a->gate_stride == 0;
    bad = check_mats(a->rows, a->cols,
                     {{a->y, a->y_stride, xb, "y"}, {a->dy, a->dy_stride, xb, "dy"}, {a->dh, a->dh_stride, tb, "dh"},
                      {a->branch, a->branch_stride, tb, "branch"}, {a->dx, a->dx_stride, xb, "dx"}, {a->dbranch, a->dbranch_stride, tb, "dbranch"},
                      {a->gate, channel ? a->cols : a->gate_stride, gb, "gate"}, {a->dgate, channel ? a->cols : a->dgate_stride, channel ? 4 : gb, "dgate"},
                      {a->pre_weight, a->cols, wb, "pre_weight"}, {a->post_weight, a->cols, wb, "post_weight"},
                      {a->post_bias, a->cols, wb, "post_bias"}, {a->dpre_weight, a->cols, 4, "dpre_weight"}, {a->dpre_bias, a->cols, 4, "dpre_bias"},
                      {a->dpost_weight, a->cols, 4, "dpost_weight"}, {a->dpost_bias, a->cols, 4, "dpost_bias"}});
    if (!bad.empty()) return fail(CCB_ERR_INVALID, me, bad);
    if (a->cols == 0) return CCB_OK;
    const bool sums = a->dpre_weight || a->dpre_bias || a->dpost_weight || a->dpost_bias || (channel && a->dgate);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->rows == 0) {  // sums over no rows
      for (void* v : {a->dpre_weight, a->dpre_bias, a->dpost_weight, a->dpost_bias, channel ? a->dgate : nullptr})
        if (v) {
          const cudaError_t e = cudaMemsetAsync(v, 0, (size_t)a->cols * 4, st);
          if (e != cudaSuccess) return fail(CCB_ERR_DRIVER, me, std::string("cudaMemsetAsync: ") + cudaGetErrorString(e));
        }
      return CCB_OK;
    }
    if (bad.empty() && !a->branch && (a->dbranch || a->gate || a->dgate || a->post_weight || a->post_bias || a->dpost_weight || a->dpost_bias))
      bad = "without a branch there is no gate, post_weight, post_bias or gradient of them";
    if (bad.empty() && a->dgate && !a->gate) bad = "dgate needs the gate";
    if (bad.empty() && !a->post_norm && (a->post_weight || a->post_bias || a->dpost_weight || a->dpost_bias)) bad = "post_weight and post_bias need post_norm";
    if (bad.empty() && !a->dh && (a->pre_weight || a->dpre_weight || a->dpre_bias)) bad = "pre_weight, dpre_weight and dpre_bias need dh";
    if (!bad.empty()) return fail(CCB_ERR_INVALID, me, bad);
    if (!a->y && a->dh) return fail(CCB_ERR_INVALID, me, "null pointer: y");
    if (!a->dy && !a->dh) return fail(CCB_ERR_INVALID, me, "neither dy nor dh is given");
    if (a->base > ~0ull - (u64)a->rows * (u64)a->cols) return fail(CCB_ERR_INVALID, me, "base + rows * cols passes 2^64");
    if (sums && (!a->workspace || a->workspace_bytes < back_bytes(a->rows, a->cols) || !aligned(a->workspace, 16)))
      return fail(CCB_ERR_INVALID, me, "workspace of " + std::to_string(a->workspace_bytes) + " bytes: " + std::to_string(back_bytes(a->rows, a->cols)) +
                                           " are needed, 16-byte aligned");
    int sms = 0;
    if (const int rc = sm_count(me, &sms)) return rc;
    const BackP p = {a->y, a->dy, a->dh, a->branch, a->gate, a->pre_weight, a->post_weight, a->post_bias, a->dx, a->dbranch,
                     channel ? nullptr : a->dgate,
                     {(float*)a->dpre_weight, (float*)a->dpre_bias, (float*)a->dpost_weight, (float*)a->dpost_bias, channel ? (float*)a->dgate : nullptr},
                     (float*)a->workspace, a->rows, a->cols, a->y_stride, a->dy_stride, a->dh_stride, a->branch_stride, a->gate_stride, a->dx_stride,
                     a->dbranch_stride, a->dgate_stride, (float)a->eps, (float)a->scale, a->gate_dtype, a->weight_dtype, a->act, a->post_norm,
                     make_drop(a->p, a->seed, a->offset, a->base)};
    by_type<Backward>(a->dtype, a->x_dtype, a->kind, p, sms, st);
    return launched(me);
  })
}
