// ccb_nn_grouped_matmul and ccb_nn_grouped_matmul_dw: products grouped by
// expert. The row ranges of the experts live in device memory, so every block
// lays the tiles out for itself: it clamps the offsets, counts the row tiles
// of each segment and scans the counts in shared memory.
#include "nn_common.cuh"

namespace ccb_nn {
namespace {

constexpr int kMaxExperts = 1024;
constexpr unsigned kErrOffsets = 64u;

struct GroupP {
  const void *x, *w;
  const int* off;
  void* out;
  unsigned* err;
  i64 k, n, xs, we, ws, os;
  int rows, experts;
};
struct GroupDwP {
  const void *x, *dy;
  const int* off;
  void* out;
  unsigned* err;
  i64 k, n, xs, ys, oe, os;
  int rows, experts;
};

// Row ranges and their tiles of `bm` rows. Segment s in [1, experts] is
// expert s - 1; segments 0 and experts + 1 are the rows that belong to none.
struct Segments {
  int row[kMaxExperts + 3];   // segment s is rows [row[s], row[s + 1])
  int tile[kMaxExperts + 3];  // its first tile; [segments] is the count
};

// Called by the whole block (blockDim.x a multiple of 32).
__device__ __forceinline__ void lay_out(Segments& g, const int* off, int experts, int rows, int bm, unsigned* err) {
  const int segs = experts + 2;
  for (int s = threadIdx.x; s <= experts; s += blockDim.x) g.row[s + 1] = off[s];
  if (threadIdx.x == 0) {
    g.row[0] = 0;
    g.row[segs] = rows;
  }
  __syncthreads();
  if (threadIdx.x < 32) {  // running maximum of the clamped offsets, then tile counts, 32 at a time
    const int lane = threadIdx.x;
    int high = 0;
    bool bad = false;
    for (int s0 = 1; s0 <= experts + 1; s0 += 32) {
      const int s = s0 + lane;
      const bool in = s <= experts + 1;
      const int raw = in ? g.row[s] : 0;
      int v = min(max(raw, 0), rows);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = max(v, u);
      }
      v = max(v, high);
      if (in) {
        bad |= v != raw;
        g.row[s] = v;
      }
      high = __shfl_sync(0xffffffffu, v, 31);
    }
    if (__any_sync(0xffffffffu, bad) && lane == 0 && err) atomicOr(err, kErrOffsets);
    __syncwarp();
    int base = 0;
    for (int s0 = 0; s0 < segs; s0 += 32) {
      const int s = s0 + lane;
      const int c = s < segs ? (g.row[s + 1] - g.row[s] + bm - 1) / bm : 0;
      int v = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (s < segs) g.tile[s] = base + v - c;
      base += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) g.tile[segs] = base;
  }
  __syncthreads();
}
// The segment that holds row tile t < tile[segs].
__device__ __forceinline__ int segment_of(const Segments& g, int segs, int t) {
  int lo = 0, hi = segs - 1;  // the last segment whose first tile is <= t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (g.tile[mid] <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// ------------------------------------------------- CUDA cores, any alignment
// 64 x 64 tiles, 16 of the contraction at a time, 4 x 4 results a thread.
constexpr int kB = 64, kK = 16;

__device__ __forceinline__ void simt_step(const float (*a)[kB + 4], const float (*b)[kB + 4], float acc[4][4], int tx, int ty) {
#pragma unroll
  for (int k = 0; k < kK; ++k) {
    float av[4], bv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) av[i] = a[k][ty * 4 + i];
#pragma unroll
    for (int j = 0; j < 4; ++j) bv[j] = b[k][tx * 4 + j];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
  }
}

template <class T, bool WT>
__global__ void __launch_bounds__(256) grouped_any(const __grid_constant__ GroupP p) {
  __shared__ Segments g;
  __shared__ float sa[kK][kB + 4], sb[kK][kB + 4];
  lay_out(g, p.off, p.experts, p.rows, kB, p.err);
  const int segs = p.experts + 2, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const i64 nt = (p.n + kB - 1) / kB, total = nt * g.tile[segs];
  const T* x = static_cast<const T*>(p.x);
  for (i64 t = blockIdx.x; t < total; t += gridDim.x) {
    const int mt = (int)(t / nt);
    const i64 n0 = (t % nt) * kB;
    const int s = segment_of(g, segs, mt);
    const int r0 = g.row[s] + (mt - g.tile[s]) * kB, r1 = min(g.row[s + 1], r0 + kB);
    float acc[4][4] = {};
    if (s >= 1 && s <= p.experts) {
      const T* w = static_cast<const T*>(p.w) + (s - 1) * p.we;
      for (i64 k0 = 0; k0 < p.k; k0 += kK) {
        for (int i = threadIdx.x; i < kB * kK; i += 256) {
          const int m = i / kK, k = i % kK;
          sa[k][m] = r0 + m < r1 && k0 + k < p.k ? to_f<T>(x[(i64)(r0 + m) * p.xs + k0 + k]) : 0.0f;
        }
        for (int i = threadIdx.x; i < kB * kK; i += 256) {
          const int k = WT ? i % kK : i / kB, n = WT ? i / kK : i % kB;
          sb[k][n] = n0 + n < p.n && k0 + k < p.k ? to_f<T>(w[WT ? (n0 + n) * p.ws + k0 + k : (k0 + k) * p.ws + n0 + n]) : 0.0f;
        }
        __syncthreads();
        simt_step(sa, sb, acc, tx, ty);
        __syncthreads();
      }
    }
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j) {
        const i64 r = r0 + ty * 4 + i, c = n0 + tx * 4 + j;
        if (r < r1 && c < p.n) static_cast<T*>(p.out)[r * p.os + c] = from_f<T>(acc[i][j]);
      }
  }
}

template <class T, class TO>
__global__ void __launch_bounds__(256) grouped_dw_any(const __grid_constant__ GroupDwP p) {
  __shared__ Segments g;
  __shared__ float sa[kK][kB + 4], sb[kK][kB + 4];
  lay_out(g, p.off, p.experts, p.rows, kB, p.err);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const i64 kt = (p.k + kB - 1) / kB, nt = (p.n + kB - 1) / kB, total = kt * nt * p.experts;
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  for (i64 t = blockIdx.x; t < total; t += gridDim.x) {
    const int e = (int)(t / (kt * nt));
    const i64 m0 = (t / nt % kt) * kB, n0 = (t % nt) * kB;
    const int r1 = g.row[e + 2];
    float acc[4][4] = {};
    for (i64 r0 = g.row[e + 1]; r0 < r1; r0 += kK) {
      for (int i = threadIdx.x; i < kB * kK; i += 256) {
        const int k = i / kB, c = i % kB;
        const bool in = r0 + k < r1;
        sa[k][c] = in && m0 + c < p.k ? to_f<T>(x[(r0 + k) * p.xs + m0 + c]) : 0.0f;
        sb[k][c] = in && n0 + c < p.n ? to_f<T>(dy[(r0 + k) * p.ys + n0 + c]) : 0.0f;
      }
      __syncthreads();
      simt_step(sa, sb, acc, tx, ty);
      __syncthreads();
    }
    TO* out = static_cast<TO*>(p.out) + e * p.oe;
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j) {
        const i64 r = m0 + ty * 4 + i, c = n0 + tx * 4 + j;
        if (r < p.k && c < p.n) out[r * p.os + c] = from_f<TO>(acc[i][j]);
      }
  }
}

template <class T>
void any(const GroupP& p, bool wt, int sms, cudaStream_t st) {
  const i64 tiles = ((p.rows + kB - 1) / kB + p.experts + 1) * ((p.n + kB - 1) / kB), most = (i64)sms * 4;
  const unsigned grid = (unsigned)(tiles < most ? tiles : most);
  if (wt)
    grouped_any<T, true><<<grid, 256, 0, st>>>(p);
  else
    grouped_any<T, false><<<grid, 256, 0, st>>>(p);
}
template <class T, class TO>
void any_dw(const GroupDwP& p, int sms, cudaStream_t st) {
  const i64 tiles = ((p.k + kB - 1) / kB) * ((p.n + kB - 1) / kB) * p.experts, most = (i64)sms * 4;
  grouped_dw_any<T, TO><<<(unsigned)(tiles < most ? tiles : most), 256, 0, st>>>(p);
}

std::string check_sizes(i64 rows, i64 experts, i64 k, i64 n, int dtype) {
  if (rows < 0 || rows > INT_MAX) return "rows must be in [0, 2^31)";
  if (experts < 1 || experts > kMaxExperts) return "experts must be in [1, " + std::to_string(kMaxExperts) + "]";
  if (k < 0 || n < 0 || k > INT_MAX || n > INT_MAX) return "k and n must be in [0, 2^31)";
  if (!float_type(dtype)) return "dtype code " + std::to_string(dtype) + " (0 f32, 4 bf16, 5 f16)";
  return "";
}
std::string check_mat(const void* p, i64 rows, i64 cols, i64 stride, int bytes, const char* name) {
  if (!sane(rows, cols, stride) || (rows > 1 && stride < cols)) return std::string(name) + "'s row stride is shorter than a row or out of range";
  if (!aligned(p, bytes)) return std::string(name) + " is not aligned to its element type";
  return "";
}
// a stack of matrices: `stride` elements from one to the next
std::string check_stack(const void* p, i64 count, i64 rows, i64 cols, i64 stride, i64 row_stride, int bytes, const char* name) {
  const std::string bad = check_mat(p, rows, cols, row_stride, bytes, name);
  if (!bad.empty()) return bad;
  if (count > 1 && rows > 0 && cols > 0 && (stride < (rows - 1) * row_stride + cols || !sane(count, cols, stride)))
    return std::string(name) + "'s stride is shorter than a matrix or out of range";
  return "";
}
std::string check_grouped(const ccb_nn_grouped_matmul_t* a) {
  std::string bad = check_sizes(a->rows, a->experts, a->k, a->n, a->dtype);
  const int b = type_bytes(a->dtype);
  if (bad.empty()) bad = check_mat(a->x, a->rows, a->k, a->x_stride, b, "x");
  if (bad.empty()) bad = check_mat(a->out, a->rows, a->n, a->out_stride, b, "out");
  if (bad.empty())
    bad = check_stack(a->w, a->experts, a->transpose_w ? a->n : a->k, a->transpose_w ? a->k : a->n, a->w_stride, a->w_row_stride, b, "w");
  return bad;
}
std::string check_dw(const ccb_nn_grouped_matmul_dw_t* a) {
  std::string bad = check_sizes(a->rows, a->experts, a->k, a->n, a->dtype);
  const int b = type_bytes(a->dtype);
  if (bad.empty() && a->out_dtype != a->dtype && a->out_dtype != CCB_F32) bad = "out_dtype must be dtype or f32";
  if (bad.empty()) bad = check_mat(a->x, a->rows, a->k, a->x_stride, b, "x");
  if (bad.empty()) bad = check_mat(a->dy, a->rows, a->n, a->dy_stride, b, "dy");
  if (bad.empty()) bad = check_stack(a->out, a->experts, a->k, a->n, a->out_stride, a->out_row_stride, type_bytes(a->out_dtype), "out");
  return bad;
}
size_t workspace_of(const ccb_nn_grouped_matmul_t*) { return 0; }
size_t workspace_of(const ccb_nn_grouped_matmul_dw_t*) { return 0; }

}  // namespace
}  // namespace ccb_nn

using namespace ccb_nn;

extern "C" int ccb_nn_grouped_matmul_workspace(const ccb_nn_grouped_matmul_t* a, size_t* bytes) {
  static const char* const me = "ccb_nn_grouped_matmul_workspace";
  CCB_NN_GUARD(me, {
    if (!a || !bytes) return fail(CCB_ERR_INVALID, me, "null pointer");
    const std::string bad = check_grouped(a);
    if (!bad.empty()) return fail(CCB_ERR_INVALID, me, bad);
    *bytes = workspace_of(a);
    return CCB_OK;
  })
}

extern "C" int ccb_nn_grouped_matmul_dw_workspace(const ccb_nn_grouped_matmul_dw_t* a, size_t* bytes) {
  static const char* const me = "ccb_nn_grouped_matmul_dw_workspace";
  CCB_NN_GUARD(me, {
    if (!a || !bytes) return fail(CCB_ERR_INVALID, me, "null pointer");
    const std::string bad = check_dw(a);
    if (!bad.empty()) return fail(CCB_ERR_INVALID, me, bad);
    *bytes = workspace_of(a);
    return CCB_OK;
  })
}

extern "C" int ccb_nn_grouped_matmul(const ccb_nn_grouped_matmul_t* a, void* stream) {
  static const char* const me = "ccb_nn_grouped_matmul";
  CCB_NN_GUARD(me, {
    if (!a) return fail(CCB_ERR_INVALID, me, "null argument block");
    const std::string bad = check_grouped(a);
    if (!bad.empty()) return fail(CCB_ERR_INVALID, me, bad);
    if (a->rows == 0 || a->n == 0) return CCB_OK;
    if (!a->offsets || !a->out || (a->k > 0 && (!a->x || !a->w))) return fail(CCB_ERR_INVALID, me, "null pointer");
    if (!aligned(a->offsets, 4) || !aligned(a->err, 4)) return fail(CCB_ERR_INVALID, me, "offsets or err is not aligned to 4 bytes");
    int sms = 0;
    if (const int rc = sm_count(me, &sms)) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const GroupP p = {a->x, a->w, a->offsets, a->out, a->err, a->k, a->n, a->x_stride, a->w_stride, a->w_row_stride, a->out_stride, (int)a->rows, (int)a->experts};
    if (a->dtype == CCB_F32)
      any<float>(p, a->transpose_w, sms, st);
    else if (a->dtype == CCB_BF16)
      any<__nv_bfloat16>(p, a->transpose_w, sms, st);
    else
      any<__half>(p, a->transpose_w, sms, st);
    return launched(me);
  })
}

extern "C" int ccb_nn_grouped_matmul_dw(const ccb_nn_grouped_matmul_dw_t* a, void* stream) {
  static const char* const me = "ccb_nn_grouped_matmul_dw";
  CCB_NN_GUARD(me, {
    if (!a) return fail(CCB_ERR_INVALID, me, "null argument block");
    const std::string bad = check_dw(a);
    if (!bad.empty()) return fail(CCB_ERR_INVALID, me, bad);
    if (a->k == 0 || a->n == 0) return CCB_OK;
    if (!a->offsets || !a->out || (a->rows > 0 && (!a->x || !a->dy))) return fail(CCB_ERR_INVALID, me, "null pointer");
    if (!aligned(a->offsets, 4) || !aligned(a->err, 4)) return fail(CCB_ERR_INVALID, me, "offsets or err is not aligned to 4 bytes");
    int sms = 0;
    if (const int rc = sm_count(me, &sms)) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const GroupDwP p = {a->x, a->dy, a->offsets, a->out, a->err, a->k, a->n, a->x_stride, a->dy_stride, a->out_stride, a->out_row_stride, (int)a->rows, (int)a->experts};
    if (a->dtype == CCB_F32)
      any_dw<float, float>(p, sms, st);
    else if (a->dtype == CCB_BF16 && a->out_dtype == CCB_F32)
      any_dw<__nv_bfloat16, float>(p, sms, st);
    else if (a->dtype == CCB_BF16)
      any_dw<__nv_bfloat16, __nv_bfloat16>(p, sms, st);
    else if (a->out_dtype == CCB_F32)
      any_dw<__half, float>(p, sms, st);
    else
      any_dw<__half, __half>(p, sms, st);
    return launched(me);
  })
}
