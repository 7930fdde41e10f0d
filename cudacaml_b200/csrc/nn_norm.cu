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
#include <initializer_list>
#include <type_traits>

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

// -------------------------------------------------------- rows read once
// A group of `tpr` threads (whole warps) holds a row, PIECES times 8 elements
// a thread, and copies the rows that come next into a ring in shared memory
// meanwhile (cp.async: no registers, and nothing waits for the loads). VEC
// (cols a multiple of 8; pointers and strides of 16 bytes): a thread's elements
// are consecutive, and it copies and reads its own alone, so that there is no
// barrier. Otherwise they are tpr apart, and the group copies the 16-byte
// pieces of memory that hold the row between its threads. A block holds
// blockDim.x / tpr rows at a time and takes every grid-th set.
constexpr int kE = 8;

template <bool VEC>
struct Place {
  int t, tpr, cols;
  __device__ __forceinline__ int at(int i) const { return VEC ? t * kE + i : i * tpr + t; }
  __device__ __forceinline__ bool on(int i) const { return VEC ? t * kE < cols : i * tpr + t < cols; }
  // Where a thread has several pieces: the k-th.
  __device__ __forceinline__ Place piece(int k) const { return {VEC ? t + k * tpr : t + k * kE * tpr, tpr, cols}; }
};

// Bytes of one matrix's part of a slot of the ring. VEC: planes of 16 bytes
// for each thread of the block (free of bank conflicts whatever a place
// holds); else a row and its unaligned ends for each group.
template <class A, bool VEC, int PIECES>
__host__ __device__ inline unsigned part_bytes(int cols, int block, int tpr) {
  return VEC ? (unsigned)(PIECES * (sizeof(A) / 2) * block * 16) : (unsigned)(block / tpr) * (((unsigned)cols * (unsigned)sizeof(A) + 31u) & ~15u);
}
template <class A, bool VEC, int PIECES>
struct Part {
  // `to`: the thread's place (VEC) or the group's, in the matrix's part.
  static __device__ __forceinline__ void fetch(unsigned to, const A* row, const Place<VEC>& w) {
    if constexpr (VEC) {
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        if (!w.piece(k).on(0)) break;
#pragma unroll
        for (int h = 0; h < (int)sizeof(A) / 2; ++h)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + (k * (int)sizeof(A) / 2 + h) * blockDim.x * 16),
                       "l"(reinterpret_cast<const char*>(row + w.piece(k).at(0)) + 16 * h)
                       : "memory");
      }
    } else {
      const u64 a = reinterpret_cast<u64>(row);
      const int bytes = (int)(a & 15) + w.cols * (int)sizeof(A);
      for (int c = w.t * 16; c < bytes; c += w.tpr * 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + c), "l"((a & ~15ull) + c), "r"(min(16, bytes - c)) : "memory");
    }
  }
  // Piece k as F32, from the place that `row` was copied to.
  static __device__ __forceinline__ void get(float* v, unsigned from, const A* row, const Place<VEC>& w, int k) {
    if constexpr (VEC) {
      unsigned u[kE * sizeof(A) / 4];
#pragma unroll
      for (int h = 0; h < (int)sizeof(A) / 2; ++h)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(u[4 * h]), "=r"(u[4 * h + 1]), "=r"(u[4 * h + 2]), "=r"(u[4 * h + 3])
                     : "r"(from + (k * (int)sizeof(A) / 2 + h) * blockDim.x * 16));
#pragma unroll
      for (int i = 0; i < kE; ++i) {
        if constexpr (sizeof(A) == 4)
          v[i] = __uint_as_float(u[i]);
        else if constexpr (std::is_same<A, __nv_bfloat16>::value)
          v[i] = __uint_as_float(i & 1 ? u[i >> 1] & 0xFFFF0000u : u[i >> 1] << 16);
        else
          v[i] = __half2float(__ushort_as_half((unsigned short)(i & 1 ? u[i >> 1] >> 16 : u[i >> 1])));
      }
    } else {
      const Place<VEC> q = w.piece(k);
      const unsigned at = from + (unsigned)(reinterpret_cast<u64>(row) & 15);
#pragma unroll
      for (int i = 0; i < kE; ++i) {
        v[i] = 0.0f;
        if (!q.on(i)) continue;
        if constexpr (sizeof(A) == 4) {
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[i]) : "r"(at + 4 * q.at(i)));
        } else {
          unsigned short h;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(at + 2 * q.at(i)));
          v[i] = std::is_same<A, __nv_bfloat16>::value ? __uint_as_float((unsigned)h << 16) : __half2float(__ushort_as_half(h));
        }
      }
    }
  }
};
template <class A, bool VEC>
__device__ __forceinline__ void store8(A* row, const float* v, const Place<VEC>& w) {
  if constexpr (VEC) {
    if (!w.on(0)) return;
    A* p = row + w.at(0);
    if constexpr (sizeof(A) == 4) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint4 u;
      u.x = pack2<A>(v[0], v[1]);
      u.y = pack2<A>(v[2], v[3]);
      u.z = pack2<A>(v[4], v[5]);
      u.w = pack2<A>(v[6], v[7]);
      *reinterpret_cast<uint4*>(p) = u;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kE; ++i)
      if (w.on(i)) row[w.at(i)] = from_f<A>(v[i]);
  }
}
// A vector over the columns, of a type known at run time; `none` where there
// is no vector or no column.
template <bool VEC>
__device__ __forceinline__ void vec8(float* v, const void* p, int dtype, float none, const Place<VEC>& w) {
#pragma unroll
  for (int j = 0; j < kE; ++j) v[j] = p && w.on(j) ? load_as(p, dtype, w.at(j)) : none;
}
// The vectors over the columns, kept in F32 in shared memory from row to row
// (beside the ring there is no L1 left to keep them), as 16-byte halves in
// planes of a group's threads; the groups share them.
struct Kept {
  unsigned at, plane;
  __device__ __forceinline__ void put(int slot, const float* v) const {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at + (2 * slot + h) * plane), "f"(v[4 * h]), "f"(v[4 * h + 1]), "f"(v[4 * h + 2]), "f"(v[4 * h + 3])
                   : "memory");
  }
  __device__ __forceinline__ void get(int slot, float* v) const {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[4 * h]), "=f"(v[4 * h + 1]), "=f"(v[4 * h + 2]), "=f"(v[4 * h + 3]) : "r"(at + (2 * slot + h) * plane));
  }
};
// How a launch holds its rows: threads of a row, slots of the ring and their
// bytes, where the vectors are kept and where the generator's words go.
struct Hold {
  int tpr, ahead;
  unsigned slot, kept, words;
};

// Sums of N values over a group, the same bits in every thread: by shuffles in
// each warp, then over the warps' results, in two buffers in turn, so that one
// barrier a sum is enough.
struct Group {
  float* s;  // [2][warps][4]
  int warps, span, id, threads, turn;
  __device__ __forceinline__ void meet() const {
    if (warps == 1)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(threads) : "memory");
  }
  __device__ __forceinline__ Group(float* all, int tpr) : warps(tpr >> 5), id(threadIdx.x / tpr), threads(tpr), turn(0) {
    s = all + id * warps * 8;
    span = 1;
    while (span < warps) span *= 2;
  }
  template <int N>
  __device__ __forceinline__ void sum(float* v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
    if (warps == 1) return;
    float* b = s + turn * warps * 4;
    turn ^= 1;
    const int lane = threadIdx.x & 31;
    if (lane == 0) {
      const int warp = (threadIdx.x >> 5) - id * warps;
#pragma unroll
      for (int n = 0; n < N; ++n) b[warp * 4 + n] = v[n];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(threads) : "memory");
    const int l = lane & (span - 1);
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = l < warps ? b[l * 4 + n] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      if (o < span)
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  }
};

// The generator's words of a thread's 8 elements of a row whose first index is
// e0. Consecutive elements (VEC): two of its blocks, or three where the index
// is no multiple of 4. Single ones: a warp's 32 elements of one step lie in at
// most 9 blocks, so the warp computes the 72 of all steps between its lanes
// and hands the words out through its part of shared memory.
constexpr int kWarpWords = 9 * kE * 4;
template <bool VEC>
__device__ __forceinline__ void words8(unsigned* u, const Drop& d, u64 e0, const Place<VEC>& w, unsigned char* places) {
  if constexpr (VEC) {
    philox8(d, e0 + (u64)w.at(0), u);
  } else {
    uint4* out = reinterpret_cast<uint4*>(places) + (threadIdx.x >> 5) * (kWarpWords / 4);
    const int lane = threadIdx.x & 31;
    const u64 e = e0 + (u64)(w.t - lane);  // the warp's first element of step 0
    __syncwarp();
    for (int b = lane; b < 9 * kE; b += 32) {
      const int i = b / 9;
      unsigned x[4];
      philox4(d, ((e + (u64)(i * w.tpr)) >> 2) + (u64)(b - 9 * i), x);
      out[b] = make_uint4(x[0], x[1], x[2], x[3]);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kE; ++i) u[i] = reinterpret_cast<const unsigned*>(out)[36 * i + (int)((e + (u64)(i * w.tpr)) & 3) + lane];
  }
}

// act(g) from the hardware's exponential and reciprocal: a few units in the
// last place, below the rounding of any 16-bit result and within 1e-6 in F32.
__device__ __forceinline__ void act8(int act, float* g) {
  if (act == 1) {
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      float e;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g[i] * -1.4426950408889634f));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(g[i]) : "f"(1.0f + e));
    }
  } else if (act == 2) {
#pragma unroll
    for (int i = 0; i < kE; ++i) g[i] = tanhf(g[i]);
  }
}
// act'(g) times v, from a = act(g)
__device__ __forceinline__ void slope8(int act, const float* a, float* v) {
  if (act == 1) {
#pragma unroll
    for (int i = 0; i < kE; ++i) v[i] *= a[i] * (1.0f - a[i]);
  } else if (act == 2) {
#pragma unroll
    for (int i = 0; i < kE; ++i) v[i] *= 1.0f - a[i] * a[i];
  }
}
// The gate's row where it is not a matrix of T: one for all, or in f32.
__device__ __forceinline__ const void* gate_row(const void* gate, int gdt, i64 gs, i64 r) {
  return gate ? static_cast<const char*>(gate) + r * gs * (gdt == CCB_F32 ? 4 : 2) : nullptr;
}

// Row r of a matrix: one 32 x 32 -> 64 product (the launch sees to it that a
// row's bytes fit) instead of a 64-bit one, and no pointer kept from row to row.
template <class A>
__device__ __forceinline__ const A* row_at(const void* m, unsigned r, i64 stride) {
  return reinterpret_cast<const A*>(static_cast<const char*>(m) + (u64)r * (unsigned)(stride * (i64)sizeof(A)));
}
template <class A>
__device__ __forceinline__ A* row_at(void* m, unsigned r, i64 stride) {
  return reinterpret_cast<A*>(static_cast<char*>(m) + (u64)r * (unsigned)(stride * (i64)sizeof(A)));
}
// Waits until at most n of the thread's groups of copies are on their way.
__device__ __forceinline__ void copied(int n) {
  if (n == 1)
    asm volatile("cp.async.wait_group 1;" ::: "memory");
  else if (n == 2)
    asm volatile("cp.async.wait_group 2;" ::: "memory");
  else
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}
// The row in hand is in its slot and the next one's copies are issued: one
// slot ahead of a full ring, since the slot before the row in hand is free.
template <bool VEC, class F>
__device__ __forceinline__ void turn_ring(const Group& g, int ahead, F fetch) {
  if (ahead == 1) {
    if (!VEC) g.meet();
    fetch();
    copied(0);
    if (!VEC) g.meet();
  } else if (VEC) {
    fetch();
    copied(ahead - 1);
  } else {
    copied(ahead - 2);
    g.meet();  // everyone's copies are in, and everyone is done with the row before
    fetch();
  }
}

template <class T, class TX, bool VEC, int PIECES>
__global__ void __launch_bounds__(512) norm_rows(const __grid_constant__ NormP p, int kind, const Hold hold) {
  __shared__ __align__(16) float s[16 * 8];
  extern __shared__ __align__(16) unsigned char places[];
  typedef Part<TX, VEC, PIECES> PX;
  typedef Part<T, VEC, PIECES> PT;
  const int tpr = hold.tpr, ahead = hold.ahead;
  Group g(s, tpr);
  const Place<VEC> w0 = {(int)threadIdx.x - g.id * tpr, tpr, (int)p.cols};
  const float inv = 1.0f / (float)p.cols, f = p.scale * p.d.factor;
  const bool channel = p.gate && p.gs == 0, full = p.gate && !channel && p.gdt != CCB_F32;
  const unsigned sets = blockDim.x / tpr, first = blockIdx.x * sets + g.id, step = gridDim.x * sets, rows = (unsigned)p.rows;
  const unsigned all = (unsigned)__cvta_generic_to_shared(places);
  const unsigned ox = VEC ? threadIdx.x * 16 : g.id * (part_bytes<TX, VEC, PIECES>(p.cols, blockDim.x, tpr) / sets);
  const unsigned ob = part_bytes<TX, VEC, PIECES>(p.cols, blockDim.x, tpr) + (VEC ? threadIdx.x * 16 : g.id * (part_bytes<T, VEC, PIECES>(p.cols, blockDim.x, tpr) / sets));
  const unsigned og = ob + part_bytes<T, VEC, PIECES>(p.cols, blockDim.x, tpr), end = all + ahead * hold.slot;
  // kept, for each piece: w2, w1, then c2, c1 and a channel gate's act, as far as there are any
  const Kept kept = {all + hold.kept + w0.t * 16, (unsigned)tpr * 16};
  const int c1_at = 2 + (p.c2 != nullptr), gate_at = c1_at + (p.c1 != nullptr), slots = gate_at + channel;
  if (g.id == 0) {
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const Place<VEC> w = w0.piece(k);
      float v[kE];
      vec8(v, p.w2, p.wdt, 1.0f, w);
      kept.put(k * slots, v);
      vec8(v, p.w1, p.wdt, 1.0f, w);
      kept.put(k * slots + 1, v);
      if (p.c2) {
        vec8(v, p.c2, p.wdt, 0.0f, w);
        kept.put(k * slots + 2, v);
      }
      if (p.c1) {
        vec8(v, p.c1, p.wdt, 0.0f, w);
        kept.put(k * slots + c1_at, v);
      }
      if (channel) {
        vec8(v, p.gate, p.gdt, 0.0f, w);
        act8(p.act, v);
        kept.put(k * slots + gate_at, v);
      }
    }
  }
  unsigned coming = first, to = all;
  auto fetch = [&]() {
    if (coming < rows) {
      PX::fetch(to + ox, row_at<TX>(p.x, coming, p.xs), w0);
      if (p.b) PT::fetch(to + ob, row_at<T>(p.b, coming, p.bs), w0);
      if (full) PT::fetch(to + og, row_at<T>(p.gate, coming, p.gs), w0);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    coming += step;
    to = to + hold.slot == end ? all : to + hold.slot;
  };
  if constexpr (VEC)  // columns that there are not read as 0
    for (unsigned j = all + threadIdx.x * 16; j < end; j += blockDim.x * 16) asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(j), "r"(0) : "memory");
  __syncthreads();
  for (int a = 0; a + 1 < ahead; ++a) fetch();
  unsigned here = all;
  for (unsigned r = first; r < rows; r += step) {
    turn_ring<VEC>(g, ahead, fetch);
    float y[PIECES][kE], t[1];
    float m2 = 0.0f, r2 = 1.0f;
    const T* brow = row_at<T>(p.b, r, p.bs);
    if (p.b && p.post) {
      if (kind == 1) {
        t[0] = 0.0f;
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
          float b[kE];
          PT::get(b, here + ob, brow, w0, k);
#pragma unroll
          for (int i = 0; i < kE; ++i) t[0] += b[i];
        }
        g.sum<1>(t);
        m2 = t[0] * inv;
      }
      t[0] = 0.0f;
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        float b[kE];
        PT::get(b, here + ob, brow, w0, k);
#pragma unroll
        for (int i = 0; i < kE; ++i) {
          if (kind == 1) b[i] = w0.piece(k).on(i) ? b[i] - m2 : 0.0f;
          t[0] += b[i] * b[i];
        }
      }
      g.sum<1>(t);
      r2 = rsqrtf(t[0] * inv + p.eps);
    }
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const Place<VEC> w = w0.piece(k);
      if (p.b) {
        float b[kE], v[kE];
        PT::get(b, here + ob, brow, w0, k);
        kept.get(k * slots, v);
        if (kind == 1) {
#pragma unroll
          for (int i = 0; i < kE; ++i) b[i] -= m2;
        }
#pragma unroll
        for (int i = 0; i < kE; ++i) b[i] = b[i] * r2 * v[i];
        if (p.c2) {
          kept.get(k * slots + 2, v);
#pragma unroll
          for (int i = 0; i < kE; ++i) b[i] += v[i];
        }
        if (p.gate) {
          if (channel) {
            kept.get(k * slots + gate_at, v);
          } else {
            if (full)
              PT::get(v, here + og, row_at<T>(p.gate, r, p.gs), w0, k);
            else
              vec8(v, gate_row(p.gate, p.gdt, p.gs, r), p.gdt, 0.0f, w);
            act8(p.act, v);
          }
#pragma unroll
          for (int i = 0; i < kE; ++i) b[i] *= v[i];
        }
        PX::get(y[k], here + ox, row_at<TX>(p.x, r, p.xs), w0, k);
        if (p.d.on) {
          unsigned u[kE];
          words8<VEC>(u, p.d, p.d.base + (u64)r * (unsigned)p.cols, w, places + hold.words);
#pragma unroll
          for (int i = 0; i < kE; ++i) y[k][i] += u[i] > p.d.last ? f * b[i] : 0.0f;
        } else {
#pragma unroll
          for (int i = 0; i < kE; ++i) y[k][i] += f * b[i];
        }
      } else {
        PX::get(y[k], here + ox, row_at<TX>(p.x, r, p.xs), w0, k);
      }
      if (p.y) store8<TX>(row_at<TX>(p.y, r, p.ys), y[k], w);
    }
    here = here + hold.slot == end ? all : here + hold.slot;
    if (!p.h) continue;
    float m1 = 0.0f;
    if (kind == 1) {
      t[0] = 0.0f;
#pragma unroll
      for (int k = 0; k < PIECES; ++k)
#pragma unroll
        for (int i = 0; i < kE; ++i)
          if (w0.piece(k).on(i)) t[0] += y[k][i];
      g.sum<1>(t);
      m1 = t[0] * inv;
    }
    t[0] = 0.0f;
#pragma unroll
    for (int k = 0; k < PIECES; ++k)
#pragma unroll
      for (int i = 0; i < kE; ++i) {
        if (kind == 1) y[k][i] -= m1;
        if (w0.piece(k).on(i)) t[0] += y[k][i] * y[k][i];
      }
    g.sum<1>(t);
    const float r1 = rsqrtf(t[0] * inv + p.eps);
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      float v[kE];
      kept.get(k * slots + 1, v);
#pragma unroll
      for (int i = 0; i < kE; ++i) y[k][i] = y[k][i] * r1 * v[i];
      if (p.c1) {
        kept.get(k * slots + c1_at, v);
#pragma unroll
        for (int i = 0; i < kE; ++i) y[k][i] += v[i];
      }
      store8<T>(row_at<T>(p.h, r, p.hs), y[k], w0.piece(k));
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// The gradient. MORE: also the sums of the biases' and of a channel gate's
// gradient. A row takes two sums over it (the statistics and the first norm's
// terms; the second norm's terms), three for the layer norm; between them the
// row is read again from the ring, piece by piece, which leaves registers for
// the sums over rows: they stay in them for all of a thread's rows.
template <class T, class TX, bool VEC, int PIECES, bool MORE>
__global__ void __launch_bounds__(512) norm_back_rows(const __grid_constant__ BackP p, int kind, const Hold hold) {
  __shared__ __align__(16) float s[16 * 8];
  extern __shared__ __align__(16) unsigned char places[];
  typedef Part<TX, VEC, PIECES> PX;
  typedef Part<T, VEC, PIECES> PT;
  const int tpr = hold.tpr, ahead = hold.ahead;
  Group g(s, tpr);
  const Place<VEC> w0 = {(int)threadIdx.x - g.id * tpr, tpr, (int)p.cols};
  const float inv = 1.0f / (float)p.cols, f = p.scale * p.d.factor;
  const bool channel = p.gate && p.gs == 0, full = p.gate && !channel && p.gdt != CCB_F32, norm2 = p.b && p.post;
  const unsigned sets = blockDim.x / tpr, first = blockIdx.x * sets + g.id, step = gridDim.x * sets, rows = (unsigned)p.rows;
  const unsigned all = (unsigned)__cvta_generic_to_shared(places), end = all + ahead * hold.slot;
  const unsigned nx = part_bytes<TX, VEC, PIECES>(p.cols, blockDim.x, tpr), nt = part_bytes<T, VEC, PIECES>(p.cols, blockDim.x, tpr);
  const unsigned oy = VEC ? threadIdx.x * 16 : g.id * (nx / sets), ody = oy + nx, odh = 2 * nx + (VEC ? threadIdx.x * 16 : g.id * (nt / sets)), ob = odh + nt,
                 og = ob + nt;
  float acc[MORE ? kVecs : 2][PIECES * kE];  // dw1, dw2, then dc1, dc2, dgate
#pragma unroll
  for (int v = 0; v < (MORE ? kVecs : 2); ++v)
#pragma unroll
    for (int i = 0; i < PIECES * kE; ++i) acc[v][i] = 0.0f;
  // kept, for each piece: w1, w2, then c2 and a channel gate's act, as far as there are any
  const Kept kept = {all + hold.kept + w0.t * 16, (unsigned)tpr * 16};
  const int gate_at = 2 + (p.c2 != nullptr), slots = gate_at + channel;
  if (g.id == 0) {
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const Place<VEC> w = w0.piece(k);
      float v[kE];
      vec8(v, p.w1, p.wdt, 1.0f, w);
      kept.put(k * slots, v);
      vec8(v, p.w2, p.wdt, 1.0f, w);
      kept.put(k * slots + 1, v);
      if (p.c2) {
        vec8(v, p.c2, p.wdt, 0.0f, w);
        kept.put(k * slots + 2, v);
      }
      if (channel) {
        vec8(v, p.gate, p.gdt, 0.0f, w);
        act8(p.act, v);
        kept.put(k * slots + gate_at, v);
      }
    }
  }
  unsigned coming = first, to = all;
  auto fetch = [&]() {
    if (coming < rows) {
      if (p.dh) {
        PX::fetch(to + oy, row_at<TX>(p.y, coming, p.ys), w0);
        PT::fetch(to + odh, row_at<T>(p.dh, coming, p.dhs), w0);
      }
      if (p.dy) PX::fetch(to + ody, row_at<TX>(p.dy, coming, p.dys), w0);
      if (p.b) PT::fetch(to + ob, row_at<T>(p.b, coming, p.bs), w0);
      if (full) PT::fetch(to + og, row_at<T>(p.gate, coming, p.gs), w0);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    coming += step;
    to = to + hold.slot == end ? all : to + hold.slot;
  };
  if constexpr (VEC)  // columns that there are not read as 0
    for (unsigned j = all + threadIdx.x * 16; j < end; j += blockDim.x * 16) asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(j), "r"(0) : "memory");
  __syncthreads();
  for (int a = 0; a + 1 < ahead; ++a) fetch();
  unsigned here = all;
  for (unsigned r = first; r < rows; r += step) {
    turn_ring<VEC>(g, ahead, fetch);
    // the row's parts, by piece
    auto get_y = [&](float* v, int k) { PX::get(v, here + oy, row_at<TX>(p.y, r, p.ys), w0, k); };
    auto get_dy = [&](float* v, int k) { PX::get(v, here + ody, row_at<TX>(p.dy, r, p.dys), w0, k); };
    auto get_dh = [&](float* v, int k) { PT::get(v, here + odh, row_at<T>(p.dh, r, p.dhs), w0, k); };
    auto get_b = [&](float* v, int k) { PT::get(v, here + ob, row_at<T>(p.b, r, p.bs), w0, k); };
    float m1 = 0.0f, f1 = 0.0f, m2 = 0.0f;
    if (kind == 1) {
      float t[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        float a[kE], b[kE];
        if (p.dh) {
          get_y(a, k);
#pragma unroll
          for (int i = 0; i < kE; ++i) t[0] += a[i];
          get_dh(a, k);
          kept.get(k * slots, b);
#pragma unroll
          for (int i = 0; i < kE; ++i) t[1] += a[i] * b[i];
        }
        if (norm2) {
          get_b(a, k);
#pragma unroll
          for (int i = 0; i < kE; ++i) t[2] += a[i];
        }
      }
      g.sum<3>(t);
      m1 = t[0] * inv;
      f1 = t[1] * inv;
      m2 = t[2] * inv;
    }
    float q[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const Place<VEC> w = w0.piece(k);
      float a[kE], b[kE], c[kE];
      if (p.dh) {
        get_y(a, k);
        get_dh(b, k);
        kept.get(k * slots, c);
#pragma unroll
        for (int i = 0; i < kE; ++i) {
          if (kind == 1) a[i] = w.on(i) ? a[i] - m1 : 0.0f;
          q[0] += a[i] * a[i];
          q[1] += b[i] * c[i] * a[i];
        }
      }
      if (norm2) {
        get_b(a, k);
#pragma unroll
        for (int i = 0; i < kE; ++i) {
          if (kind == 1) a[i] = w.on(i) ? a[i] - m2 : 0.0f;
          q[2] += a[i] * a[i];
        }
      }
    }
    g.sum<3>(q);
    const float r1 = rsqrtf(q[0] * inv + p.eps), a1 = q[1] * inv * r1, r2 = norm2 ? rsqrtf(q[2] * inv + p.eps) : 1.0f;
    float g2[PIECES][kE], t[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const Place<VEC> w = w0.piece(k);
      float d[kE], a[kE], b[kE], c[kE];
      if (p.dy)
        get_dy(d, k);
      else
#pragma unroll
        for (int i = 0; i < kE; ++i) d[i] = 0.0f;
      if (p.dh) {
        get_y(a, k);
        get_dh(b, k);
        kept.get(k * slots, c);
        if (kind == 1) {
#pragma unroll
          for (int i = 0; i < kE; ++i) a[i] = w.on(i) ? a[i] - m1 : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kE; ++i) {
          const float hat = a[i] * r1;
          d[i] += r1 * (b[i] * c[i] - hat * a1 - f1);
          acc[0][k * kE + i] += b[i] * hat;
          if (MORE) acc[2][k * kE + i] += b[i];
        }
      }
      if (p.dx) store8<TX>(row_at<TX>(p.dx, r, p.dxs), d, w);
      if (!p.b) continue;
      if (p.d.on) {
        unsigned u[kE];
        words8<VEC>(u, p.d, p.d.base + (u64)r * (unsigned)p.cols, w, places + hold.words);
#pragma unroll
        for (int i = 0; i < kE; ++i) d[i] = u[i] > p.d.last ? f * d[i] : 0.0f;  // dz
      } else {
#pragma unroll
        for (int i = 0; i < kE; ++i) d[i] *= f;
      }
      get_b(b, k);
      kept.get(k * slots + 1, c);
      if (kind == 1) {  // 0 - mean is not 0
#pragma unroll
        for (int i = 0; i < kE; ++i) {
          b[i] -= m2;
          if (!w.on(i)) b[i] = d[i] = 0.0f;
        }
      }
#pragma unroll
      for (int i = 0; i < kE; ++i) b[i] *= r2;  // hat
      if (p.gate) {
        if (channel) {
          kept.get(k * slots + gate_at, a);
        } else {
          if (full)
            PT::get(a, here + og, row_at<T>(p.gate, r, p.gs), w0, k);
          else
            vec8(a, gate_row(p.gate, p.gdt, p.gs, r), p.gdt, 0.0f, w);
          act8(p.act, a);
        }
        float u[kE];
        if (p.c2) {
          kept.get(k * slots + 2, u);
#pragma unroll
          for (int i = 0; i < kE; ++i) u[i] = d[i] * (b[i] * c[i] + u[i]);
        } else {
#pragma unroll
          for (int i = 0; i < kE; ++i) u[i] = d[i] * b[i] * c[i];
        }
        slope8(p.act, a, u);
#pragma unroll
        for (int i = 0; i < kE; ++i) {
          if (MORE) acc[4][k * kE + i] += u[i];
          d[i] *= a[i];  // du
        }
        if (p.dgate) {
          if (p.gdt == CCB_F32)
            store8<float>(row_at<float>(p.dgate, r, p.dgs), u, w);
          else
            store8<T>(row_at<T>(p.dgate, r, p.dgs), u, w);
        }
      }
#pragma unroll
      for (int i = 0; i < kE; ++i) {
        acc[1][k * kE + i] += d[i] * b[i];
        if (MORE) acc[3][k * kE + i] += d[i];
        g2[k][i] = d[i] * c[i];
        t[0] += g2[k][i] * b[i];
        if (kind == 1) t[1] += g2[k][i];
      }
    }
    if (p.db) {
      float a2 = 0.0f, f2 = 0.0f;
      if (p.post) {
        if (kind == 1)
          g.sum<2>(t);
        else
          g.sum<1>(t);
        a2 = t[0] * inv * r2 * r2;
        f2 = kind == 1 ? t[1] * inv * r2 : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        if (p.post) {
          float b[kE];
          get_b(b, k);
#pragma unroll
          for (int i = 0; i < kE; ++i) g2[k][i] = r2 * g2[k][i] - (b[i] - m2) * a2 - f2;
        }
        store8<T>(row_at<T>(p.db, r, p.dbs), g2[k], w0.piece(k));
      }
    }
    here = here + hold.slot == end ? all : here + hold.slot;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  // the block's partial sums: its groups', in order
  float* turn = reinterpret_cast<float*>(places);
#pragma unroll
  for (int a = 0; a < (MORE ? kVecs : 2); ++a) {
    const int v = a == 0 ? 0 : a == 1 ? 2 : a == 2 ? 1 : a;
    if (!p.vec[v]) continue;
    if (sets > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < PIECES * kE; ++i) turn[i * blockDim.x + threadIdx.x] = acc[a][i];
      __syncthreads();
      if (g.id == 0)
#pragma unroll
        for (int i = 0; i < PIECES * kE; ++i)
          for (int o = 1; o < (int)sets; ++o) acc[a][i] += turn[i * blockDim.x + o * tpr + threadIdx.x];
    }
    float* part = p.part + ((i64)blockIdx.x * kVecs + v) * p.cols;
    if (g.id == 0)
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        const Place<VEC> w = w0.piece(k);
#pragma unroll
        for (int i = 0; i < kE; ++i)
          if (w.on(i)) part[w.at(i)] = acc[a][k * kE + i];
      }
  }
}

// Column sums of the blocks' partials: a warp's 32 columns, 8 warps that each
// take every eighth block, their results added in order.
__global__ void __launch_bounds__(kBlock) norm_back_sum(const __grid_constant__ BackP p, int blocks) {
  __shared__ float s[kBlock];
  float* out = p.vec[blockIdx.y];
  if (!out) return;
  const i64 c = (i64)blockIdx.x * 32 + (threadIdx.x & 31);
  float t = 0.0f;
  if (c < p.cols)
    for (int i = threadIdx.x >> 5; i < blocks; i += kBlock / 32) t += p.part[((i64)i * kVecs + blockIdx.y) * p.cols + c];
  s[threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.x < 32 && c < p.cols) {
    for (int i = 1; i < kBlock / 32; ++i) t += s[32 * i + threadIdx.x];
    out[c] = t;
  }
}

constexpr i64 kBackBlocks = 296;  // most blocks (and partial sums) of the gradient; at least the SMs

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

// How rows are held, the block's threads (0: rows are too long) and its shared
// memory. `part(block, tpr)`: bytes of a slot of the ring; `vectors`: kept ones;
// `least`: bytes a thread needs at the end, in the same place. As many groups
// as 512 threads hold, fewer where their rows and the next ones do not fit.
struct Shape {
  Hold hold;
  int block, smem;
};
constexpr int kMostShared = 226 * 1024;
template <class P>
Shape shape_of(i64 cols, int pieces, bool vec, int vectors, int least, P part) {
  Shape f = {};
  const i64 tpr = (cols + pieces * kE * 32 - 1) / (pieces * kE * 32) * 32;
  if (tpr > 512) return f;
  f.hold.tpr = (int)tpr;
  const int kept = (int)tpr * pieces * kE * 4 * vectors;
  for (int want = 2; want >= 1 && !f.block; --want)
    for (int groups = 512 / (int)tpr; groups >= 1 && !f.block; --groups) {
      const int block = groups * (int)tpr, slot = (int)part(block, (int)tpr), words = vec ? 0 : block / 32 * kWarpWords * 4;
      const int ahead = (kMostShared - kept - words) / slot;
      if (ahead < want) continue;
      f.block = block;
      f.hold.ahead = ahead > 3 ? 3 : ahead;
      f.hold.slot = (unsigned)slot;
      f.hold.kept = (unsigned)(f.hold.ahead * slot);
      f.hold.words = f.hold.kept + (unsigned)kept;
      f.smem = (int)f.hold.words + words;
      if (f.smem < block * least) f.smem = block * least;
    }
  return f;
}
// Row strides that 32-bit products reach
bool near(std::initializer_list<i64> strides) {
  for (i64 t : strides)
    if (t >= (1ll << 30)) return false;
  return true;
}
// 16-byte accesses along every row
bool wide(i64 cols, std::initializer_list<const void*> ptrs, std::initializer_list<i64> strides) {
  if (cols % 8 != 0) return false;
  for (const void* q : ptrs)
    if (!aligned(q, 16)) return false;
  for (i64 t : strides)
    if (t % 8 != 0) return false;
  return true;
}
// Raises a kernel's shared-memory limit once for each device.
template <class K>
bool room_for(K* kernel, bool (&ready)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && __atomic_load_n(&ready[dev], __ATOMIC_RELAXED)) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared) != cudaSuccess) return false;
  if (dev >= 0 && dev < 64) __atomic_store_n(&ready[dev], true, __ATOMIC_RELAXED);
  return true;
}

template <class T, class TX, int KIND>
struct Forward {
  template <bool VEC, int PIECES>
  static bool rows(const NormP& p, int sms, cudaStream_t st) {
    static bool ready[64];
    const int matrices = (p.b != nullptr) + (p.gate && p.gs != 0 && p.gdt != CCB_F32);
    const Shape f = shape_of(p.cols, PIECES, VEC, 2 + (p.c1 != nullptr) + (p.c2 != nullptr) + (p.gate && p.gs == 0), 0, [&](int block, int tpr) {
      return part_bytes<TX, VEC, PIECES>(p.cols, block, tpr) + matrices * part_bytes<T, VEC, PIECES>(p.cols, block, tpr);
    });
    if (!f.block || !room_for(norm_rows<T, TX, VEC, PIECES>, ready)) return false;
    const i64 groups = f.block / f.hold.tpr, sets = (p.rows + groups - 1) / groups;
    norm_rows<T, TX, VEC, PIECES><<<(unsigned)(sets < sms ? sets : sms), f.block, f.smem, st>>>(p, KIND, f.hold);
    return true;
  }
  static bool by_width(const NormP& p, int sms, cudaStream_t st) {
    if (!near({p.xs, p.bs, p.gs, p.ys, p.hs})) return false;
    if (!wide(p.cols, {p.x, p.b, p.gate, p.y, p.h}, {p.xs, p.bs, p.gs, p.ys, p.hs})) return rows<false, 1>(p, sms, st);
    // What a thread does once a row (its sums, addresses, copies) is some 300
    // instructions: 32 elements share them, fewer where a warp holds the row.
    // The shape goes by the columns alone: a row's result does not depend on
    // the rows beside it.
    return p.cols <= 256 ? rows<true, 1>(p, sms, st) : p.cols <= 512 || (p.cols > 2048 && p.cols <= 4096) || sizeof(TX) == 4 ? rows<true, 2>(p, sms, st) : rows<true, 4>(p, sms, st);
  }
  static void run(const NormP& p, int sms, cudaStream_t st) {
    if (by_width(p, sms, st)) return;
    const i64 most = (i64)sms * 8;
    norm_any<T, TX, KIND><<<(unsigned)(p.rows < most ? p.rows : most), kBlock, 0, st>>>(p);
  }
};

template <class T, class TX, int KIND>
struct Backward {
  // The blocks of the launch, 0 if a row is too long.
  template <bool VEC, int PIECES, bool MORE>
  static int rows(const BackP& p, int sms, cudaStream_t st) {
    static bool ready[64];
    const Shape f = shape_of(p.cols, PIECES, VEC, 2 + (p.c2 != nullptr) + (p.gate && p.gs == 0), PIECES * kE * 4, [&](int block, int tpr) {
      return 2 * part_bytes<TX, VEC, PIECES>(p.cols, block, tpr) + 3 * part_bytes<T, VEC, PIECES>(p.cols, block, tpr);
    });
    if (!f.block || !room_for(norm_back_rows<T, TX, VEC, PIECES, MORE>, ready)) return 0;
    const i64 groups = f.block / f.hold.tpr, sets = (p.rows + groups - 1) / groups;
    const int most = sms < kBackBlocks ? sms : (int)kBackBlocks, grid = (int)(sets < most ? sets : most);
    norm_back_rows<T, TX, VEC, PIECES, MORE><<<grid, f.block, f.smem, st>>>(p, KIND, f.hold);
    return grid;
  }
  // Rows of 16 elements a thread, so that a block of 512 threads (128 registers
  // each) holds two of 4096 columns and one waits for its sums while the other
  // computes; of 8 where there are few columns. The shape does not go by the
  // rows or by which sums over them are asked for (all five spill some
  // registers), so that a row's results do not either.
  template <bool MORE>
  static int by_width(const BackP& p, int sms, cudaStream_t st) {
    if (!near({p.ys, p.dys, p.dhs, p.bs, p.gs, p.dxs, p.dbs, p.dgs})) return 0;
    if (!wide(p.cols, {p.y, p.dy, p.dh, p.b, p.gate, p.dx, p.db, p.dgate}, {p.ys, p.dys, p.dhs, p.bs, p.gs, p.dxs, p.dbs, p.dgs}))
      return rows<false, 1, MORE>(p, sms, st);
    if (p.cols <= 256 || (sizeof(TX) == 4 && p.cols <= 4096)) return rows<true, 1, MORE>(p, sms, st);
    return rows<true, 2, MORE>(p, sms, st);
  }
  static void run(const BackP& p, int sms, cudaStream_t st) {
    int grid = p.vec[1] || p.vec[3] || p.vec[4] ? by_width<true>(p, sms, st) : by_width<false>(p, sms, st);
    if (!grid) {
      grid = (int)(p.rows < kBackBlocks ? p.rows : kBackBlocks);
      norm_back_any<T, TX, KIND><<<grid, kBlock, 0, st>>>(p);
    }
    if (p.vec[0] || p.vec[1] || p.vec[2] || p.vec[3] || p.vec[4])
      norm_back_sum<<<dim3((unsigned)((p.cols + 31) / 32), kVecs), kBlock, 0, st>>>(p, grid);
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
                     a->weight_dtype, a->act, a->post_norm, make_drop(a->p, a->seed, a->offset, a->base, (u64)a->rows * (u64)a->cols)};
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
                     make_drop(a->p, a->seed, a->offset, a->base, (u64)a->rows * (u64)a->cols)};
    by_type<Backward>(a->dtype, a->x_dtype, a->kind, p, sms, st);
    return launched(me);
  })
}
