// Shared by ccb_nn_block_norm (nn_norm.cu) and its gradient (nn_norm_back.cu): the norm after a block, its gate,
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
#pragma once
#include <initializer_list>
#include <type_traits>

#include "nn_common.cuh"

namespace ccb_nn {
namespace {

constexpr int kBlock = 256;

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

// -------------------------------------------------------- rows read once
// A group of `tpr` threads (whole warps) holds a row, PIECES times 8 elements
// a thread, and copies the rows that come next into a ring in shared memory
// meanwhile (cp.async: no registers, and nothing waits for the loads). VEC
// (cols a multiple of 8; pointers and strides of 16 bytes): a thread's elements
// are consecutive, and it copies and reads its own alone, so that there is no
// barrier. Otherwise they are tpr apart, and the group copies the 16-byte
// pieces of memory that hold the row between its threads (the bytes before a
// row's first element in its first piece are read, inside the aligned 16 bytes
// that hold it, and not used; none are read past its last). A block holds
// blockDim.x / tpr rows at a time and takes every grid-th set.
constexpr int kE = 8;

template <class T>
constexpr int code_of = sizeof(T) == 4 ? CCB_F32 : std::is_same<T, __half>::value ? CCB_F16 : CCB_BF16;

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
  for (int j = 0; j < kE; ++j) v[j] = none;
  if (!p) return;
  if (dtype == CCB_F32) {  // the type is asked for once, so that the loads overlap
#pragma unroll
    for (int j = 0; j < kE; ++j)
      if (w.on(j)) v[j] = static_cast<const float*>(p)[w.at(j)];
  } else {
#pragma unroll
    for (int j = 0; j < kE; ++j)
      if (w.on(j)) v[j] = load_as(p, dtype, w.at(j));
  }
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
// Eight elements at a time by the packed F32 instructions: two results for the
// issue slot of one, and issue slots are what bounds these loops.
__device__ __forceinline__ void fma2(float* o, float a0, float a1, float b0, float b1, float c0, float c1) {
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(o[0]), "=f"(o[1])
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mul2(float* o, float a0, float a1, float b0, float b1) {
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}\n"
      : "=f"(o[0]), "=f"(o[1])
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
// o = a * b, a * s, a * b + c, a * s + c, and s += a . b in two halves
__device__ __forceinline__ void mul8(float* o, const float* a, const float* b) {
#pragma unroll
  for (int i = 0; i < kE; i += 2) mul2(o + i, a[i], a[i + 1], b[i], b[i + 1]);
}
__device__ __forceinline__ void mul8(float* o, const float* a, float s) {
#pragma unroll
  for (int i = 0; i < kE; i += 2) mul2(o + i, a[i], a[i + 1], s, s);
}
__device__ __forceinline__ void fma8(float* o, const float* a, const float* b, const float* c) {
#pragma unroll
  for (int i = 0; i < kE; i += 2) fma2(o + i, a[i], a[i + 1], b[i], b[i + 1], c[i], c[i + 1]);
}
__device__ __forceinline__ void fma8(float* o, const float* a, float s, const float* c) {
#pragma unroll
  for (int i = 0; i < kE; i += 2) fma2(o + i, a[i], a[i + 1], s, s, c[i], c[i + 1]);
}
__device__ __forceinline__ void dot8(float* s, const float* a, const float* b) {
#pragma unroll
  for (int i = 0; i < kE; i += 2) fma2(s, a[i], a[i + 1], b[i], b[i + 1], s[0], s[1]);
}

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
// e0 (d.same, and a multiple of 4 with VEC). Consecutive elements: two of its
// blocks. Single ones: a warp's 32 elements of one step lie in at
// most 9 blocks, so the warp computes the 72 of all steps between its lanes
// and hands the words out through its part of shared memory.
constexpr int kWarpWords = 9 * kE * 4;
template <bool VEC>
__device__ __forceinline__ void words8(unsigned* u, const Drop& d, u64 e0, const Place<VEC>& w, unsigned char* places) {
  if constexpr (VEC) {
    philox<2, true>(d, (e0 + (u64)w.at(0)) >> 2, u);
  } else {
    uint4* out = reinterpret_cast<uint4*>(places) + (threadIdx.x >> 5) * (kWarpWords / 4);
    const int lane = threadIdx.x & 31;
    const u64 e = e0 + (u64)(w.t - lane);  // the warp's first element of step 0
    __syncwarp();
    for (int b = lane; b < 9 * kE; b += 32) {
      const int i = b / 9;
      unsigned x[4];
      philox<1, true>(d, ((e + (u64)(i * w.tpr)) >> 2) + (u64)(b - 9 * i), x);
      out[b] = make_uint4(x[0], x[1], x[2], x[3]);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kE; ++i) u[i] = reinterpret_cast<const unsigned*>(out)[36 * i + (int)((e + (u64)(i * w.tpr)) & 3) + lane];
  }
}

// act(g) from the hardware's exponential and reciprocal. The sigmoid's 2^t, t =
// -g log2(e), has the relative error of t's rounding, |t| 2^-24: below that of
// any 16-bit gate, but 3e-6 of an F32 gate's at -80. FINE takes t's rounding and
// log2(e)'s along and is within ten units of 2^-24 everywhere (its gates are cut
// to +-88, where the sigmoid is 1 or below the least normal number).
template <bool FINE>
__device__ __forceinline__ void act8(int act, float* g) {
  if (act == 1 && FINE) {
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      float x = -g[i], e;
      asm("max.NaN.f32 %0, %0, 0fC2B00000;\n\tmin.NaN.f32 %0, %0, 0f42B00000;" : "+f"(x));  // -88, 88
      const float t = x * 1.44269502f, rest = fmaf(x, 1.44269502f, -t) + x * 1.92596303e-8f;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
      e = fmaf(e, rest * 0.693147181f, e);
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(g[i]) : "f"(1.0f + e));
    }
  } else if (act == 1) {
#pragma unroll
    for (int i = 0; i < kE; i += 2) {
      float e[2];
      mul2(e, g[i], g[i + 1], -1.4426950408889634f, -1.4426950408889634f);
      asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e[0]));
      asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e[1]));
      fma2(e, e[0], e[1], 1.0f, 1.0f, 1.0f, 1.0f);
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(g[i]) : "f"(e[0]));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(g[i + 1]) : "f"(e[1]));
    }
  } else if (act == 2) {  // 1 - 2 / (1 + e^2g); below 0.55, where that cancels, the series to x^13 (3e-7 at its end)
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      const float x = g[i], t = x * x;
      float p = 21844.0f / 6081075.0f;
      p = fmaf(p, t, -1382.0f / 155925.0f);
      p = fmaf(p, t, 62.0f / 2835.0f);
      p = fmaf(p, t, -17.0f / 315.0f);
      p = fmaf(p, t, 2.0f / 15.0f);
      p = fmaf(p, t, -1.0f / 3.0f);
      p = fmaf(p * t, x, x);
      float e, r;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * 2.8853900817779268f));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
      g[i] = fabsf(x) < 0.55f ? p : fmaf(-2.0f, r, 1.0f);
    }
  }
}
// act'(g) times v, from a = act(g)
__device__ __forceinline__ void slope8(int act, const float* a, float* v) {
  if (act == 0) return;
  float t[kE];
#pragma unroll
  for (int i = 0; i < kE; i += 2) {
    if (act == 1) {
      fma2(t + i, a[i], a[i + 1], -1.0f, -1.0f, 1.0f, 1.0f);
      mul2(t + i, t[i], t[i + 1], a[i], a[i + 1]);
    } else {
      fma2(t + i, -a[i], -a[i + 1], a[i], a[i + 1], 1.0f, 1.0f);
    }
  }
  mul8(v, v, t);
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

// The element types a call may have: dtype, and the residual stream in it or in
// f32. The f16 ones by themselves, for a file of their own.
#define CCB_NN_CASE(dt, xdt, T, TX)         \
  if (dtype == dt && x_dtype == xdt) {      \
    if (kind == 0)                          \
      Go<T, TX, 0>::run(a...);              \
    else                                    \
      Go<T, TX, 1>::run(a...);              \
    return;                                 \
  }
template <template <class, class, int> class Go, class... A>
void by_f16(int dtype, int x_dtype, int kind, A... a) {
  CCB_NN_CASE(CCB_F16, CCB_F16, __half, __half)
  CCB_NN_CASE(CCB_F16, CCB_F32, __half, float)
}
template <template <class, class, int> class Go, class... A>
void by_type_but_f16(int dtype, int x_dtype, int kind, A... a) {
  CCB_NN_CASE(CCB_F32, CCB_F32, float, float)
  CCB_NN_CASE(CCB_BF16, CCB_BF16, __nv_bfloat16, __nv_bfloat16)
  CCB_NN_CASE(CCB_BF16, CCB_F32, __nv_bfloat16, float)
}
#undef CCB_NN_CASE

// How rows are held, the block's threads (0: rows are too long) and its shared
// memory. `part(block, tpr)`: bytes of a slot of the ring; `vectors`: kept ones;
// `least`: bytes a thread needs at the end, in the same place. As many groups
// as `threads` hold, fewer where their rows and the next ones do not fit.
struct Shape {
  Hold hold;
  int block, smem;
};
constexpr int kMostShared = 226 * 1024;
template <class P>
Shape shape_of(i64 cols, int pieces, int threads, bool vec, int vectors, int least, P part) {
  Shape f = {};
  const i64 tpr = (cols + pieces * kE * 32 - 1) / (pieces * kE * 32) * 32;
  if (tpr > threads) return f;
  f.hold.tpr = (int)tpr;
  const int kept = (int)tpr * pieces * kE * 4 * vectors;
  for (int want = 2; want >= 1 && !f.block; --want)
    for (int groups = threads / (int)tpr; groups >= 1 && !f.block; --groups) {
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
