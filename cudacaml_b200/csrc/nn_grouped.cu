// ccb_nn_grouped_matmul and ccb_nn_grouped_matmul_dw: products grouped by
// expert. The row ranges of the experts live in device memory, so every block
// lays the tiles out for itself: it clamps the offsets, counts the row tiles
// of each segment and scans the counts in shared memory.
#include <type_traits>

#include "ccb_skel.cuh"
#include "dyn.hpp"
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

// ------------------------------------------------- nothing to contract over
// Zeros, and the offsets' check.
template <class T>
__global__ void __launch_bounds__(256) clear_out(T* out, i64 mats, i64 rows, i64 cols, i64 oe, i64 os, const int* off, int experts, int tokens, unsigned* err) {
  __shared__ Segments g;
  if (blockIdx.x == 0) lay_out(g, off, experts, tokens, 256, err);
  const i64 each = rows * cols;
  for (i64 i = (i64)blockIdx.x * 256 + threadIdx.x; i < mats * each; i += (i64)gridDim.x * 256) {
    const i64 m = i / each, r = (i - m * each) / cols;
    out[m * oe + r * os + (i - m * each - r * cols)] = from_f<T>(0.0f);
  }
}
int clear(int dtype, void* out, i64 mats, i64 rows, i64 cols, i64 oe, i64 os, const int* off, i64 experts, i64 tokens, unsigned* err, int sms, cudaStream_t st,
          const char* me) {
  const i64 work = (mats * rows * cols + 255) / 256, most = (i64)sms * 8;
  const unsigned grid = (unsigned)(work < most ? work : most);
  if (dtype == CCB_F32)
    clear_out<<<grid, 256, 0, st>>>(static_cast<float*>(out), mats, rows, cols, oe, os, off, (int)experts, (int)tokens, err);
  else  // the two 16-bit zeros are the same
    clear_out<<<grid, 256, 0, st>>>(static_cast<__half*>(out), mats, rows, cols, oe, os, off, (int)experts, (int)tokens, err);
  return launched(me);
}

// ------------------------------------- CUDA cores, few rows an expert, any alignment
// Bound by reading the matrices of the experts that have rows (64 rows over 50
// of 64 experts of 1024 x 2048 f32: 96 us, 4.4 TB/s; transposed 127 us, 3.3
// TB/s; 64 x 64 tiles before it left most SMs idle: 445 us for 32 rows over 12
// experts of 2048 x 1024, 38 us now; 64 rows over 50 of 64 of 1023 x 2047 bf16
// 82 us, 2.6 TB/s by single elements): a block takes up
// to 8 rows of one expert, a block of output columns and a part of the
// contraction, keeps the rows' values in shared memory and reads every weight
// once, in order. Parts are summed by add_parts, so that the SMs are filled
// whatever the shape.
constexpr int kFewRows = 8, kFewCols = 512, kFewColsT = 64, kFewK = 1024, kFewThreads = 128;

struct FewP {
  GroupP g;
  int splits;
  i64 split_stride, part;  // elements between parts' results, of the contraction in a part
};

template <class T, class TO, bool WT>
__global__ void __launch_bounds__(kFewThreads) grouped_few(const __grid_constant__ FewP q) {
  __shared__ Segments g;
  __shared__ __align__(16) float xs[kFewRows * kFewK];  // [k][row], or [row][k] for a transposed w
  const GroupP& p = q.g;
  lay_out(g, p.off, p.experts, p.rows, kFewRows, p.err);
  const int segs = p.experts + 2;
  const i64 nc = (p.n + (WT ? kFewColsT : kFewCols) - 1) / (WT ? kFewColsT : kFewCols), total = nc * q.splits * g.tile[segs];
  const T* x = static_cast<const T*>(p.x);
  for (i64 t = blockIdx.x; t < total; t += gridDim.x) {
    const int split = (int)(t / nc % q.splits), mt = (int)(t / nc / q.splits), s = segment_of(g, segs, mt);
    const int r0 = g.row[s] + (mt - g.tile[s]) * kFewRows, rows = min(g.row[s + 1] - r0, kFewRows);
    const bool real = s >= 1 && s <= p.experts;
    const i64 n0 = (t % nc) * (WT ? kFewColsT : kFewCols), k0 = split * q.part, k1 = real ? min(p.k, k0 + q.part) : k0;
    const T* w = static_cast<const T*>(p.w) + (real ? (s - 1) * p.we : 0);
    TO* out = static_cast<TO*>(p.out) + split * q.split_stride;
    float acc[4][kFewRows] = {};
    // the rows' values, and 0 to the end of the last step
    const int kn = (int)(k1 - k0), kz = WT ? (kn + 255) & ~255 : (kn + 7) & ~7;
    __syncthreads();
#pragma unroll 8
    for (int i = threadIdx.x; i < kFewRows * kz; i += kFewThreads) {
      const int r = i / kz, k = i - r * kz;
      xs[WT ? r * kFewK + k : k * kFewRows + r] = r < rows && k < kn ? to_f<T>(x[(i64)(r0 + r) * p.xs + k0 + k]) : 0.0f;
    }
    __syncthreads();
    // 16 weights in hand and the next 16 on their way; of 16-bit ones twice as many
    constexpr int kStep = sizeof(T) == 4 ? 4 : 8;
    float v[kStep][4];
    T u[kStep][4];  // as read: a conversion in the fetch would wait for its load
    const T none = from_f<T>(0.0f);
    if constexpr (!WT) {
      bool on[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) on[j] = n0 + threadIdx.x + j * kFewThreads < p.n;
      const T* at = w + k0 * p.ws + n0 + threadIdx.x;
      auto fetch = [&](T (*to)[4], int k) {
#pragma unroll
        for (int i = 0; i < kStep; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) to[i][j] = on[j] && k + i < kn ? at[(k + i) * p.ws + j * kFewThreads] : none;
      };
      fetch(u, 0);
      for (int k = 0; k < kn; k += kStep) {
#pragma unroll
        for (int i = 0; i < 4 * kStep; ++i) v[i >> 2][i & 3] = to_f<T>(u[i >> 2][i & 3]);
        fetch(u, k + kStep);
#pragma unroll
        for (int i = 0; i < kStep; ++i) {
          const float4 a = *reinterpret_cast<const float4*>(xs + (k + i) * kFewRows), b = *reinterpret_cast<const float4*>(xs + (k + i) * kFewRows + 4);
          const float xv[kFewRows] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) acc[j][r] = fmaf(xv[r], v[i][j], acc[j][r]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const i64 c = n0 + threadIdx.x + j * kFewThreads;
        if (c >= p.n) continue;
#pragma unroll
        for (int r = 0; r < kFewRows; ++r)
          if (r < rows) out[(i64)(r0 + r) * p.os + c] = from_f<TO>(acc[j][r]);
      }
    } else {
      const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
      for (int c0 = warp * 4; c0 < kFewColsT && n0 + c0 < p.n; c0 += kFewThreads / 32 * 4) {
        const T* at[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          at[j] = w + min(n0 + c0 + j, p.n - 1) * p.ws + k0;  // a column too many repeats the last
#pragma unroll
          for (int r = 0; r < kFewRows; ++r) acc[j][r] = 0.0f;
        }
        auto fetch = [&](T (*to)[4], int k) {
#pragma unroll
          for (int i = 0; i < kStep; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) to[i][j] = k + 32 * i < kn ? at[j][k + 32 * i] : none;
        };
        fetch(u, lane);
        for (int k = lane; k < kz; k += 32 * kStep) {
#pragma unroll
          for (int i = 0; i < 4 * kStep; ++i) v[i >> 2][i & 3] = to_f<T>(u[i >> 2][i & 3]);
          fetch(u, k + 32 * kStep);
#pragma unroll
          for (int i = 0; i < kStep; ++i) {
            float xv[kFewRows];
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) xv[r] = xs[r * kFewK + k + 32 * i];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int r = 0; r < kFewRows; ++r) acc[j][r] = fmaf(xv[r], v[i][j], acc[j][r]);
          }
        }
        // the warp's 32 sums, halved from step to step: lane 8 j + r ends with column j of row r
        float* a = &acc[0][0];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
          for (int i = 0; i < o; ++i) {
            const float give = lane & o ? a[i] : a[i + o], keep = lane & o ? a[i + o] : a[i];
            a[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
          }
        const int r = lane & 7;
        const i64 c = n0 + c0 + (lane >> 3);
        if (r < rows && c < p.n) out[(i64)(r0 + r) * p.os + c] = from_f<TO>(a[0]);
      }
    }
  }
}

template <class T, class TO>
void few(const FewP& q, bool wt, int sms, cudaStream_t st) {
  const i64 cols = wt ? kFewColsT : kFewCols, tiles = (q.g.rows / kFewRows + q.g.experts + 2) * ((q.g.n + cols - 1) / cols) * q.splits, most = (i64)sms * 5;
  const unsigned grid = (unsigned)(tiles < most ? tiles : most);
  if (wt)
    grouped_few<T, TO, true><<<grid, kFewThreads, 0, st>>>(q);
  else
    grouped_few<T, TO, false><<<grid, kFewThreads, 0, st>>>(q);
}

// ------------------------------------------------------------ tensor cores
// One kernel for the three products, on pairs of SMs (cta_group::2). The MMA's
// 256-high M side holds output features (a weight's columns, or dy's), its N
// side the ragged dimension: the tokens of one expert, or x's columns for dw.
// So a short range costs what it holds (N is any multiple of 32), the pair's
// accumulators have consecutive features in consecutive TMEM lanes, and a
// warp's stores of one token are contiguous without a transpose.
//
// Warps of each CTA: 0 TMA producer (a ring of 6 stages, 64 of the contraction
// each: 128 features of the M side and half of the N side), 1 MMA issuer (of
// the even CTA, for both), 2-9 drain one of two accumulators while the other
// fills, 10 (dw) clears the rows past an expert's end: the contraction runs
// over rows there, so what the next expert holds must not reach the sum. Both
// CTAs' copies complete on the even CTA's barrier; copies whose rows have to
// be cleared complete on the CTA's own, and warp 10 passes them on.
//
// Every tile is dealt out round-robin; a segment's rows are cut evenly, so
// that no tile is a short remainder. Why pairs and 256 x 256: a step of 64 moves
// 32 KiB into each SM for 512 cycles of its tensor pipe, and L2 feeds some 10
// TB/s. Measured on one B200: one group of 8192 x 8192 x 4096 bf16 334-366 us
// (1500-1645 TFLOP/s; bound by power, the clock falls to 1.6 GHz), 16384 rows
// over 16 experts of 4096 x 4096 375-405 us, one row for each of 64 experts of
// 2048 x 2048 81 us (6.6 TB/s, bound by HBM), the gradient of 64 experts'
// 4096 x 1024 from 32 rows 103-116 us (4.6-5.2 TB/s, bound by its writes).
namespace tcg {
constexpr int kFeat = 256, kTok = 256, kBK = 64, kStages = 6;
constexpr unsigned kABytes = 128 * kBK * 2, kBBytes = 128 * kBK * 2, kStageBytes = kABytes + kBBytes;
constexpr unsigned kTmemCols = 512;
constexpr int kDrain = 8, kThreads = 32 * (3 + kDrain);  // draining warps; all
constexpr unsigned kErrWait = 16u;

struct Tail {  // after the ring
  ccb::u64 full[kStages], empty[kStages], part[kStages], accf[2], acce[2], done;
  unsigned tmem;
  unsigned stop;         // a wait ran out in either CTA: nothing more is issued
  unsigned issued;       // stages that the producer has filled or begun to
  alignas(128) unsigned char out[kDrain][2048];  // a draining warp's 32 tokens x 32 features
  Segments g;
};
constexpr unsigned kSmem = kStages * kStageBytes + sizeof(Tail) + 1024;
static_assert(kSmem <= 232448, "shared memory of a block");

// Elements of f32 operands: expert e, step k of the contraction, feature f or
// token (column of x, for dw) t, in units of elements.
struct Plain {
  const float *m, *n;
  i64 me, mk, mf, nk, nt;
};

struct P {
  ccb::TmaDesc ta, tb;  // M side, N side
  const int* off;
  void* out;
  unsigned* err;
  i64 os, oe;           // strides of out: a row, an expert's matrix (dw)
  i64 split_stride;     // elements from one part's result to the next
  int rows, experts, n, k, splits, format;
  int a2, b2;           // whether one copy takes two 64-wide blocks of an MN-major operand
  int vec;              // out takes 16-byte stores
  unsigned polls;       // of a wait, before it gives up
  Plain plain;          // f32 operands as the caller gave them
};

// Barriers and tiles are addressed by 32-bit shared addresses throughout: one
// thread issues the copies and one the MMAs, at some five cycles an
// instruction, so every instruction of their loops counts (a step of the
// contraction is 512 cycles of the tensor pipe).
__device__ __forceinline__ bool try_wait(unsigned bar, unsigned parity) {
  unsigned ok;
  asm volatile("{\n .reg .pred q;\n mbarrier.try_wait.parity.shared::cta.b64 q, [%1], %2;\n selp.u32 %0, 1, 0, q;\n}\n"
               : "=r"(ok)
               : "r"(bar), "r"(parity)
               : "memory");
  return ok != 0;
}
// A wait of a whole warp: true once the phase is over. It is bounded: when it
// has run out it raises the error bit and both CTAs' stop flags, which every
// wait of either CTA looks at while it polls, and from then on each role ends at
// its next wait that is not already over, without another copy, MMA, commit or
// arrival; what is on its way by then is waited for at the kernel's end. A false
// return is the same for all lanes.
struct Waiter {
  unsigned stop, peer_stop, polls;  // shared addresses of the flags
  unsigned* err;
  __device__ __forceinline__ bool operator()(unsigned bar, unsigned parity) const {
    if (__all_sync(0xffffffffu, try_wait(bar, parity))) return true;
    for (unsigned it = 1; it < polls; ++it) {
      if (__all_sync(0xffffffffu, try_wait(bar, parity))) return true;
      unsigned flag;
      asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(flag) : "r"(stop) : "memory");
      if (__any_sync(0xffffffffu, flag != 0)) return false;
    }
    if ((threadIdx.x & 31) == 0) {
      if (err) atomicOr(err, kErrWait);
      asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(stop), "r"(1) : "memory");
      asm volatile("st.relaxed.cluster.shared::cluster.u32 [%0], %1;" ::"r"(peer_stop), "r"(1) : "memory");
    }
    __syncwarp();
    return false;
  }
};
// The same after a stop, for what was issued before it and ends by itself.
__device__ __forceinline__ void wait_out(unsigned bar, unsigned parity) {
  for (unsigned it = 0; it < ccb::MBAR_SPIN_LIMIT; ++it)
    if (try_wait(bar, parity)) return;
}
__device__ __forceinline__ void expect(unsigned bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Arrivals on a barrier of either CTA. A release at cluster scope waits until
// every earlier store of the thread, those to `out` too, has been performed,
// some 3 us under load, so none is asked for where nothing in memory is handed
// over: the other CTA's producer says how many bytes its copies bring (which the
// barrier counts itself), a draining warp that its loads from the accumulator are
// done (they are: tcgen05.wait::ld). The clearing warp hands over its own CTA's
// shared memory, to the CTA's own tensor core, and its proxy fence has already
// made that visible (a release at cluster scope there: the gradient of 30
// experts' 4096 x 1024 from 8192 rows 113 us instead of 95).
__device__ __forceinline__ void arrive(unsigned bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void expect_relaxed(unsigned bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void arrive_relaxed(unsigned bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void commit(unsigned bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void load4(unsigned dst, const ccb::TmaDesc* map, int x, int y, int z, int w, unsigned bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"((unsigned long long)map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void mma(unsigned d, ccb::u64 a, ccb::u64 b, unsigned idesc, unsigned accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
               "r"(accumulate)
               : "memory");
}
// A word of the other CTA's shared memory.
__device__ __forceinline__ unsigned peer_word(const unsigned* local, unsigned rank) {
  unsigned v;
  asm volatile("ld.volatile.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(ccb::tc2::peer_addr(local, rank)) : "memory");
  return v;
}
// Operand descriptors of 16-bit tiles with the 128-byte swizzle. K-major:
// 128-byte rows of 64 along the contraction, 8-row groups 1024 bytes apart, 16
// of the contraction 32 bytes further. MN-major: 64 along M or N are one
// 128-byte row, one row for each step of the contraction, 8-row groups 1024
// bytes apart, the next 64 along M or N 8192 bytes on, 16 of the contraction
// 2048 bytes further. The start address is in units of 16 bytes.
template <bool MN>
__device__ __forceinline__ ccb::u64 desc(unsigned tile) {
  return ccb::tc::sdesc(tile, MN ? 8192u : 16u, 1024u, ccb::tc::LAYOUT_SW128);
}
template <bool MN>
__device__ __forceinline__ constexpr unsigned desc_step() { return (MN ? 2048u : 32u) >> 4; }

// 32 lanes x 32 columns of the accumulator in the fragments of 8x8 matrices:
// v[16 h + 4 j + 2 i + b] is feature 16 h + 8 i + lane / 4, token 8 j + 2 (lane % 4) + b.
__device__ __forceinline__ void load_fragments(unsigned taddr, unsigned* v) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[16 * h]), "=r"(v[16 * h + 1]), "=r"(v[16 * h + 2]), "=r"(v[16 * h + 3]), "=r"(v[16 * h + 4]), "=r"(v[16 * h + 5]),
                   "=r"(v[16 * h + 6]), "=r"(v[16 * h + 7]), "=r"(v[16 * h + 8]), "=r"(v[16 * h + 9]), "=r"(v[16 * h + 10]), "=r"(v[16 * h + 11]),
                   "=r"(v[16 * h + 12]), "=r"(v[16 * h + 13]), "=r"(v[16 * h + 14]), "=r"(v[16 * h + 15])
                 : "r"(taddr + ((unsigned)(16 * h) << 16)));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// A warp's 32 features x 32 tokens to `out` (its first feature and token), in
// 16 bits: turned through shared memory so that a lane stores 16 bytes of one
// token (four packed transposing stores of 8x8 matrices; 64-byte rows, their
// 16-byte pieces swapped by row pair against bank conflicts). Written in
// phases, each of independent instructions: a warp alone on its scheduler pays
// every latency.
template <class TO>
__device__ __forceinline__ void drain16(unsigned taddr, bool zero, unsigned buf, TO* out, i64 os, int tokens, int feats, bool vec, int lane) {
  unsigned v[32], h[16];
  if (zero) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = 0;
  } else {
    load_fragments(taddr, v);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) h[i] = pack2<TO>(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
  // token 8 j + lane % 8, piece lane / 8: the swap depends on the lane alone
  const unsigned put = buf + (lane & 7) * 64 + (((lane >> 3) ^ ((lane >> 1) & 3)) << 4);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(put + j * 512), "r"(h[2 * j]), "r"(h[2 * j + 1]),
                 "r"(h[8 + 2 * j]), "r"(h[8 + 2 * j + 1])
                 : "memory");
  __syncwarp();
  if (vec && feats >= 8) {
    // token 8 j + lane / 4, piece lane % 4
    const unsigned get = buf + (lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) << 4);
    uint4 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[j].x), "=r"(w[j].y), "=r"(w[j].z), "=r"(w[j].w) : "r"(get + j * 512) : "memory");
    const int f = (lane & 3) * 8, tok = lane >> 2;
    TO* dst = out + tok * os + f;
    if (tokens >= 32 && feats >= 32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(dst + 8 * j * os) = w[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (8 * j + tok < tokens && f + 8 <= feats) *reinterpret_cast<uint4*>(dst + 8 * j * os) = w[j];
    }
  }
  // what is left of unaligned rows and of the last features: lane by lane
  const int done = vec ? feats & ~7 : 0;
  if (done < feats && done < 32) {
    const bool on = lane >= done && lane < feats;
    TO* dst = out + lane;
#pragma unroll 8
    for (int t = 0; t < 32; ++t) {
      unsigned short h;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(buf + t * 64 + (((lane >> 3) ^ ((t >> 1) & 3)) << 4) + (lane & 7) * 2) : "memory");
      if (on && t < tokens) *reinterpret_cast<unsigned short*>(dst + t * os) = h;
    }
  }
  __syncwarp();
}
template <class TO>
__device__ __forceinline__ void store32(const float* v, TO* out, i64 os, int tokens, int feats, int lane) {
  if (lane >= feats) return;
  TO* dst = out + lane;
  if (tokens >= 32) {
#pragma unroll
    for (int i = 0; i < 32; ++i) dst[i * os] = v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < tokens) dst[i * os] = v[i];
  }
}
// A result of f32 operands that came out as NaN, from the operands themselves:
// an infinite operand times a plane of the other that is 0 is NaN, also where
// that operand is not 0. In F32, eight steps at a time up to a NaN that is one:
// a few loads where NaN is everywhere, some K / 10 us where a row of x holds one
// infinity (the other roles' waits last 16 s).
__device__ __noinline__ float again(const Plain& q, int e, i64 k0, i64 k1, i64 f, i64 t) {
  const float *m = q.m + e * q.me + f * q.mf, *n = q.n + t * q.nt;
  float s = 0.0f;
  for (i64 k = k0; k < k1 && s == s; k += 8) {
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = k + i < k1 ? m[(k + i) * q.mk] : 0.0f;
      b[i] = k + i < k1 ? n[(k + i) * q.nk] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(a[i], b[i], s);
  }
  return s;
}
// The same in 32 bits: lanes are features, a store is one token's 128 bytes.
__device__ __forceinline__ void drain32(unsigned taddr, bool zero, float* out, i64 os, int tokens, int feats, int lane) {
  float v[32];
  if (zero) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = 0.0f;
  } else {
    ccb::tc::ld32(taddr, v);
  }
  store32(v, out, os, tokens, feats, lane);
}

// One thread of a converged warp. The loops that issue copies and MMAs are run
// by whole warps and only the instructions themselves by the elected thread:
// with one lane in the loop the compiler cannot keep descriptors, barriers and
// counters in uniform registers (a step's MMAs and commits took 407 cycles so,
// 157 this way; a 256 x 256 x 64 step is 512 cycles of the tensor pipe).
__device__ __forceinline__ bool elect_one() {
  unsigned ok;
  asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(ok));
  return ok != 0;
}

struct Tile {
  int expert;      // -1: rows of no expert
  int r0, r1;      // rows: of the result (forward), of the contraction (dw)
  int f0, c0;      // first feature; first column of x (dw)
  int nn;          // N of the MMA
  int b0, b1;      // steps of the contraction
  int split;
};
// f32 operands are sums hi + mid + lo of three 16-bit planes (WIDE), and a
// product is the six of their products down to 2^-16 of the largest, added up
// from the smallest.
//
// The accumulator truncates. Over a contraction of one sign that is a bias, of
// about 2^-23.4 of the sum so far for each MMA of bf16 and 2^-22.2 of f16: 8e-5
// and 1e-4 after 16384. Where the result is F32 and a contraction may be long
// (w's gradient; f32 operands), it is cut into chunks, each summed from 0 (in
// its six terms), and the draining warps add the chunks up in registers,
// rounding to nearest. Reading an accumulator takes some 370 cycles from the
// MMAs (their operands and it share tensor memory): one expert's 4096 x 4096 from
// 16384 rows takes 368 us in one go, 387 by chunks of 8 steps (512 rows), 412 of
// 4; the six terms of an f32 step make a chunk long enough at 4.
enum { kWhole = 0, kChunk = 8, kChunkWide = 4 };
template <int CHUNK>
__device__ __forceinline__ int chunk_end(int a, int b1) { return CHUNK ? min(a + CHUNK, b1) : b1; }
template <bool WIDE>
__device__ __forceinline__ constexpr int terms() { return WIDE ? 6 : 1; }
// The planes of a term.
template <bool WIDE>
__device__ __forceinline__ int plane_m(int term) { return WIDE ? (0x001102 >> (4 * term)) & 15 : 0; }
template <bool WIDE>
__device__ __forceinline__ int plane_n(int term) { return WIDE ? (0x010120 >> (4 * term)) & 15 : 0; }
enum { kForward = 0, kForwardT = 1, kDw = 2 };

template <int MODE>
__device__ __forceinline__ unsigned tiles_of(const P& p, const Segments& g) {
  const unsigned nf = (p.n + kFeat - 1) / kFeat;
  if (MODE == kDw) return nf * ((p.k + kTok - 1) / kTok) * p.experts * p.splits;
  return nf * g.tile[p.experts + 2] * p.splits;
}
// Tile t: features innermost, then the parts of the contraction, then tokens:
// the pairs work on one expert's matrix at a time, which stays in L2.
template <int MODE>
__device__ __forceinline__ Tile tile_at(const P& p, const Segments& g, unsigned t) {
  Tile o;
  const unsigned nf = (p.n + kFeat - 1) / kFeat;
  o.f0 = (int)(t % nf) * kFeat;
  t /= nf;
  o.split = (int)(t % (unsigned)p.splits);
  t /= (unsigned)p.splits;
  int steps;
  if (MODE == kDw) {
    const unsigned nc = (p.k + kTok - 1) / kTok;
    o.c0 = (int)(t % nc) * kTok;
    o.expert = (int)(t / nc);
    o.r0 = g.row[o.expert + 1];
    o.r1 = g.row[o.expert + 2];
    o.nn = p.k - o.c0 > kTok / 2 ? kTok : kTok / 2;
    steps = (o.r1 - o.r0 + kBK - 1) / kBK;
  } else {
    const int s = segment_of(g, p.experts + 2, (int)t);
    const int first = g.row[s], rows = g.row[s + 1] - first, parts = g.tile[s + 1] - g.tile[s], i = (int)t - g.tile[s];
    const int each = (rows + parts - 1) / parts;
    o.expert = s >= 1 && s <= p.experts ? s - 1 : -1;
    o.r0 = first + min(i * each, rows);
    o.r1 = first + min((i + 1) * each, rows);
    o.c0 = 0;
    o.nn = max((o.r1 - o.r0 + 31) & ~31, 32);
    steps = o.expert < 0 ? 0 : (p.k + kBK - 1) / kBK;
  }
  o.b0 = (int)((i64)steps * o.split / p.splits);
  o.b1 = (int)((i64)steps * (o.split + 1) / p.splits);
  return o;
}
// Whether a step of a dw tile reaches past its expert's rows.
template <int MODE>
__device__ __forceinline__ bool clears(const Tile& o, int kb) {
  return MODE == kDw && o.r1 - o.r0 - kb * kBK < kBK;
}

template <class TO, int MODE, bool WIDE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) grouped_tc(const __grid_constant__ P p) {
  using namespace ccb;
  constexpr int CHUNK = WIDE ? kChunkWide : MODE == kDw && sizeof(TO) == 4 ? kChunk : kWhole;
  extern __shared__ __align__(1024) unsigned char smem[];
  const unsigned raw = smem_u32(smem), pad = (1024u - (raw & 1023u)) & 1023u;
  const unsigned ring = raw + pad;
  Tail& s = *reinterpret_cast<Tail*>(smem + pad + kStages * kStageBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned rank = tc2::cta_rank();
  const unsigned pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  lay_out(s.g, p.off, p.experts, p.rows, kTok, p.err);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.full[i], 2);  // each CTA's producer (or its clearing warp), and both CTAs' bytes
      mbar_init(&s.empty[i], 1);
      mbar_init(&s.part[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.accf[i], 1);
      mbar_init(&s.acce[i], 2 * kDrain);  // the draining warps of both CTAs
    }
    mbar_init(&s.done, 1);
    s.stop = 0;
    mbar_fence_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc::fence_before();
  tc2::cluster_sync();
  tc::fence_after();
  const unsigned tmem = s.tmem;
  const unsigned tiles = tiles_of<MODE>(p, s.g);
  const Waiter wait = {smem_u32(&s.stop), tc2::peer_addr(&s.stop, rank ^ 1u), p.polls, p.err};
  const bool one = elect_one();
  const unsigned full = smem_u32(&s.full[0]), empty = smem_u32(&s.empty[0]), part = smem_u32(&s.part[0]), accf = smem_u32(&s.accf[0]),
                 acce = smem_u32(&s.acce[0]);
  const unsigned lead_full = tc2::peer_addr(&s.full[0], 0), lead_acce = tc2::peer_addr(&s.acce[0], 0);

  // each role returns at its end, or when a wait says that the kernel is to stop
  if (warp == 0) {
    unsigned st, turn;  // 8 * stage, turns of the ring
    auto produce = [&]() {
      unsigned at = ring, phase = 1;  // the stage's address
      st = turn = 0;
      for (unsigned t = pair; t < tiles; t += pairs) {
        const Tile o = tile_at<MODE>(p, s.g, t);
        const int half = o.nn >> 1, f = o.f0 + (int)rank * 128, c = o.c0 + (int)rank * half, tok = o.r0 + (int)rank * half;
        // tokens come as one copy of 128 rows, those that are not the tile's in vain (boxes of 16 or 64: the same up to 200
        // rows an expert of 4096 x 1024, 94 us against 89 at 270, 106-114 against 104 at 400)
        const unsigned bytes = kABytes + (MODE == kDw && !p.b2 ? half * 128u : kBBytes);
        int a = o.b0;
        do {
          const int z = chunk_end<CHUNK>(a, o.b1);
          for (int term = 0; term < terms<WIDE>(); ++term)
            for (int kb = a; kb < z; ++kb) {
              if (!wait(empty + st, phase)) return;
              if (one) {
                unsigned bar = lead_full + st;
                const int pm = plane_m<WIDE>(term), pn = plane_n<WIDE>(term);
                if (clears<MODE>(o, kb)) {
                  bar = part + st;
                  expect(bar, bytes);
                } else if (rank == 0) {
                  expect(full + st, bytes);
                } else {
                  expect_relaxed(bar, bytes);
                }
                const int k0 = kb * kBK;
                const unsigned sb = at + kABytes;
                if (MODE == kDw) {
                  const int r = o.r0 + k0;
                  if (p.a2) {
                    load4(at, &p.ta, 0, r, f >> 6, pm, bar);
                  } else {
                    load4(at, &p.ta, f, r, pm, 0, bar);
                    load4(at + 8192u, &p.ta, f + 64, r, pm, 0, bar);
                  }
                  if (p.b2) {
                    load4(sb, &p.tb, 0, r, c >> 6, pn, bar);
                  } else {
                    load4(sb, &p.tb, c, r, pn, 0, bar);
                    if (half > 64) load4(sb + 8192u, &p.tb, c + 64, r, pn, 0, bar);
                  }
                } else {
                  const int e = pm * p.experts + o.expert;
                  if (MODE == kForwardT) {
                    load4(at, &p.ta, k0, f, e, 0, bar);
                  } else if (p.a2) {
                    load4(at, &p.ta, 0, k0, f >> 6, e, bar);
                  } else {
                    load4(at, &p.ta, f, k0, e, 0, bar);
                    load4(at + 8192u, &p.ta, f + 64, k0, e, 0, bar);
                  }
                  load4(sb, &p.tb, k0, tok, pn, 0, bar);
                }
              }
              __syncwarp();
              st += 8;
              at += kStageBytes;
              if (st == 8 * kStages) {
                st = 0;
                at = ring;
                phase ^= 1u;
                ++turn;
              }
            }
          a = z;
        } while (a < o.b1);
      }
    };
    produce();
    if (lane == 0) s.issued = turn * kStages + (st >> 3);
  } else if (warp == 1) {
    auto multiply = [&]() {
      constexpr bool amn = MODE != kForwardT, bmn = MODE == kDw;
      const unsigned base = (1u << 4) | ((unsigned)p.format << 7) | ((unsigned)p.format << 10) | ((amn ? 1u : 0u) << 15) | ((bmn ? 1u : 0u) << 16) | (16u << 24);
      const u64 a0 = desc<amn>(ring), b0 = desc<bmn>(ring + kABytes);
      const unsigned empty0 = tc2::peer_addr(&s.empty[0], 0), empty1 = tc2::peer_addr(&s.empty[0], 1);
      const unsigned accf0 = tc2::peer_addr(&s.accf[0], 0), accf1 = tc2::peer_addr(&s.accf[0], 1);
      unsigned at = 0, phase = 0, it = 0;
      u64 a = a0, bd = b0;
      for (unsigned t = pair; t < tiles; t += pairs) {
        const Tile o = tile_at<MODE>(p, s.g, t);
        const unsigned idesc = base | ((unsigned)(o.nn >> 3) << 17);
        int from = o.b0;
        do {
          const int to = chunk_end<CHUNK>(from, o.b1);
          const unsigned ab = it & 1u, d = tmem + ab * kTok;
          if (!wait(acce + 8 * ab, ((it >> 1) & 1u) ^ 1u)) return;
          tc::fence_after();
          for (int term = 0; term < terms<WIDE>(); ++term)
            for (int kb = from; kb < to; ++kb) {
              const unsigned more = term > 0 || kb > from ? 1u : 0u;
              if (!wait(full + at, phase)) return;
              tc::fence_after();
              if (one) {
                if (clears<MODE>(o, kb)) {
                  const int kks = (o.r1 - o.r0 - kb * kBK + 15) / 16;
                  for (int kk = 0; kk < kks; ++kk) mma(d, a + kk * desc_step<amn>(), bd + kk * desc_step<bmn>(), idesc, kk > 0 ? 1u : more);
                } else {
#pragma unroll
                  for (int kk = 0; kk < kBK / 16; ++kk) mma(d, a + kk * desc_step<amn>(), bd + kk * desc_step<bmn>(), idesc, kk > 0 ? 1u : more);
                }
                commit(empty0 + at);
                commit(empty1 + at);
              }
              __syncwarp();
              at += 8;
              a += kStageBytes >> 4;
              bd += kStageBytes >> 4;
              if (at == 8 * kStages) {
                at = 0;
                a = a0;
                bd = b0;
                phase ^= 1u;
              }
            }
          if (one) {
            commit(accf0 + 8 * ab);
            commit(accf1 + 8 * ab);
          }
          __syncwarp();
          ++it;
          from = to;
        } while (from < o.b1);
      }
    };
    if (rank == 0) multiply();
  } else if (warp < 2 + kDrain) {
    auto drain = [&]() {
      const int q = warp & 3, other = (warp - 2) >> 2;  // its quarter of the lanes; every other 32 columns
      unsigned it = 0;
      for (unsigned t = pair; t < tiles; t += pairs) {
        const Tile o = tile_at<MODE>(p, s.g, t);
        const int f = o.f0 + (int)rank * 128 + q * 32;
        const int count = MODE == kDw ? min(p.k - o.c0, o.nn) : o.r1 - o.r0;
        TO* out = static_cast<TO*>(p.out) + o.split * p.split_stride + f + (MODE == kDw ? o.expert * p.oe + (i64)o.c0 * p.os : (i64)o.r0 * p.os);
        const unsigned acc0 = tmem + ((unsigned)(q * 32) << 16);
        if (CHUNK != kWhole && (WIDE || o.b1 - o.b0 > CHUNK)) {
          float sum[kTok / 64][32];
#pragma unroll
          for (int g = 0; g < kTok / 64; ++g)
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[g][i] = 0.0f;
          int a = o.b0;
          do {
            const unsigned ab = it & 1u;
            if (!wait(accf + 8 * ab, (it >> 1) & 1u)) return;
            tc::fence_after();
            if (f < p.n && a < o.b1) {
#pragma unroll
              for (int g = 0; g < kTok / 64; ++g) {
                const int c = 32 * other + 64 * g;
                if (c < count) {
                  float v[32];
                  __syncwarp();
                  tc::ld32(acc0 + ab * kTok + c, v);
#pragma unroll
                  for (int i = 0; i < 32; ++i) sum[g][i] += v[i];
                }
              }
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) arrive_relaxed(lead_acce + 8 * ab);
            ++it;
            a = chunk_end<CHUNK>(a, o.b1);
          } while (a < o.b1);
          if (f < p.n) {
#pragma unroll
            for (int g = 0; g < kTok / 64; ++g) {
              const int c = 32 * other + 64 * g;
              if (c < count) store32(sum[g], out + c * p.os, p.os, count - c, p.n - f, lane);
            }
            if constexpr (WIDE) {
              bool nan = false;
#pragma unroll
              for (int g = 0; g < kTok / 64; ++g)
#pragma unroll
                for (int i = 0; i < 32; ++i) nan |= sum[g][i] != sum[g][i];
              if (nan && f + lane < p.n) {  // columns past `count` may hold anything: the loop passes them over
                const i64 k0 = (MODE == kDw ? o.r0 : 0) + (i64)o.b0 * kBK, k1 = min(k0 + (i64)(o.b1 - o.b0) * kBK, (i64)(MODE == kDw ? o.r1 : p.k));
                for (int c = 32 * other; c < count; c += c % 32 == 31 ? 33 : 1) {
                  TO* at = out + lane + c * p.os;
                  if (*at != *at) *at = again(p.plain, MODE == kDw ? 0 : o.expert, k0, k1, f + lane, MODE == kDw ? o.c0 + c : o.r0 + c);
                }
              }
            }
          }
          continue;
        }
        const unsigned ab = it & 1u;
        if (!wait(accf + 8 * ab, (it >> 1) & 1u)) return;
        tc::fence_after();
        if (f < p.n) {
          for (int c = 32 * other; c < count; c += 32 * (kDrain / 4)) {
            if constexpr (sizeof(TO) == 2)
              drain16<TO>(acc0 + ab * kTok + c, o.b0 >= o.b1, smem_u32(s.out[warp - 2]), out + c * p.os, p.os, count - c, p.n - f, p.vec, lane);
            else
              drain32(acc0 + ab * kTok + c, o.b0 >= o.b1, out + c * p.os, p.os, count - c, p.n - f, lane);
            __syncwarp();
          }
        }
        tc::fence_before();
        __syncwarp();
        if (lane == 0) arrive_relaxed(lead_acce + 8 * ab);
        ++it;
      }
    };
    drain();
  } else if (MODE == kDw) {
    // a lane has one 16-byte piece of each row: two 64-wide blocks of the M side, then the N side's
    auto clear_rows = [&]() {
      unsigned stage = 0, phases = 0;  // bit i: parity of part[i]
      for (unsigned t = pair; t < tiles; t += pairs) {
        const Tile o = tile_at<MODE>(p, s.g, t);
        int a = o.b0;
        do {
          const int z = chunk_end<CHUNK>(a, o.b1);
          for (int term = 0; term < terms<WIDE>(); ++term)
            for (int kb = a; kb < z; ++kb) {
              if (clears<MODE>(o, kb)) {
                if (!wait(part + 8 * stage, (phases >> stage) & 1u)) return;
                phases ^= 1u << stage;
                const int left = o.r1 - o.r0 - kb * kBK, to = (left + 15) & ~15;
                uint4* at = reinterpret_cast<uint4*>(smem + pad + stage * kStageBytes + (lane >> 3) * 8192 + (lane & 7) * 16);
                for (int r = left; r < to; ++r) at[r * 8] = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive(lead_full + 8 * stage);
              }
              stage = stage + 1 == kStages ? 0 : stage + 1;
            }
          a = z;
        } while (a < o.b1);
      }
    };
    clear_rows();
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  tc2::cluster_sync();
  tc::fence_after();
  if (s.stop) {  // in both CTAs or in neither
    // Every role has ended. What is on its way: the MMAs, whose commit says when
    // they are over, and the copies. Those into a stage that is cleared complete
    // on the CTA's own barrier, the others on the even CTA's, whose phase ends
    // with an announcement by each producer and all bytes announced; where one
    // producer got further than the other (by at most the ring), the other
    // announces none for the stages in between.
    if (warp == 1) {
      if (rank == 0 && one) {
        commit(tc2::peer_addr(&s.done, 0));
        commit(tc2::peer_addr(&s.done, 1));
      }
      __syncwarp();
      wait_out(smem_u32(&s.done), 0);
    }
    if (warp == 0 && lane == 0) {
      const unsigned mine = s.issued, other = peer_word(&s.issued, rank ^ 1u), last = mine > other ? mine : other;
      // which of the stages' last copies are of rows that are cleared, and what each barrier `part` of this CTA has counted
      unsigned clear = 0, armed = 0, odd = 0;
      if (MODE == kDw) {
        unsigned j = 0;
        for (unsigned t = pair; t < tiles && j < last; t += pairs) {
          const Tile o = tile_at<MODE>(p, s.g, t);
          int a = o.b0;
          do {
            const int z = chunk_end<CHUNK>(a, o.b1);
            for (int term = 0; term < terms<WIDE>(); ++term)
              for (int kb = a; kb < z && j < last; ++kb, ++j) {
                const unsigned bit = 1u << (j % kStages);
                clear = clears<MODE>(o, kb) ? clear | bit : clear & ~bit;
                if (clears<MODE>(o, kb) && j < mine) {
                  armed |= bit;
                  odd ^= bit;
                }
              }
            a = z;
          } while (a < o.b1);
        }
      }
      for (unsigned i = 0; i < kStages; ++i)
        if ((armed >> i) & 1u) wait_out(part + 8 * i, ((odd >> i) & 1u) ^ 1u);
      for (unsigned j = mine; j < other; ++j)
        if (!((clear >> (j % kStages)) & 1u)) arrive(lead_full + 8 * (j % kStages));
      if (rank == 0)
        for (unsigned j = last > kStages ? last - kStages : 0; j < last; ++j)
          if (!((clear >> (j % kStages)) & 1u)) wait_out(full + 8 * (j % kStages), (j / kStages) & 1u);
    }
    __syncwarp();
    __syncthreads();
    tc2::cluster_sync();
    tc::fence_after();
  }
  __syncwarp();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// The sum of the parts of a divided contraction, in order: four results a
// thread, of one row of `out` (cols a multiple of 4, or one at a time). Some 3
// us for 32 x 1024 results of 4 parts: a launch, little else.
template <class TO, int N>
__global__ void __launch_bounds__(256) add_parts(const float* part, i64 stride, int parts, TO* out, i64 rows, i64 cols, i64 os, i64 mats, i64 oe) {
  const i64 each = rows * cols, total = mats * each / N;
  for (i64 i = (i64)blockIdx.x * 256 + threadIdx.x; i < total; i += (i64)gridDim.x * 256) {
    float v[N] = {};
    const float* at = part + i * N;
    for (int s = 0; s < parts; ++s, at += stride) {
      if constexpr (N == 4) {
        const float4 u = *reinterpret_cast<const float4*>(at);
        v[0] += u.x, v[1] += u.y, v[2] += u.z, v[3] += u.w;
      } else {
        v[0] += *at;
      }
    }
    const i64 e = i * N;
    i64 to = e;
    if (os != cols || (mats > 1 && oe != each)) {
      const i64 m = e / each, r = (e - m * each) / cols;
      to = m * oe + r * os + (e - m * each - r * cols);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) out[to + j] = from_f<TO>(v[j]);
  }
}

// A tensor map over 16-bit elements; dimensions of extent 1 get a legal stride.
bool encode(ccb::TmaDesc* out, int format, const void* base, int rank, const i64* dims, const i64* strides /* elements, rank - 1 */, const int* box) {
  const ccb::Driver& d = ccb::driver();
  if (!d.ok || !aligned(base, 16)) return false;
  cuuint64_t gd[4], gs[3];
  cuuint32_t bx[4], one[4] = {1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) {
    if (dims[i] < 1 || dims[i] >= (1ll << 32)) return false;
    gd[i] = (cuuint64_t)dims[i];
    bx[i] = (cuuint32_t)box[i];
    if (i > 0) {
      const i64 st = dims[i] == 1 ? 8 : strides[i - 1];
      if (st % 8 != 0 || st < 8 || st >= (1ll << 38)) return false;
      gs[i - 1] = (cuuint64_t)st * 2;
    }
  }
  static_assert(sizeof(CUtensorMap) == sizeof(ccb::TmaDesc), "tensor map size");
  return d.cuTensorMapEncodeTiled(reinterpret_cast<CUtensorMap*>(out), format ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                                  (cuuint32_t)rank, const_cast<void*>(base), gd, gs, bx, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class TO, int MODE, bool WIDE = false>
int go(const P& p, int sms, cudaStream_t st, const char* me) {
  static bool ready[64];  // the kernel's shared-memory limit was raised on the device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !__atomic_load_n(&ready[dev], __ATOMIC_RELAXED)) {
    const cudaError_t e = cudaFuncSetAttribute(grouped_tc<TO, MODE, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return fail(CCB_ERR_DRIVER, me, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) __atomic_store_n(&ready[dev], true, __ATOMIC_RELAXED);
  }
  grouped_tc<TO, MODE, WIDE><<<(unsigned)(sms & ~1), kThreads, kSmem, st>>>(p);
  return launched(me);
}
}  // namespace tcg

std::string check_sizes(i64 rows, i64 experts, i64 k, i64 n, int dtype) {
  if (rows < 0 || rows > INT_MAX - 1024) return "rows must be in [0, 2^31 - 1025]";
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


// ---------------------------------------------------------------- packing
// Operands that the tensor cores cannot take as they lie: f32, cut into three
// bf16 planes by truncation (8 significant bits each, so that hi + mid + lo is
// the number itself and no plane rounds up past the largest), and 16-bit ones
// whose rows are not aligned, copied. Rows of a plane are dense but for the
// last 16 bytes. A number that is not finite is its first plane alone (`again` has
// the products that this makes NaN). Bound by
// memory, 10 bytes an f32 element; 4096 rows over 8 experts of 1024 x 4096 f32
// take 220 us in all (CUDA-core tiles: 2029).
struct PackP {
  const void* in;
  unsigned short* out;
  i64 stride, row_stride, mats, rows;
  unsigned cols, ld;
};
struct PackBoth {
  PackP p[2];
};
template <class T>
__global__ void __launch_bounds__(256) pack_planes(const __grid_constant__ PackBoth both) {
  const PackP& q = both.p[blockIdx.y];
  const unsigned pieces = q.ld / 8;
  const i64 total = q.mats * q.rows * pieces, plane = q.mats * q.rows * q.ld;
  for (i64 i = (i64)blockIdx.x * 256 + threadIdx.x; i < total; i += (i64)gridDim.x * 256) {
    const i64 row = i / pieces, m = q.mats == 1 ? 0 : row / q.rows;
    const unsigned c = (unsigned)(i - row * pieces) * 8;
    const T* p = static_cast<const T*>(q.in) + m * q.stride + (row - m * q.rows) * q.row_stride + c;
    unsigned short* o = q.out + row * q.ld + c;
    if constexpr (sizeof(T) == 4) {
      alignas(16) unsigned short v[3][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = c + j < q.cols ? (float)p[j] : 0.0f;
        const float hi = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
        const bool fine = (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u;
        const float r = fine ? x - hi : 0.0f, mid = __uint_as_float(__float_as_uint(r) & 0xFFFF0000u), lo = r - mid;
        // a NaN keeps a bit of its fraction
        v[0][j] = (unsigned short)((__float_as_uint(x) >> 16) | (x != x ? 0x40u : 0u));
        v[1][j] = (unsigned short)(__float_as_uint(mid) >> 16);
        v[2][j] = (unsigned short)(__float_as_uint(lo) >> 16);
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4*>(o + k * plane) = *reinterpret_cast<const uint4*>(v[k]);
    } else {
      alignas(16) unsigned short v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < q.cols ? reinterpret_cast<const unsigned short*>(p)[j] : (unsigned short)0;
      *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(v);
    }
  }
}

// A stack of matrices as the copy engine reads it: in place, or packed.
struct Operand {
  const void* p;
  i64 mats, rows, cols, stride, row_stride;  // elements
  int planes;
  bool packs;
  i64 ld() const { return packs ? (cols + 7) / 8 * 8 : row_stride; }
  size_t bytes() const { return packs ? ((size_t)planes * mats * rows * ld() * 2 + 255) / 256 * 256 : 0; }
};
i64 ceil_div(i64 a, i64 b) { return (a + b - 1) / b; }
// 16-byte aligned rows of 16-bit elements
bool lies_well(const void* p, i64 mats, i64 rows, i64 stride, i64 row_stride) {
  return aligned(p, 16) && (rows <= 1 || (row_stride % 8 == 0 && row_stride < (1ll << 38))) && (mats <= 1 || (stride % 8 == 0 && stride < (1ll << 38)));
}
Operand operand(int dtype, const void* p, i64 mats, i64 rows, i64 cols, i64 stride, i64 row_stride) {
  Operand o = {p, mats, rows, cols, stride, row_stride, dtype == CCB_F32 ? 3 : 1, false};
  o.packs = dtype == CCB_F32 || !lies_well(p, mats, rows, stride, row_stride);
  return o;
}
// Packs the operands that have to be into `room` (and moves it on), in one launch.
int settle(Operand* a, Operand* b, int dtype, char** room, int sms, cudaStream_t st, const char* me) {
  PackBoth both = {};
  int n = 0;
  i64 work = 0;
  for (Operand* o : {a, b}) {
    if (!o->packs) continue;
    const i64 ld = o->ld();
    PackP& q = both.p[n++];
    q = {o->p, reinterpret_cast<unsigned short*>(*room), o->stride, o->row_stride, o->mats, o->rows, (unsigned)o->cols, (unsigned)ld};
    const i64 w = ceil_div(o->mats * o->rows * (ld / 8), 256);
    work = w > work ? w : work;
    *room += o->bytes();
    o->p = q.out;
    o->row_stride = ld;
    o->stride = o->rows * ld;
  }
  if (n == 0) return CCB_OK;
  const i64 most = (i64)sms * 16;
  const dim3 grid((unsigned)(work < most ? work : most), (unsigned)n);
  if (dtype == CCB_F32)
    pack_planes<float><<<grid, 256, 0, st>>>(both);
  else
    pack_planes<__half><<<grid, 256, 0, st>>>(both);
  return launched(me);
}

// In how many parts a contraction of `steps` is cut where there are too few
// tiles to fill the 74 pairs: the cheapest by a model of waves of tiles
// (0.35 us a step; a part's result is written and read in F32 at 5 TB/s, and
// their sum is a launch). `tiles` is the most that the sizes can give, since
// only the device knows which experts have rows.
int parts_of(i64 tiles, i64 steps, i64 result) {
  constexpr double kStep = 0.35, kSum = 2.5, kByte = 1.0 / 5e6;
  constexpr i64 kPairs = 74;
  int best = 1;
  double least = 0.0;
  for (int s = 1; s <= 32 && (s == 1 || steps / s >= 4); ++s) {
    const double t = (double)((tiles * s + kPairs - 1) / kPairs) * (double)((steps + s - 1) / s) * kStep + (s > 1 ? kSum + (double)result * s * 8 * kByte : 0.0);
    if (s == 1 || t < least) {
      least = t;
      best = s;
    }
  }
  return best;
}

// What a call does, by its sizes, types, strides and alignment alone.
struct Plan {
  bool tensor;     // on the tensor cores; else rows are few
  Operand w, x;    // M side, N side
  int parts;       // of the contraction
  i64 result;      // elements of one part's
  size_t bytes() const { return (tensor ? w.bytes() + x.bytes() : 0) + (parts > 1 ? (size_t)parts * result * sizeof(float) : 0); }
};
Plan plan_of(const ccb_nn_grouped_matmul_t* a) {
  Plan p = {};
  if (a->rows == 0 || a->n == 0 || a->k == 0) return p;
  const i64 some = a->experts < a->rows ? a->experts : a->rows;
  p.w = operand(a->dtype, a->w, a->experts, a->transpose_w ? a->n : a->k, a->transpose_w ? a->k : a->n, a->w_stride, a->w_row_stride);
  p.x = operand(a->dtype, a->x, 1, a->rows, a->k, 0, a->x_stride);
  // Packing reads and writes every expert's matrix: it pays from some rows an
  // expert on. In us, CUDA cores against packing and tensor cores: F32, 32 rows
  // of 12 experts, 2048 x 1024: 38 / 110; 128 rows of 16, 256 x 512: 11 / 17;
  // 700 rows of 20, 1024 x 1024: 76 / 84, transposed 113 / 82; 1003 rows of 6,
  // 515 x 129: 29 / 19; 200 rows of 2, 2000 x 2000: 68 / 38. BF16, 32 rows of
  // 12, 2047 x 1023: 27 / 44, transposed 33 / 45.
  p.tensor = !p.w.packs || a->rows >= 16 * some;
  p.result = a->rows * a->n;
  if (!p.tensor) {  // two tiles for each of five blocks an SM, and no part above what shared memory takes
    const i64 tiles = ceil_div(a->n, a->transpose_w ? kFewColsT : kFewCols) * (some + a->rows / kFewRows), most = ceil_div(a->k, a->transpose_w ? 512 : 256 / type_bytes(a->dtype)), least = ceil_div(a->k, kFewK);
    const i64 want = ceil_div(10 * 148, tiles);
    p.parts = (int)(want < least ? least : want > most ? most : want);
    return p;
  }
  p.parts = parts_of(ceil_div(a->n, tcg::kFeat) * (some + a->rows / tcg::kTok), ceil_div(a->k, tcg::kBK) * (p.w.planes == 3 ? 6 : 1), p.result);
  return p;
}
Plan plan_of(const ccb_nn_grouped_matmul_dw_t* a) {
  Plan p = {};
  if (a->rows == 0 || a->n == 0 || a->k == 0) return p;
  p.w = operand(a->dtype, a->dy, 1, a->rows, a->n, 0, a->dy_stride);
  p.x = operand(a->dtype, a->x, 1, a->rows, a->k, 0, a->x_stride);
  p.tensor = true;
  p.result = a->experts * a->k * a->n;
  p.parts = parts_of(ceil_div(a->n, tcg::kFeat) * ceil_div(a->k, tcg::kTok) * a->experts, ceil_div(a->rows, a->experts * tcg::kBK) * (p.w.planes == 3 ? 6 : 1), p.result);
  return p;
}
// "" if the workspace is enough
template <class A>
std::string check_workspace(const A* a, const Plan& p) {
  const size_t need = p.bytes();
  if (need == 0 || (a->workspace && aligned(a->workspace, 16) && a->workspace_bytes >= need)) return "";
  return "workspace of " + std::to_string(a->workspace_bytes) + " bytes: " + std::to_string(need) + " are needed, 16-byte aligned";
}

template <class TO>
int sum_parts(const tcg::P& p, TO* out, i64 rows, i64 cols, i64 os, i64 mats, i64 oe, int sms, cudaStream_t st, const char* me) {
  const bool four = cols % 4 == 0 && p.split_stride % 4 == 0;
  const i64 blocks = ceil_div(rows * cols * mats, four ? 1024 : 256), most = (i64)sms * 8;
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  const float* part = static_cast<const float*>(p.out);
  if (four)
    tcg::add_parts<TO, 4><<<grid, 256, 0, st>>>(part, p.split_stride, p.splits, out, rows, cols, os, mats, oe);
  else
    tcg::add_parts<TO, 1><<<grid, 256, 0, st>>>(part, p.split_stride, p.splits, out, rows, cols, os, mats, oe);
  return launched(me);
}

// The map of an MN-major operand: `outer` matrices of `rows` (the contraction)
// by `cols`. Where rows are whole 64-wide blocks, one copy takes two of them:
// the blocks are a dimension of their own.
bool encode_mn(ccb::TmaDesc* m, int fmt, const void* base, i64 cols, i64 rows, i64 outer, i64 stride, i64 outer_stride, int* two) {
  *two = cols % 64 == 0;
  if (*two) {
    const i64 d[4] = {64, rows, cols / 64, outer}, st[3] = {stride, 64, outer_stride};
    const int box[4] = {64, 64, 2, 1};
    return tcg::encode(m, fmt, base, 4, d, st, box);
  }
  const i64 d[4] = {cols, rows, outer, 1}, st[3] = {stride, outer_stride, 8};
  const int box[4] = {64, 64, 1, 1};
  return tcg::encode(m, fmt, base, 4, d, st, box);
}

unsigned wait_polls = ccb::MBAR_SPIN_LIMIT;  // ccb_nn_wait_polls

// The parts that both directions share.
tcg::P tensor_params(const Plan& plan, const int* off, unsigned* err, int dtype, i64 rows, i64 experts, i64 k, i64 n) {
  tcg::P p = {};
  p.off = off;
  p.err = err;
  p.rows = (int)rows;
  p.experts = (int)experts;
  p.n = (int)n;
  p.k = (int)k;
  p.splits = plan.parts;
  p.format = dtype != CCB_F16;
  p.polls = __atomic_load_n(&wait_polls, __ATOMIC_RELAXED);
  return p;
}

int tensor_forward(const ccb_nn_grouped_matmul_t* a, Plan plan, int sms, cudaStream_t st, const char* me) {
  tcg::P p = tensor_params(plan, a->offsets, a->err, a->dtype, a->rows, a->experts, a->k, a->n);
  char* room = static_cast<char*>(a->workspace);
  if (const int rc = settle(&plan.w, &plan.x, a->dtype, &room, sms, st, me)) return rc;
  const i64 xd[4] = {a->k, a->rows, plan.x.planes, 1}, xs[3] = {plan.x.row_stride, a->rows * plan.x.row_stride, 8};
  const int xb[4] = {64, 128, 1, 1};
  bool ok = tcg::encode(&p.tb, p.format, plan.x.p, 4, xd, xs, xb);
  if (a->transpose_w) {
    const i64 wd[4] = {a->k, a->n, a->experts * plan.w.planes, 1}, ws[3] = {plan.w.row_stride, plan.w.stride, 8};
    const int wb[4] = {64, 128, 1, 1};
    ok = ok && tcg::encode(&p.ta, p.format, plan.w.p, 4, wd, ws, wb);
  } else {
    ok = ok && encode_mn(&p.ta, p.format, plan.w.p, a->n, a->k, a->experts * plan.w.planes, plan.w.row_stride, plan.w.stride, &p.a2);
  }
  if (!ok) return fail(CCB_ERR_DRIVER, me, "cuTensorMapEncodeTiled refused x or w");
  if (a->dtype == CCB_F32)
    p.plain = {static_cast<const float*>(a->w), static_cast<const float*>(a->x), a->w_stride, a->transpose_w ? 1 : a->w_row_stride,
               a->transpose_w ? a->w_row_stride : 1, 1, a->x_stride};
  p.out = a->out;
  p.os = a->out_stride;
  p.vec = aligned(a->out, 16) && a->out_stride % 8 == 0;
  const bool parts = p.splits > 1;
  if (parts) {
    p.out = room;
    p.os = a->n;
    p.split_stride = plan.result;
  }
  if (a->dtype == CCB_F32) {
    if (const int rc = a->transpose_w ? tcg::go<float, tcg::kForwardT, true>(p, sms, st, me) : tcg::go<float, tcg::kForward, true>(p, sms, st, me)) return rc;
    return parts ? sum_parts(p, (float*)a->out, a->rows, a->n, a->out_stride, 1, 0, sms, st, me) : CCB_OK;
  }
  if (parts) {
    if (const int rc = a->transpose_w ? tcg::go<float, tcg::kForwardT>(p, sms, st, me) : tcg::go<float, tcg::kForward>(p, sms, st, me)) return rc;
    return p.format ? sum_parts(p, (__nv_bfloat16*)a->out, a->rows, a->n, a->out_stride, 1, 0, sms, st, me)
                    : sum_parts(p, (__half*)a->out, a->rows, a->n, a->out_stride, 1, 0, sms, st, me);
  }
  if (a->transpose_w) return p.format ? tcg::go<__nv_bfloat16, tcg::kForwardT>(p, sms, st, me) : tcg::go<__half, tcg::kForwardT>(p, sms, st, me);
  return p.format ? tcg::go<__nv_bfloat16, tcg::kForward>(p, sms, st, me) : tcg::go<__half, tcg::kForward>(p, sms, st, me);
}

template <class T>
int few_of(FewP* q, const ccb_nn_grouped_matmul_t* a, int sms, cudaStream_t st, const char* me) {
  if (q->splits == 1) {
    few<T, T>(*q, a->transpose_w, sms, st);
    return launched(me);
  }
  q->g.out = a->workspace;
  q->g.os = a->n;
  q->split_stride = a->rows * a->n;
  few<T, float>(*q, a->transpose_w, sms, st);
  if (const int rc = launched(me)) return rc;
  tcg::P p = {};
  p.out = a->workspace;
  p.splits = q->splits;
  p.split_stride = q->split_stride;
  return sum_parts(p, static_cast<T*>(a->out), a->rows, a->n, a->out_stride, 1, 0, sms, st, me);
}
int few_forward(const ccb_nn_grouped_matmul_t* a, const Plan& plan, int sms, cudaStream_t st, const char* me) {
  FewP q = {{a->x, a->w, a->offsets, a->out, a->err, a->k, a->n, a->x_stride, a->w_stride, a->w_row_stride, a->out_stride, (int)a->rows, (int)a->experts},
            plan.parts, 0, ceil_div(a->k, plan.parts)};
  if (a->dtype == CCB_F32) return few_of<float>(&q, a, sms, st, me);
  return a->dtype == CCB_BF16 ? few_of<__nv_bfloat16>(&q, a, sms, st, me) : few_of<__half>(&q, a, sms, st, me);
}

int tensor_dw(const ccb_nn_grouped_matmul_dw_t* a, Plan plan, int sms, cudaStream_t st, const char* me) {
  tcg::P p = tensor_params(plan, a->offsets, a->err, a->dtype, a->rows, a->experts, a->k, a->n);
  char* room = static_cast<char*>(a->workspace);
  if (const int rc = settle(&plan.w, &plan.x, a->dtype, &room, sms, st, me)) return rc;
  if (!encode_mn(&p.tb, p.format, plan.x.p, a->k, a->rows, plan.x.planes, plan.x.row_stride, a->rows * plan.x.row_stride, &p.b2) ||
      !encode_mn(&p.ta, p.format, plan.w.p, a->n, a->rows, plan.w.planes, plan.w.row_stride, a->rows * plan.w.row_stride, &p.a2))
    return fail(CCB_ERR_DRIVER, me, "cuTensorMapEncodeTiled refused x or dy");
  if (a->dtype == CCB_F32) p.plain = {static_cast<const float*>(a->dy), static_cast<const float*>(a->x), 0, a->dy_stride, 1, a->x_stride, 1};
  p.out = a->out;
  p.os = a->out_row_stride;
  p.oe = a->out_stride;
  p.vec = aligned(a->out, 16) && a->out_row_stride % 8 == 0 && (a->experts == 1 || a->out_stride % 8 == 0);
  const bool parts = p.splits > 1;
  if (parts) {
    p.out = room;
    p.os = a->n;
    p.oe = a->k * a->n;
    p.split_stride = plan.result;
  }
  if (parts || a->out_dtype == CCB_F32) {
    if (const int rc = a->dtype == CCB_F32 ? tcg::go<float, tcg::kDw, true>(p, sms, st, me) : tcg::go<float, tcg::kDw>(p, sms, st, me)) return rc;
    if (!parts) return CCB_OK;
    if (a->out_dtype == CCB_F32) return sum_parts(p, (float*)a->out, a->k, a->n, a->out_row_stride, a->experts, a->out_stride, sms, st, me);
    return p.format ? sum_parts(p, (__nv_bfloat16*)a->out, a->k, a->n, a->out_row_stride, a->experts, a->out_stride, sms, st, me)
                    : sum_parts(p, (__half*)a->out, a->k, a->n, a->out_row_stride, a->experts, a->out_stride, sms, st, me);
  }
  return p.format ? tcg::go<__nv_bfloat16, tcg::kDw>(p, sms, st, me) : tcg::go<__half, tcg::kDw>(p, sms, st, me);
}

}  // namespace
}  // namespace ccb_nn

using namespace ccb_nn;

extern "C" int ccb_nn_grouped_matmul_workspace(const ccb_nn_grouped_matmul_t* a, size_t* bytes) {
  static const char* const me = "ccb_nn_grouped_matmul_workspace";
  CCB_NN_GUARD(me, {
    if (!a || !bytes) return fail(CCB_ERR_INVALID, me, "null pointer");
    const std::string bad = check_grouped(a);
    if (!bad.empty()) return fail(CCB_ERR_INVALID, me, bad);
    *bytes = plan_of(a).bytes();
    return CCB_OK;
  })
}

extern "C" int ccb_nn_grouped_matmul_dw_workspace(const ccb_nn_grouped_matmul_dw_t* a, size_t* bytes) {
  static const char* const me = "ccb_nn_grouped_matmul_dw_workspace";
  CCB_NN_GUARD(me, {
    if (!a || !bytes) return fail(CCB_ERR_INVALID, me, "null pointer");
    const std::string bad = check_dw(a);
    if (!bad.empty()) return fail(CCB_ERR_INVALID, me, bad);
    *bytes = plan_of(a).bytes();
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
    const Plan plan = plan_of(a);
    const std::string small = check_workspace(a, plan);
    if (!small.empty()) return fail(CCB_ERR_INVALID, me, small);
    int sms = 0;
    if (const int rc = sm_count(me, &sms)) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (plan.tensor) return tensor_forward(a, plan, sms, st, me);
    if (plan.parts > 0) return few_forward(a, plan, sms, st, me);
    return clear(a->dtype, a->out, 1, a->rows, a->n, 0, a->out_stride, a->offsets, a->experts, a->rows, a->err, sms, st, me);
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
    const Plan plan = plan_of(a);
    const std::string small = check_workspace(a, plan);
    if (!small.empty()) return fail(CCB_ERR_INVALID, me, small);
    int sms = 0;
    if (const int rc = sm_count(me, &sms)) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (plan.tensor) return tensor_dw(a, plan, sms, st, me);
    return clear(a->out_dtype, a->out, a->experts, a->k, a->n, a->out_stride, a->out_row_stride, a->offsets, a->experts, a->rows, a->err, sms, st, me);
  })
}

extern "C" int ccb_nn_wait_polls(unsigned polls) {
  __atomic_store_n(&wait_polls, polls ? polls : ccb::MBAR_SPIN_LIMIT, __ATOMIC_RELAXED);
  return CCB_OK;
}
