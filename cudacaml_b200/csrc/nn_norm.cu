// ccb_nn_block_norm: the join of a residual block and the next block's norm.
#include "nn_norm.cuh"

namespace ccb_nn {
namespace {

// Threads of a block, at most: three rows of 4096 columns at 80 registers.
constexpr int kRowThreads = 768;

struct NormP {
  const void *x, *b, *gate, *w1, *c1, *w2, *c2;
  void *y, *h;
  i64 rows, cols, xs, bs, gs, ys, hs;
  float eps, scale;
  int gdt, wdt, act, post;
  Drop d;
};

// Rows of any length, alignment and stride, for what norm_rows does not take: a
// block walks a row once for each statistic and once for the results, reading
// it again each time (8192 x 4096 bf16 with gate and mask: 565 us; 4096 rows of
// 16384 columns 1118 us, where 12288 take 152 us by norm_rows).
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

// The join of rows that a group holds. HAS: 0 any arguments; else a normed
// branch without biases and both results, with (2) a gate as a matrix of T or
// without one (1): what a training step of an rms norm asks for, whose loops
// have no branches left to end the compiler's schedule. Bound by latency: three
// rows of 4096 leave 24 of 64 warps resident, which wait between a row's sums
// (57 % of the issue slots used, no unit near its rate). At 8192 x 4096 bf16 with a
// sigmoid gate and a mask 73 us (4.6 TB/s; 78 by HAS = 0; the generator is 17 us
// of it), a mask alone 62 us (70), neither 53 us (52; 512 columns 15 against 16);
// an f32 stream 99 us (4.4 TB/s), f32 throughout 177 us (3.8 TB/s).
template <class T, class TX, int KIND, bool VEC, int PIECES, int HAS>
__global__ void __launch_bounds__(kRowThreads) norm_rows(const __grid_constant__ NormP p, const Hold hold) {
  __shared__ __align__(16) float s[kRowThreads / 32 * 8];
  extern __shared__ __align__(16) unsigned char places[];
  typedef Part<TX, VEC, PIECES> PX;
  typedef Part<T, VEC, PIECES> PT;
  const int tpr = hold.tpr, ahead = hold.ahead;
  Group g(s, tpr);
  const Place<VEC> w0 = {(int)threadIdx.x - g.id * tpr, tpr, (int)p.cols};
  // a mean is divided, so that a constant row's is its value
  const float inv = 1.0f / (float)p.cols, f = p.scale * p.d.factor;
  const bool gate = HAS ? HAS == 2 : p.gate != nullptr, channel = !HAS && gate && p.gs == 0, full = HAS ? gate : gate && !channel && p.gdt != CCB_F32;
  const bool has_b = HAS || p.b, post = HAS || p.post, c1 = !HAS && p.c1, c2 = !HAS && p.c2;
  const unsigned sets = blockDim.x / tpr, first = blockIdx.x * sets + g.id, step = gridDim.x * sets, rows = (unsigned)p.rows;
  const unsigned all = (unsigned)__cvta_generic_to_shared(places);
  const unsigned ox = VEC ? threadIdx.x * 16 : g.id * (part_bytes<TX, VEC, PIECES>(p.cols, blockDim.x, tpr) / sets);
  const unsigned ob = part_bytes<TX, VEC, PIECES>(p.cols, blockDim.x, tpr) + (VEC ? threadIdx.x * 16 : g.id * (part_bytes<T, VEC, PIECES>(p.cols, blockDim.x, tpr) / sets));
  const unsigned og = ob + part_bytes<T, VEC, PIECES>(p.cols, blockDim.x, tpr), end = all + ahead * hold.slot;
  // kept, for each piece: w2, w1, then c2, c1 and a channel gate's act, as far as there are any
  const Kept kept = {all + hold.kept + w0.t * 16, (unsigned)tpr * 16};
  const int c1_at = 2 + c2, gate_at = c1_at + c1, slots = gate_at + channel;
  if (g.id == 0) {
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const Place<VEC> w = w0.piece(k);
      float v[kE];
      vec8(v, p.w2, p.wdt, 1.0f, w);
      kept.put(k * slots, v);
      vec8(v, p.w1, p.wdt, 1.0f, w);
      kept.put(k * slots + 1, v);
      if (c2) {
        vec8(v, p.c2, p.wdt, 0.0f, w);
        kept.put(k * slots + 2, v);
      }
      if (c1) {
        vec8(v, p.c1, p.wdt, 0.0f, w);
        kept.put(k * slots + c1_at, v);
      }
      if (channel) {
        vec8(v, p.gate, p.gdt, 0.0f, w);
        act8<true>(p.act, v);
        kept.put(k * slots + gate_at, v);
      }
    }
  }
  unsigned coming = first, to = all;
  auto fetch = [&]() {
    if (coming < rows) {
      PX::fetch(to + ox, row_at<TX>(p.x, coming, p.xs), w0);
      if (has_b) PT::fetch(to + ob, row_at<T>(p.b, coming, p.bs), w0);
      if (full) PT::fetch(to + og, row_at<T>(p.gate, coming, p.gs), w0);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    coming += step;
    to = to + hold.slot == end ? all : to + hold.slot;
  };
  if (VEC && tpr * PIECES * kE != p.cols)  // columns that there are not read as 0
    for (unsigned j = all + threadIdx.x * 16; j < end; j += blockDim.x * 16) asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(j), "r"(0) : "memory");
  __syncthreads();
  for (int a = 0; a + 1 < ahead; ++a) fetch();
  unsigned here = all;
  for (unsigned r = first; r < rows; r += step) {
    turn_ring<VEC>(g, ahead, fetch);
    float y[PIECES][kE], t[2];
    float m2 = 0.0f, r2 = 1.0f;
    const T* brow = row_at<T>(p.b, r, p.bs);
    if (has_b && post) {
      if (KIND == 1) {
        t[0] = 0.0f;
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
          float b[kE];
          PT::get(b, here + ob, brow, w0, k);
#pragma unroll
          for (int i = 0; i < kE; ++i) t[0] += b[i];
        }
        g.sum<1>(t);
        m2 = t[0] / (float)p.cols;
      }
      t[0] = t[1] = 0.0f;
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        float b[kE];
        PT::get(b, here + ob, brow, w0, k);
        if (KIND == 1) {
#pragma unroll
          for (int i = 0; i < kE; ++i) b[i] = w0.piece(k).on(i) ? b[i] - m2 : 0.0f;
        }
        dot8(t, b, b);
      }
      t[0] += t[1];
      g.sum<1>(t);
      r2 = rsqrtf(t[0] * inv + p.eps);
    }
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const Place<VEC> w = w0.piece(k);
      if (has_b) {
        float b[kE], v[kE];
        PT::get(b, here + ob, brow, w0, k);
        kept.get(k * slots, v);
        if (KIND == 1) {
#pragma unroll
          for (int i = 0; i < kE; ++i) b[i] -= m2;
        }
        mul8(b, b, r2);
        mul8(b, b, v);
        if (c2) {
          kept.get(k * slots + 2, v);
#pragma unroll
          for (int i = 0; i < kE; ++i) b[i] += v[i];
        }
        if (gate) {
          if (channel) {
            kept.get(k * slots + gate_at, v);
          } else {
            if (full) {
              PT::get(v, here + og, row_at<T>(p.gate, r, p.gs), w0, k);
              act8<sizeof(T) == 4>(p.act, v);
            } else {
              vec8(v, gate_row(p.gate, p.gdt, p.gs, r), p.gdt, 0.0f, w);
              act8<true>(p.act, v);
            }
          }
          mul8(b, b, v);
        }
        PX::get(y[k], here + ox, row_at<TX>(p.x, r, p.xs), w0, k);
        if (p.d.on) {
          unsigned u[kE];
          words8<VEC>(u, p.d, p.d.base + (u64)r * (unsigned)p.cols, w, places + hold.words);
#pragma unroll
          for (int i = 0; i < kE; ++i) b[i] = u[i] > p.d.last ? b[i] : 0.0f;
        }
        fma8(y[k], b, f, y[k]);
      } else {
        PX::get(y[k], here + ox, row_at<TX>(p.x, r, p.xs), w0, k);
      }
      if (HAS || p.y) store8<TX>(row_at<TX>(p.y, r, p.ys), y[k], w);
    }
    here = here + hold.slot == end ? all : here + hold.slot;
    if (!HAS && !p.h) continue;
    float m1 = 0.0f;
    if (KIND == 1) {
      t[0] = 0.0f;
#pragma unroll
      for (int k = 0; k < PIECES; ++k)
#pragma unroll
        for (int i = 0; i < kE; ++i)
          if (w0.piece(k).on(i)) t[0] += y[k][i];
      g.sum<1>(t);
      m1 = t[0] / (float)p.cols;
    }
    t[0] = t[1] = 0.0f;
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {  // columns that there are not: x and b are 0, but not b - mean or a bias
      if (KIND == 1 || c2) {
#pragma unroll
        for (int i = 0; i < kE; ++i) y[k][i] = w0.piece(k).on(i) ? y[k][i] - m1 : 0.0f;
      }
      dot8(t, y[k], y[k]);
    }
    t[0] += t[1];
    g.sum<1>(t);
    const float r1 = rsqrtf(t[0] * inv + p.eps);
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      float v[kE];
      kept.get(k * slots + 1, v);
      mul8(y[k], y[k], r1);
      mul8(y[k], y[k], v);
      if (c1) {
        kept.get(k * slots + c1_at, v);
#pragma unroll
        for (int i = 0; i < kE; ++i) y[k][i] += v[i];
      }
      store8<T>(row_at<T>(p.h, r, p.hs), y[k], w0.piece(k));
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <class T, class TX, int KIND>
struct Forward {
  template <bool VEC, int PIECES, int HAS>
  static bool rows(const NormP& p, int sms, cudaStream_t st) {
    static bool ready[64];
    const int matrices = (p.b != nullptr) + (HAS ? HAS == 2 : p.gate && p.gs != 0 && p.gdt != CCB_F32);
    const Shape f = shape_of(p.cols, PIECES, kRowThreads, VEC, 2 + (p.c1 != nullptr) + (p.c2 != nullptr) + (p.gate && p.gs == 0), 0, [&](int block, int tpr) {
      return part_bytes<TX, VEC, PIECES>(p.cols, block, tpr) + matrices * part_bytes<T, VEC, PIECES>(p.cols, block, tpr);
    });
    if (!f.block || !room_for(norm_rows<T, TX, KIND, VEC, PIECES, HAS>, ready)) return false;
    const i64 groups = f.block / f.hold.tpr, sets = (p.rows + groups - 1) / groups;
    norm_rows<T, TX, KIND, VEC, PIECES, HAS><<<(unsigned)(sets < sms ? sets : sms), f.block, f.smem, st>>>(p, f.hold);
    return true;
  }
  static bool by_width(const NormP& p, int sms, cudaStream_t st) {
    if (!near({p.xs, p.bs, p.gs, p.ys, p.hs}) || (p.d.on && !p.d.same)) return false;
    // rows that share no 16-byte piece: 16 elements a thread only where 8 do not reach
    // (4096 x 6499 bf16: 205 us, 439 by norm_any)
    if ((p.d.base & 3) || !wide(p.cols, {p.x, p.b, p.gate, p.y, p.h}, {p.xs, p.bs, p.gs, p.ys, p.hs}))
      return p.cols <= kRowThreads * kE ? rows<false, 1, 0>(p, sms, st) : rows<false, 2, 0>(p, sms, st);
    // What a thread does once a row (its sums, addresses, copies) is some 300
    // instructions: 16 elements share them, fewer where a warp holds the row (65536
    // rows of 256 columns: 35 us by 8 elements a thread, 57 by 16; of 320 71 and 63;
    // 32 would spill at the registers that three rows of 4096 leave). The shape goes
    // by the columns alone: a row's result does not depend on the rows beside it.
    const bool one = p.cols <= 256;
    if (p.b && p.post && p.y && p.h && !p.c1 && !p.c2) {
      if (!p.gate) return one ? rows<true, 1, 1>(p, sms, st) : rows<true, 2, 1>(p, sms, st);
      if (p.gs && p.gdt == code_of<T>) return one ? rows<true, 1, 2>(p, sms, st) : rows<true, 2, 2>(p, sms, st);
    }
    return one ? rows<true, 1, 0>(p, sms, st) : rows<true, 2, 0>(p, sms, st);
  }
  static void run(const NormP& p, int sms, cudaStream_t st) {
    if (by_width(p, sms, st)) return;
    const i64 most = (i64)sms * 8;
    norm_any<T, TX, KIND><<<(unsigned)(p.rows < most ? p.rows : most), kBlock, 0, st>>>(p);
  }
};

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
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->dtype == CCB_F16)
      by_f16<Forward>(a->dtype, a->x_dtype, a->kind, p, sms, st);
    else
      by_type_but_f16<Forward>(a->dtype, a->x_dtype, a->kind, p, sms, st);
    return launched(me);
  })
}
