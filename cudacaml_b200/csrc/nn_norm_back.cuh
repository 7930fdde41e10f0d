// The gradient of the join of a residual block and the next block's norm.
#pragma once
#include "nn_norm.cuh"

namespace ccb_nn {

constexpr int kVecs = 5;  // dpre_weight, dpre_bias, dpost_weight, dpost_bias, dgate of a channel

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
// The f16 ones (nn_norm_back_f16.cu: half the time of a build).
__attribute__((visibility("hidden"))) void backward_f16(int x_dtype, int kind, const BackP& p, int sms, cudaStream_t st);

namespace {

// The gradient for any length, alignment and stride, for what norm_back_rows
// does not take (8192 x 4096 bf16: 1767 us; 4096 rows of 12288 columns 3.5 ms, of
// 16384 5.2 ms). A block takes every grid-th row
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

// The gradient. MORE: also the sums of the biases' and of a channel gate's
// gradient. A row takes two sums over it (the statistics and the first norm's
// terms; the second norm's terms), three for the layer norm; between them the
// row is read again from the ring, piece by piece, which leaves registers for
// the sums over rows: they stay in them for all of a thread's rows. HAS: 0 any
// arguments; else all of rms norms without biases, with (2) a gate as a matrix of
// T or without one (1), in loops without branches that end the compiler's
// schedule. Bound by latency: two rows of 4096 leave 15 of 64 warps resident
// (51 % of the issue slots used). 8192 x 4096 bf16 with gate and mask 124 us (4.3
// TB/s; 135 by HAS = 0), without either 88 us (94); an f32 stream 210 us, f32
// throughout 309 us; with MORE a channel gate 188 us, its biases too 215 us, those
// of the layer norm 251 us: five sums, whichever are asked for, spill registers.
template <class T, class TX, int KIND, bool VEC, int PIECES, bool MORE, int HAS>
__global__ void __launch_bounds__(512) norm_back_rows(const __grid_constant__ BackP p, const Hold hold) {
  __shared__ __align__(16) float s[16 * 8];
  extern __shared__ __align__(16) unsigned char places[];
  typedef Part<TX, VEC, PIECES> PX;
  typedef Part<T, VEC, PIECES> PT;
  const int tpr = hold.tpr, ahead = hold.ahead;
  Group g(s, tpr);
  const Place<VEC> w0 = {(int)threadIdx.x - g.id * tpr, tpr, (int)p.cols};
  // a mean is divided, so that a constant row's is its value
  const float inv = 1.0f / (float)p.cols, f = p.scale * p.d.factor;
  const bool gate = HAS ? HAS == 2 : p.gate != nullptr, channel = !HAS && gate && p.gs == 0, full = HAS ? gate : gate && !channel && p.gdt != CCB_F32,
             has_dh = HAS || p.dh, has_dy = HAS || p.dy, has_b = HAS || p.b, has_db = HAS || p.db, post = HAS || p.post, norm2 = has_b && post, c2 = !HAS && p.c2;
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
  const int gate_at = 2 + c2, slots = gate_at + channel;
  if (g.id == 0) {
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const Place<VEC> w = w0.piece(k);
      float v[kE];
      vec8(v, p.w1, p.wdt, 1.0f, w);
      kept.put(k * slots, v);
      vec8(v, p.w2, p.wdt, 1.0f, w);
      kept.put(k * slots + 1, v);
      if (c2) {
        vec8(v, p.c2, p.wdt, 0.0f, w);
        kept.put(k * slots + 2, v);
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
      if (has_dh) {
        PX::fetch(to + oy, row_at<TX>(p.y, coming, p.ys), w0);
        PT::fetch(to + odh, row_at<T>(p.dh, coming, p.dhs), w0);
      }
      if (has_dy) PX::fetch(to + ody, row_at<TX>(p.dy, coming, p.dys), w0);
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
    // the row's parts, by piece
    auto get_y = [&](float* v, int k) { PX::get(v, here + oy, row_at<TX>(p.y, r, p.ys), w0, k); };
    auto get_dy = [&](float* v, int k) { PX::get(v, here + ody, row_at<TX>(p.dy, r, p.dys), w0, k); };
    auto get_dh = [&](float* v, int k) { PT::get(v, here + odh, row_at<T>(p.dh, r, p.dhs), w0, k); };
    auto get_b = [&](float* v, int k) { PT::get(v, here + ob, row_at<T>(p.b, r, p.bs), w0, k); };
    float m1 = 0.0f, f1 = 0.0f, m2 = 0.0f;
    if (KIND == 1) {
      float t[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        float a[kE], b[kE];
        if (has_dh) {
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
      m1 = t[0] / (float)p.cols;
      f1 = t[1] * inv;
      m2 = t[2] / (float)p.cols;
    }
    float q0[2] = {}, q1[2] = {}, q2[2] = {};
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const Place<VEC> w = w0.piece(k);
      float a[kE], b[kE], c[kE];
      if (has_dh) {
        get_y(a, k);
        get_dh(b, k);
        kept.get(k * slots, c);
        if (KIND == 1) {
#pragma unroll
          for (int i = 0; i < kE; ++i) a[i] = w.on(i) ? a[i] - m1 : 0.0f;
        }
        dot8(q0, a, a);
        mul8(b, b, c);
        dot8(q1, b, a);
      }
      if (norm2) {
        get_b(a, k);
        if (KIND == 1) {
#pragma unroll
          for (int i = 0; i < kE; ++i) a[i] = w.on(i) ? a[i] - m2 : 0.0f;
        }
        dot8(q2, a, a);
      }
    }
    float q[3] = {q0[0] + q0[1], q1[0] + q1[1], q2[0] + q2[1]};
    g.sum<3>(q);
    const float r1 = rsqrtf(q[0] * inv + p.eps), a1 = q[1] * inv * r1, r2 = norm2 ? rsqrtf(q[2] * inv + p.eps) : 1.0f;
    float g2[PIECES][kE], t[2] = {0.0f, 0.0f}, t0[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const Place<VEC> w = w0.piece(k);
      float d[kE], a[kE], b[kE], c[kE];
      if (has_dy)
        get_dy(d, k);
      else
#pragma unroll
        for (int i = 0; i < kE; ++i) d[i] = 0.0f;
      if (has_dh) {
        get_y(a, k);
        get_dh(b, k);
        kept.get(k * slots, c);
        if (KIND == 1) {
#pragma unroll
          for (int i = 0; i < kE; ++i) a[i] = w.on(i) ? a[i] - m1 : 0.0f;
        }
        mul8(a, a, r1);  // hat
        fma8(acc[0] + k * kE, b, a, acc[0] + k * kE);
        if (MORE) {
#pragma unroll
          for (int i = 0; i < kE; ++i) acc[2][k * kE + i] += b[i];
        }
        mul8(b, b, c);
        fma8(b, a, -a1, b);
        if (KIND == 1) {
#pragma unroll
          for (int i = 0; i < kE; ++i) b[i] -= f1;
        }
        fma8(d, b, r1, d);
      }
      if (HAS || p.dx) store8<TX>(row_at<TX>(p.dx, r, p.dxs), d, w);
      if (!has_b) continue;
      if (p.d.on) {
        unsigned u[kE];
        words8<VEC>(u, p.d, p.d.base + (u64)r * (unsigned)p.cols, w, places + hold.words);
#pragma unroll
        for (int i = 0; i < kE; ++i) d[i] = u[i] > p.d.last ? d[i] : 0.0f;
      }
      mul8(d, d, f);  // dz
      get_b(b, k);
      kept.get(k * slots + 1, c);
      if (KIND == 1) {  // 0 - mean is not 0
#pragma unroll
        for (int i = 0; i < kE; ++i) {
          b[i] -= m2;
          if (!w.on(i)) b[i] = d[i] = 0.0f;
        }
      }
      mul8(b, b, r2);  // hat
      if (gate) {
        if (channel) {
          kept.get(k * slots + gate_at, a);
        } else {
          if (full) {
            PT::get(a, here + og, row_at<T>(p.gate, r, p.gs), w0, k);
            act8<sizeof(T) == 4>(p.act, a);
          } else {
            vec8(a, gate_row(p.gate, p.gdt, p.gs, r), p.gdt, 0.0f, w);
            act8<true>(p.act, a);
          }
        }
        float u[kE];
        if (c2) {
          kept.get(k * slots + 2, u);
          fma8(u, b, c, u);
        } else {
          mul8(u, b, c);
        }
        mul8(u, u, d);
        slope8(p.act, a, u);
        if (MORE) {
#pragma unroll
          for (int i = 0; i < kE; ++i) acc[4][k * kE + i] += u[i];
        }
        mul8(d, d, a);  // du
        if (HAS || p.dgate) {
          if (!HAS && p.gdt == CCB_F32)
            store8<float>(row_at<float>(p.dgate, r, p.dgs), u, w);
          else
            store8<T>(row_at<T>(p.dgate, r, p.dgs), u, w);
        }
      }
      fma8(acc[1] + k * kE, d, b, acc[1] + k * kE);
      if (MORE) {
#pragma unroll
        for (int i = 0; i < kE; ++i) acc[3][k * kE + i] += d[i];
      }
      mul8(g2[k], d, c);
      dot8(t0, g2[k], b);
      if (KIND == 1) {
#pragma unroll
        for (int i = 0; i < kE; ++i) t[1] += g2[k][i];
      }
    }
    t[0] = t0[0] + t0[1];
    if (has_db) {
      float a2 = 0.0f, f2 = 0.0f;
      if (post) {
        if (KIND == 1)
          g.sum<2>(t);
        else
          g.sum<1>(t);
        a2 = t[0] * inv * r2 * r2;
        f2 = KIND == 1 ? t[1] * inv * r2 : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        if (post) {
          float b[kE];
          get_b(b, k);
          if (KIND == 1) {
#pragma unroll
            for (int i = 0; i < kE; ++i) b[i] -= m2;
          }
          mul8(g2[k], g2[k], r2);
          fma8(g2[k], b, -a2, g2[k]);
          if (KIND == 1) {
#pragma unroll
            for (int i = 0; i < kE; ++i) g2[k][i] -= f2;
          }
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
// take every eighth block, their results added in order (3 us for 148 blocks of
// 4096 columns and two sums; 32 warps the same).
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

template <class T, class TX, int KIND>
struct Backward {
  // The blocks of the launch, 0 if a row is too long.
  template <bool VEC, int PIECES, bool MORE, int HAS>
  static int rows(const BackP& p, int sms, cudaStream_t st) {
    static bool ready[64];
    const Shape f = shape_of(p.cols, PIECES, 512, VEC, 2 + (p.c2 != nullptr) + (p.gate && p.gs == 0), PIECES * kE * 4, [&](int block, int tpr) {
      return 2 * part_bytes<TX, VEC, PIECES>(p.cols, block, tpr) + 3 * part_bytes<T, VEC, PIECES>(p.cols, block, tpr);
    });
    if (!f.block || !room_for(norm_back_rows<T, TX, KIND, VEC, PIECES, MORE, HAS>, ready)) return 0;
    const i64 groups = f.block / f.hold.tpr, sets = (p.rows + groups - 1) / groups;
    const int most = sms < kBackBlocks ? sms : (int)kBackBlocks, grid = (int)(sets < most ? sets : most);
    norm_back_rows<T, TX, KIND, VEC, PIECES, MORE, HAS><<<grid, f.block, f.smem, st>>>(p, f.hold);
    return grid;
  }
  // Rows of 16 elements a thread, so that a block of 512 threads (128 registers
  // each) holds two of 4096 columns and one waits for its sums while the other
  // computes; of 8 where there are few columns (65536 x 256 bf16: 63 us, by 16 98;
  // 65536 x 320 127 and 106), of an f32 stream, whose ring holds fewer rows, up to
  // 4096 (16.8 million elements f32 of 512 columns 142 us and 152, of 2048 147 and
  // 153, of 4096 166 and 167). The shape does not go by the
  // rows or by which sums over them are asked for (all five spill some
  // registers), so that a row's results do not either.
  template <bool MORE>
  static int by_width(const BackP& p, int sms, cudaStream_t st) {
    if (!near({p.ys, p.dys, p.dhs, p.bs, p.gs, p.dxs, p.dbs, p.dgs}) || (p.d.on && !p.d.same)) return 0;
    // rows that share no 16-byte piece: 16 elements a thread only where 8 do not reach
    // (4096 x 6499 bf16: 300 us, 1612 by norm_back_any)
    if ((p.d.base & 3) || !wide(p.cols, {p.y, p.dy, p.dh, p.b, p.gate, p.dx, p.db, p.dgate}, {p.ys, p.dys, p.dhs, p.bs, p.gs, p.dxs, p.dbs, p.dgs}))
      return p.cols <= 512 * kE ? rows<false, 1, MORE, 0>(p, sms, st) : rows<false, 2, MORE, 0>(p, sms, st);
    const bool one = p.cols <= 256 || (sizeof(TX) == 4 && p.cols <= 4096);
    if constexpr (!MORE) {
      if (p.dh && p.dy && p.b && p.post && p.dx && p.db && !p.c2) {
        if (!p.gate) return one ? rows<true, 1, false, 1>(p, sms, st) : rows<true, 2, false, 1>(p, sms, st);
        if (p.gs && p.dgate && p.gdt == code_of<T>) return one ? rows<true, 1, false, 2>(p, sms, st) : rows<true, 2, false, 2>(p, sms, st);
      }
    }
    return one ? rows<true, 1, MORE, 0>(p, sms, st) : rows<true, 2, MORE, 0>(p, sms, st);
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

}  // namespace
}  // namespace ccb_nn
