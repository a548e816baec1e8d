// Norms before and after a block, fused with its gate and residual scale (gfx950).
//
//   b^ = N(block),  u = post_w b^,  y = x + scale gate u,  h = pre_w N(y)
//   rms:   N(a) = a / sqrt(mean(a^2) + eps)
//   layer: N(a) = (a - mean(a)) / sqrt(var(a) + eps)
//
// Backward, from dy and dh (y^ = N(y), r = the reciprocal in N, q = pre_w dh; means over the row):
//   T = dy + r_y (q - y^ mean(q y^) [- mean(q)])           layer terms in brackets
//   dx = T,  dpre_w = sum dh y^,  dgate = sum scale T u,  dscale = sum T gate u
//   du = scale gate T,  dpost_w = sum du b^,  p = post_w du
//   dblock = r_b (p - b^ mean(p b^) [- mean(p)])
//
// All of it is bound by memory: the forward reads x, block (and a full gate) and
// writes y and h once; the backward reads x, block, dy, dh and writes dx and dblock.
// It takes y from x and block again (fp32, never rounded) instead of reading the
// stored one: the same bytes, and no rounding of y enters the gradients.  Rows
// live in registers: a row belongs to TPR threads of IT vectors each, the statistics of
// the forward are kept (fp32, 2 or 4 a row) so that the backward needs two row sums.
//
// Sums over rows (weights, a shared gate, the scale): a workgroup takes a run
// of rows that share their gate row, adds up in fp32 registers and writes one partial row; a
// second kernel adds the partial rows in a fixed order.  No atomics: the same bits on every run.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "kans_api_internal.h"

namespace kans {
namespace {

struct NormArgs {
  const void *x, *block, *gate, *post_w, *pre_w;
  const float* scale_dev;  // the scale where it is a tensor, else null
  float scale, eps;
  void *y, *h;
  float* stats;            // [rows][2 (rms) or 4 (layer)]: r_b, r_y, mean_b, mean_y; or null
  long rows, gate_group;   // row r takes gate row r / gate_group
  int D;
  // backward
  const void *dy, *dh;
  void *dx, *dblock, *dgate;
  float* part;             // [chunks][parts][D] partial rows: pre_w, post_w, gate
  float* part_scale;       // [chunks]
  long span, per_chunk, chunks_per_group;  // the runs of rows: NormPlan
  int parts, at_pre, at_post, at_gate;  // rows of a chunk's partials, -1: not asked for
  int want_scale, gate_f32;  // gate_f32: dgate of a gate row for each row in fp32
};

// Elements of a vector: 16 bytes of the block's type.
template <typename TB> constexpr int vec_of() { return 16 / (int)sizeof(TB); }

template <typename T, int V> struct Vec { T e[V]; };

// V elements from p, of which `left` exist (the others 0).  Rows start at any element: the
// device takes wide accesses at any address.
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p, int left) {
  Vec<T, V> v;
  if (left >= V) {
    __builtin_memcpy(&v, p, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v.e[e] = e < left ? p[e] : (T)0.0f;
  }
  return v;
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, int left, const float* o) {
  Vec<T, V> v;
#pragma unroll
  for (int e = 0; e < V; ++e) v.e[e] = from_f32<T>(o[e]);
  if (left >= V) {
    __builtin_memcpy(p, &v, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < left) p[e] = v.e[e];
  }
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_or_one(const T* p, long at, int left) {
  if (p) return load_vec<T, V>(p + at, left);
  Vec<T, V> v;
#pragma unroll
  for (int e = 0; e < V; ++e) v.e[e] = (T)1.0f;
  return v;
}

// Sums of a and b over the TPR threads of a row, in each of them.  `slot` (0 or 1)
// alternates between consecutive calls: the barrier of a call then also separates the reads of the
// call before from the writes of the next.
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float (*lds)[2][16], int slot) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    a += __shfl_xor(a, d, 64);
    b += __shfl_xor(b, d, 64);
  }
  if constexpr (TPR > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      lds[slot][0][wave] = a;
      lds[slot][1][wave] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) {
      a += lds[slot][0][w];
      b += lds[slot][1][w];
    }
  }
}

// Mean (layer) and reciprocal size of a row's values in v (zeros outside the row).
template <bool kLayer, int TPR, int IT, int V>
__device__ __forceinline__ void row_stats(const float (&v)[IT][V], int at0, int D, float eps, float (*lds)[2][16], int& slot,
                                          float& mean, float& r) {
  float s = 0.0f, none = 0.0f;
  mean = 0.0f;
  if constexpr (kLayer) {
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) s += v[i][e];
    row_sum2<TPR>(s, none, lds, slot);
    slot ^= 1;
    mean = s / (float)D;
    s = none = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < IT; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float c = at0 + i * TPR * V + e < D ? v[i][e] - mean : 0.0f;
      s += c * c;
    }
  row_sum2<TPR>(s, none, lds, slot);
  slot ^= 1;
  r = 1.0f / __builtin_sqrtf(s / (float)D + eps);
}

template <typename TX, typename TB, bool kLayer, int TPR, int IT>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void k_resnorm_fwd(const NormArgs A) {
  constexpr int V = vec_of<TB>();
  __shared__ float lds[2][2][16];
  const int t = TPR == 64 ? threadIdx.x & 63 : threadIdx.x;
  const long row = TPR == 64 ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : (long)blockIdx.x;
  if (row >= A.rows) return;  // (TPR = 64 only, whose waves meet at no barrier)
  const int D = A.D, at0 = t * V;
  const long base = row * D;
  float y[IT][V];
  Vec<TX, V> x[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int at = at0 + i * TPR * V;
    x[i] = load_vec<TX, V>((const TX*)A.x + base + at, D - at);
  }
  int slot = 0;
  float mean_b = 0.0f, r_b = 0.0f;
  if (A.block) {
    Vec<TB, V> g[IT], pw[IT];
    float b[IT][V];
    const long grow = row / A.gate_group * D;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int at = at0 + i * TPR * V;
      const Vec<TB, V> bv = load_vec<TB, V>((const TB*)A.block + base + at, D - at);
      g[i] = load_or_one<TB, V>((const TB*)A.gate, grow + at, D - at);
      pw[i] = load_or_one<TB, V>((const TB*)A.post_w, at, D - at);
#pragma unroll
      for (int e = 0; e < V; ++e) b[i][e] = to_f32(bv.e[e]);
    }
    const float scale = A.scale_dev ? *A.scale_dev : A.scale;
    row_stats<kLayer, TPR, IT, V>(b, at0, D, A.eps, lds, slot, mean_b, r_b);
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int at = at0 + i * TPR * V;
#pragma unroll
      for (int e = 0; e < V; ++e)
        y[i][e] = at + e < D ? to_f32(x[i].e[e]) + scale * to_f32(g[i].e[e]) * ((b[i][e] - mean_b) * r_b * to_f32(pw[i].e[e])) : 0.0f;
      store_vec<TX, V>((TX*)A.y + base + at, D - at, y[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) y[i][e] = to_f32(x[i].e[e]);
  }
  Vec<TB, V> nw[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) nw[i] = load_or_one<TB, V>((const TB*)A.pre_w, at0 + i * TPR * V, D - at0 - i * TPR * V);
  float mean_y, r_y;
  row_stats<kLayer, TPR, IT, V>(y, at0, D, A.eps, lds, slot, mean_y, r_y);
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int at = at0 + i * TPR * V;
    float h[V];
#pragma unroll
    for (int e = 0; e < V; ++e) h[e] = (y[i][e] - mean_y) * r_y * to_f32(nw[i].e[e]);
    store_vec<TB, V>((TB*)A.h + base + at, D - at, h);
  }
  if (A.stats && t == 0) {
    float* s = A.stats + row * (kLayer ? 4 : 2);
    s[0] = r_b;
    s[1] = r_y;
    if constexpr (kLayer) {
      s[2] = mean_b;
      s[3] = mean_y;
    }
  }
}

// What the backward reads of one row.
template <typename TX, typename TB, int IT>
struct RowIn {
  static constexpr int V = vec_of<TB>();
  Vec<TX, V> x[IT], dy[IT];
  Vec<TB, V> b[IT], dh[IT], g[IT];
  float r_b, r_y, mean_b, mean_y;
};

template <typename TX, typename TB, bool kLayer, int TPR, int IT>
__device__ __forceinline__ void load_row(RowIn<TX, TB, IT>& in, const NormArgs& A, long row, int at0, bool gate_rows) {
  constexpr int V = vec_of<TB>();
  const long base = row * A.D;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int at = at0 + i * TPR * V, left = A.D - at;
    in.x[i] = load_vec<TX, V>((const TX*)A.x + base + at, left);
    if (A.dy) in.dy[i] = load_vec<TX, V>((const TX*)A.dy + base + at, left);
    if (A.dh) in.dh[i] = load_vec<TB, V>((const TB*)A.dh + base + at, left);
    if (A.block) in.b[i] = load_vec<TB, V>((const TB*)A.block + base + at, left);
    if (gate_rows) in.g[i] = load_vec<TB, V>((const TB*)A.gate + base + at, left);
  }
  const float* s = A.stats + row * (kLayer ? 4 : 2);
  in.r_b = s[0];
  in.r_y = s[1];
  in.mean_b = kLayer ? s[2] : 0.0f;
  in.mean_y = kLayer ? s[3] : 0.0f;
}

// One workgroup takes the rows of a chunk, four at a time where a wave holds a row (TPR = 64), else one
// after the other with the next row's loads in flight.
template <typename TX, typename TB, bool kLayer, int TPR, int IT>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void k_resnorm_bwd(const NormArgs A) {
  constexpr int V = vec_of<TB>();
  constexpr int ROWS = TPR == 64 ? 4 : 1;
  __shared__ float lds[2][2][16];
  __shared__ float sums[TPR == 64 ? IT * V * 64 : 1];
  const int t = TPR == 64 ? threadIdx.x & 63 : threadIdx.x, sub = TPR == 64 ? threadIdx.x >> 6 : 0;
  const int D = A.D, at0 = t * V;
  const long chunk = blockIdx.x, group = chunk / A.chunks_per_group;
  const long first = group * A.span + (chunk - group * A.chunks_per_group) * A.per_chunk;
  const long end = min(min(first + A.per_chunk, (group + 1) * A.span), A.rows);
  const bool gate_rows = A.gate && A.gate_group == 1;
  const float scale = A.scale_dev ? *A.scale_dev : A.scale;
  Vec<TB, V> pw[IT], nw[IT];
  RowIn<TX, TB, IT> next;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int at = at0 + i * TPR * V;
    pw[i] = load_or_one<TB, V>((const TB*)A.post_w, at, D - at);
    nw[i] = load_or_one<TB, V>((const TB*)A.pre_w, at, D - at);
    next.g[i] = load_or_one<TB, V>((const TB*)A.gate, group * D + at, gate_rows ? 0 : D - at);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      next.dy[i].e[e] = (TX)0.0f;
      next.dh[i].e[e] = (TB)0.0f;
      next.b[i].e[e] = (TB)0.0f;
    }
  }
  float s_pre[IT][V], s_post[IT][V], s_gate[IT][V], s_scale = 0.0f;
#pragma unroll
  for (int i = 0; i < IT; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) s_pre[i][e] = s_post[i][e] = s_gate[i][e] = 0.0f;
  const float inv_d = 1.0f / (float)D;
  if (first + sub < end) load_row<TX, TB, kLayer, TPR, IT>(next, A, first + sub, at0, gate_rows);
  for (long row = first + sub; row < end; row += ROWS) {
    const RowIn<TX, TB, IT> in = next;
    if (row + ROWS < end) load_row<TX, TB, kLayer, TPR, IT>(next, A, row + ROWS, at0, gate_rows);
    const long base = row * D;
    float tt[IT][V], bn[IT][V], yn[IT][V];
    float sa = 0.0f, sb = 0.0f;
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const bool ok = at0 + i * TPR * V + e < D;
        bn[i][e] = ok ? (to_f32(in.b[i].e[e]) - in.mean_b) * in.r_b : 0.0f;
        const float y = to_f32(in.x[i].e[e]) + scale * to_f32(in.g[i].e[e]) * (bn[i][e] * to_f32(pw[i].e[e]));
        yn[i][e] = ok ? (y - in.mean_y) * in.r_y : 0.0f;
        const float dh = to_f32(in.dh[i].e[e]), q = to_f32(nw[i].e[e]) * dh;
        s_pre[i][e] += dh * yn[i][e];
        sa += q * yn[i][e];
        sb += q;
      }
    row_sum2<TPR>(sa, sb, lds, 0);
    sa *= inv_d;
    sb = kLayer ? sb * inv_d : 0.0f;
    float pa = 0.0f, pb = 0.0f;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int at = at0 + i * TPR * V;
      float dg[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float q = to_f32(nw[i].e[e]) * to_f32(in.dh[i].e[e]);
        const float T = to_f32(in.dy[i].e[e]) + in.r_y * (q - yn[i][e] * sa - sb);
        tt[i][e] = T;
        const float g = to_f32(in.g[i].e[e]), u = bn[i][e] * to_f32(pw[i].e[e]);
        dg[e] = scale * T * u;
        const float du = scale * g * T;
        s_gate[i][e] += dg[e];
        s_scale += at + e < D ? T * (g * u) : 0.0f;
        s_post[i][e] += du * bn[i][e];
        const float p = du * to_f32(pw[i].e[e]);
        pa += p * bn[i][e];
        pb += at + e < D ? p : 0.0f;
      }
      if (A.dx) store_vec<TX, V>((TX*)A.dx + base + at, D - at, tt[i]);
      if (gate_rows && A.dgate) {
        if (A.gate_f32) store_vec<float, V>((float*)A.dgate + base + at, D - at, dg);
        else store_vec<TB, V>((TB*)A.dgate + base + at, D - at, dg);
      }
    }
    if (A.block) {
      row_sum2<TPR>(pa, pb, lds, 1);
      pa *= inv_d;
      pb = kLayer ? pb * inv_d : 0.0f;
      if (A.dblock) {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int at = at0 + i * TPR * V;
          float db[V];
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float p = scale * to_f32(in.g[i].e[e]) * tt[i][e] * to_f32(pw[i].e[e]);
            db[e] = in.r_b * (p - bn[i][e] * pa - pb);
          }
          store_vec<TB, V>((TB*)A.dblock + base + at, D - at, db);
        }
      }
    } else if constexpr (TPR > 64) {
      __syncthreads();  // the barrier of the second sum (row_sum2)
    }
  }
  // the chunk's partial rows
  float* part = A.part + chunk * A.parts * D;
  auto put = [&](int at_part, const float(&s)[IT][V]) {
    if (at_part < 0) return;
    float* o = part + (long)at_part * D;
    if constexpr (TPR == 64) {
      // the four waves one after the other, into one row of LDS
      for (int w = 0; w < 4; ++w) {
        if (sub == w) {
#pragma unroll
          for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
              float* c = &sums[(i * V + e) * 64 + t];
              *c = w == 0 ? s[i][e] : *c + s[i][e];
            }
        }
        __syncthreads();
      }
      for (int j = threadIdx.x; j < D; j += 256) {
        const int i = j / (64 * V), l = (j / V) & 63, e = j % V;
        o[j] = sums[(i * V + e) * 64 + l];
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int i = 0; i < IT; ++i) store_vec<float, V>(o + at0 + i * TPR * V, D - at0 - i * TPR * V, s[i]);
    }
  };
  put(A.at_pre, s_pre);
  put(A.at_post, s_post);
  put(A.at_gate, s_gate);
  if (A.want_scale) {
    constexpr int NT = TPR == 64 ? 256 : TPR;
    float none = 0.0f;
    __syncthreads();
    row_sum2<NT>(s_scale, none, lds, 0);
    if (threadIdx.x == 0) A.part_scale[chunk] = s_scale;
  }
}

// ---- rows that no workgroup's registers hold ---------------------------------------------------------
// A workgroup of 1024 threads goes over its row once for each statistic; the rows after the first time come from L2.
constexpr int kWide = 1024;

template <typename TX, typename TB, bool kLayer>
__global__ __launch_bounds__(kWide) void k_resnorm_wide_fwd(const NormArgs A) {
  __shared__ float lds[2][2][16];
  const long row = blockIdx.x;
  const int D = A.D;
  const TX* x = (const TX*)A.x + row * D;
  const TB* b = A.block ? (const TB*)A.block + row * D : nullptr;
  const TB* g = A.gate ? (const TB*)A.gate + row / A.gate_group * D : nullptr;
  const TB *pw = (const TB*)A.post_w, *nw = (const TB*)A.pre_w;
  const float scale = A.scale_dev ? *A.scale_dev : A.scale;
  int slot = 0;
  auto sum = [&](auto value) {
    float s = 0.0f, none = 0.0f;
    for (int j = threadIdx.x; j < D; j += kWide) s += value(j);
    row_sum2<kWide>(s, none, lds, slot);
    slot ^= 1;
    return s;
  };
  float mean_b = 0.0f, r_b = 0.0f, mean_y = 0.0f;
  if (b) {
    if (kLayer) mean_b = sum([&](int j) { return to_f32(b[j]); }) / (float)D;
    r_b = 1.0f / __builtin_sqrtf(sum([&](int j) { const float c = to_f32(b[j]) - mean_b; return c * c; }) / (float)D + A.eps);
  }
  auto y = [&](int j) {
    float v = to_f32(x[j]);
    if (b) v += scale * (g ? to_f32(g[j]) : 1.0f) * ((to_f32(b[j]) - mean_b) * r_b * (pw ? to_f32(pw[j]) : 1.0f));
    return v;
  };
  if (kLayer) mean_y = sum(y) / (float)D;
  const float r_y = 1.0f / __builtin_sqrtf(sum([&](int j) { const float c = y(j) - mean_y; return c * c; }) / (float)D + A.eps);
  for (int j = threadIdx.x; j < D; j += kWide) {
    const float v = y(j);
    if (b) ((TX*)A.y)[row * D + j] = from_f32<TX>(v);
    ((TB*)A.h)[row * D + j] = from_f32<TB>((v - mean_y) * r_y * (nw ? to_f32(nw[j]) : 1.0f));
  }
  if (A.stats && threadIdx.x == 0) {
    float* s = A.stats + row * (kLayer ? 4 : 2);
    s[0] = r_b;
    s[1] = r_y;
    if (kLayer) {
      s[2] = mean_b;
      s[3] = mean_y;
    }
  }
}

// A chunk's rows one after the other; the partial rows are added up in memory, each column by one thread.
template <typename TX, typename TB, bool kLayer>
__global__ __launch_bounds__(kWide) void k_resnorm_wide_bwd(const NormArgs A) {
  __shared__ float lds[2][2][16];
  const int D = A.D;
  const long chunk = blockIdx.x, group = chunk / A.chunks_per_group;
  const long first = group * A.span + (chunk - group * A.chunks_per_group) * A.per_chunk;
  const long end = min(min(first + A.per_chunk, (group + 1) * A.span), A.rows);
  const TB *pw = (const TB*)A.post_w, *nw = (const TB*)A.pre_w;
  const float scale = A.scale_dev ? *A.scale_dev : A.scale, inv_d = 1.0f / (float)D;
  float* part = A.part + chunk * A.parts * D;
  for (int j = threadIdx.x; j < D; j += kWide)
    for (int k = 0; k < A.parts; ++k) part[(long)k * D + j] = 0.0f;
  float s_scale = 0.0f;
  for (long row = first; row < end; ++row) {
    const TX* x = (const TX*)A.x + row * D;
    const TB* b = A.block ? (const TB*)A.block + row * D : nullptr;
    const TB* g = A.gate ? (const TB*)A.gate + row / A.gate_group * D : nullptr;
    const TX* dy = A.dy ? (const TX*)A.dy + row * D : nullptr;
    const TB* dh = A.dh ? (const TB*)A.dh + row * D : nullptr;
    const float* s = A.stats + row * (kLayer ? 4 : 2);
    const float r_b = s[0], r_y = s[1], mean_b = kLayer ? s[2] : 0.0f, mean_y = kLayer ? s[3] : 0.0f;
    auto bn = [&](int j) { return b ? (to_f32(b[j]) - mean_b) * r_b : 0.0f; };
    auto gt = [&](int j) { return g ? to_f32(g[j]) : 1.0f; };
    auto post = [&](int j) { return pw ? to_f32(pw[j]) : 1.0f; };
    auto yn = [&](int j) { return (to_f32(x[j]) + scale * gt(j) * (bn(j) * post(j)) - mean_y) * r_y; };
    auto qv = [&](int j) { return dh ? to_f32(dh[j]) * (nw ? to_f32(nw[j]) : 1.0f) : 0.0f; };
    float sa = 0.0f, sb = 0.0f;
    for (int j = threadIdx.x; j < D; j += kWide) {
      sa += qv(j) * yn(j);
      sb += qv(j);
    }
    row_sum2<kWide>(sa, sb, lds, 0);
    sa *= inv_d;
    sb = kLayer ? sb * inv_d : 0.0f;
    auto T = [&](int j) { return (dy ? to_f32(dy[j]) : 0.0f) + r_y * (qv(j) - yn(j) * sa - sb); };
    float pa = 0.0f, pb = 0.0f;
    for (int j = threadIdx.x; j < D; j += kWide) {
      const float t = T(j), n = bn(j), u = n * post(j), du = scale * gt(j) * t, p = du * post(j);
      if (A.dx) ((TX*)A.dx)[row * D + j] = from_f32<TX>(t);
      if (A.dgate && A.gate_group == 1) {
        if (A.gate_f32) ((float*)A.dgate)[row * D + j] = scale * t * u;
        else ((TB*)A.dgate)[row * D + j] = from_f32<TB>(scale * t * u);
      }
      if (A.at_pre >= 0 && dh) part[(long)A.at_pre * D + j] += to_f32(dh[j]) * yn(j);
      if (A.at_post >= 0) part[(long)A.at_post * D + j] += du * n;
      if (A.at_gate >= 0) part[(long)A.at_gate * D + j] += scale * t * u;
      s_scale += t * (gt(j) * u);
      pa += p * n;
      pb += p;
    }
    row_sum2<kWide>(pa, pb, lds, 1);
    pa *= inv_d;
    pb = kLayer ? pb * inv_d : 0.0f;
    if (A.block && A.dblock)
      for (int j = threadIdx.x; j < D; j += kWide) {
        const float p = scale * gt(j) * T(j) * post(j);
        ((TB*)A.dblock)[row * D + j] = from_f32<TB>(r_b * (p - bn(j) * pa - pb));
      }
  }
  if (A.want_scale) {
    float none = 0.0f;
    __syncthreads();
    row_sum2<kWide>(s_scale, none, lds, 0);
    if (threadIdx.x == 0) A.part_scale[chunk] = s_scale;
  }
}

// ---- sums of the partial rows -------------------------------------------------------------------------
struct ReduceArgs {
  const float *part, *part_scale;
  void *dpre, *dpost, *dgate;
  float* dscale;
  long chunks, chunks_per_group;
  long groups, col_tiles;
  int D, parts, at_pre, at_post, at_gate;
};

// A workgroup adds 64 columns of one output row at a time: 16 runs of partial rows, joined in a fixed order.
// Work by column tile and output row: dpre, dpost, then dgate's groups, and last the scale.
template <typename TB>
__global__ __launch_bounds__(1024) void k_resnorm_reduce(const ReduceArgs A) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, run = threadIdx.x >> 6;
  const int weights = (A.at_pre >= 0) + (A.at_post >= 0);
  const long outs = weights + (A.at_gate >= 0 ? A.groups : 0);
  for (long w = blockIdx.x; w < outs * A.col_tiles; w += gridDim.x) {
    const long out = w / A.col_tiles, g = out - weights;
    const int col = (int)(w - out * A.col_tiles) * 64 + lane;
    const int which = g >= 0 ? A.at_gate : (int)out;  // (at_pre and at_post come first, in this order)
    const long c0 = g >= 0 ? g * A.chunks_per_group : 0, c1 = g >= 0 ? c0 + A.chunks_per_group : A.chunks;
    float s = 0.0f;
    if (col < A.D)
      for (long c = c0 + run; c < c1; c += 16) s += A.part[(c * A.parts + which) * A.D + col];
    lds[run][lane] = s;
    __syncthreads();
    if (run == 0 && col < A.D) {
#pragma unroll
      for (int r = 1; r < 16; ++r) s += lds[r][lane];
      TB* o = g >= 0 ? (TB*)A.dgate + g * A.D : which == A.at_pre ? (TB*)A.dpre : (TB*)A.dpost;
      o[col] = from_f32<TB>(s);
    }
    __syncthreads();
  }
  if (A.dscale && blockIdx.x == gridDim.x - 1) {
    float* flat = &lds[0][0];
    float s = 0.0f;
    for (long c = threadIdx.x; c < A.chunks; c += 1024) s += A.part_scale[c];
    flat[threadIdx.x] = s;
    __syncthreads();
    for (int d = 512; d > 0; d >>= 1) {
      if ((int)threadIdx.x < d) flat[threadIdx.x] += flat[threadIdx.x + d];
      __syncthreads();
    }
    if (threadIdx.x == 0) *A.dscale = flat[0];
  }
}

// ---- launches ---------------------------------------------------------------------------------------
// Threads a row and vectors a thread: a wave for the rows that it holds in two vectors a lane (no barriers), else the
// fewest threads that hold the row in at most two.
template <typename TX, typename TB, bool kLayer>
hipError_t launch_fwd(const NormArgs& A, hipStream_t st) {
  constexpr int V = vec_of<TB>();
  const int vecs = (A.D + V - 1) / V;
  const dim3 rows((unsigned)A.rows), four((unsigned)((A.rows + 3) / 4));
  if (vecs <= 64) hipLaunchKernelGGL((k_resnorm_fwd<TX, TB, kLayer, 64, 1>), four, dim3(256), 0, st, A);
  else if (vecs <= 128) hipLaunchKernelGGL((k_resnorm_fwd<TX, TB, kLayer, 64, 2>), four, dim3(256), 0, st, A);
  else if (vecs <= 256) hipLaunchKernelGGL((k_resnorm_fwd<TX, TB, kLayer, 256, 1>), rows, dim3(256), 0, st, A);
  else if (vecs <= 512) hipLaunchKernelGGL((k_resnorm_fwd<TX, TB, kLayer, 256, 2>), rows, dim3(256), 0, st, A);
  else if (vecs <= 1024) hipLaunchKernelGGL((k_resnorm_fwd<TX, TB, kLayer, 512, 2>), rows, dim3(512), 0, st, A);
  else if (vecs <= 2048) hipLaunchKernelGGL((k_resnorm_fwd<TX, TB, kLayer, 1024, 2>), rows, dim3(1024), 0, st, A);
  else hipLaunchKernelGGL((k_resnorm_wide_fwd<TX, TB, kLayer>), rows, dim3(kWide), 0, st, A);
  return hipGetLastError();
}

template <typename TX, typename TB, bool kLayer>
hipError_t launch_bwd(const NormArgs& A, long chunks, hipStream_t st) {
  constexpr int V = vec_of<TB>();
  const int vecs = (A.D + V - 1) / V;
  const dim3 grid((unsigned)chunks);
  if (vecs <= 64) hipLaunchKernelGGL((k_resnorm_bwd<TX, TB, kLayer, 64, 1>), grid, dim3(256), 0, st, A);
  else if (vecs <= 128) hipLaunchKernelGGL((k_resnorm_bwd<TX, TB, kLayer, 64, 2>), grid, dim3(256), 0, st, A);
  else if (vecs <= 256) hipLaunchKernelGGL((k_resnorm_bwd<TX, TB, kLayer, 256, 1>), grid, dim3(256), 0, st, A);
  else if (vecs <= 512) hipLaunchKernelGGL((k_resnorm_bwd<TX, TB, kLayer, 256, 2>), grid, dim3(256), 0, st, A);
  else if (vecs <= 1024) hipLaunchKernelGGL((k_resnorm_bwd<TX, TB, kLayer, 512, 2>), grid, dim3(512), 0, st, A);
  else if (vecs <= 2048) hipLaunchKernelGGL((k_resnorm_bwd<TX, TB, kLayer, 1024, 2>), grid, dim3(1024), 0, st, A);
  else hipLaunchKernelGGL((k_resnorm_wide_bwd<TX, TB, kLayer>), grid, dim3(kWide), 0, st, A);
  return hipGetLastError();
}

// Calls f with the element types and the norm of a call as template arguments.
template <typename F>
hipError_t dispatch(int res_dtype, int dtype, int kind, F f) {
  auto kinds = [&](auto x, auto b) { return kind ? f(x, b, std::true_type{}) : f(x, b, std::false_type{}); };
  if (dtype == DT_F32) return kinds(0.0f, 0.0f);
  if (dtype == DT_F16) return res_dtype == DT_F32 ? kinds(0.0f, (_Float16)0.0f) : kinds((_Float16)0.0f, (_Float16)0.0f);
  return res_dtype == DT_F32 ? kinds(0.0f, (__bf16)0.0f) : kinds((__bf16)0.0f, (__bf16)0.0f);
}

// Runs of rows of the backward: enough workgroups for every CU's four SIMDs, but at least kMinRows rows each where
// there are that many, so that the partial rows stay a small part of the traffic.
struct NormPlan {
  long span, groups;                 // rows that share a gate row (all of them where none is shared), and how many such
  long per_chunk, chunks_per_group;  // rows of a run, runs of a span
  long chunks;
};
constexpr long kNormChunks = 512, kMinRows = 8;
NormPlan plan_norm(long rows, long gate_group) {
  NormPlan p;
  const long span = p.span = gate_group == 1 ? rows : gate_group;  // (a gate row for each row is not summed)
  p.groups = (rows + span - 1) / span;
  const long want = std::max(1L, kNormChunks / p.groups);
  p.per_chunk = std::min(span, std::max(kMinRows, (span + want - 1) / want));
  p.chunks_per_group = (span + p.per_chunk - 1) / p.per_chunk;
  p.chunks = p.groups * p.chunks_per_group;
  return p;
}

int check_norm(int res_dtype, int dtype, int kind, const void* x, const void* block, const void* gate, const void* post_w,
               double eps, long rows, int D, long gate_group) {
  auto known = [](int d) { return d == DT_F32 || d == DT_F16 || d == DT_BF16; };
  if (!known(res_dtype) || !known(dtype) || (res_dtype != dtype && res_dtype != DT_F32))
    return kans_fail(KANS_ERR_ARG, "residual dtype %d must be the block's (%d) or fp32", res_dtype, dtype);
  if (kind != 0 && kind != 1) return kans_fail(KANS_ERR_ARG, "norm kind %d, must be 0 (rms) or 1 (layer)", kind);
  if (rows < 0 || D <= 0) return kans_fail(KANS_ERR_ARG, "bad dims rows=%ld D=%d", rows, D);
  if (!(eps >= 0.0) || !std::isfinite(eps)) return kans_fail(KANS_ERR_ARG, "eps must be finite and >= 0");
  if (rows == 0) return 0;
  if (!x) return kans_fail(KANS_ERR_ARG, "null x");
  if (!block && (gate || post_w)) return kans_fail(KANS_ERR_ARG, "gate or post weight without a block");
  if (gate && (gate_group < 1 || gate_group > rows || rows % gate_group != 0))
    return kans_fail(KANS_ERR_ARG, "gate_group=%ld must divide the %ld rows", gate_group, rows);
  // a grid holds fewer than 2^32 threads along x, a row up to 1024
  if (rows >= (1L << 22)) return kans_fail(KANS_ERR_UNSUPPORTED, "rows=%ld, fewer than 2^22 fit a grid", rows);
  return 0;
}

}  // namespace
}  // namespace kans

using namespace kans;

extern "C" {

int kans_residual_norm_forward(int res_dtype, int dtype, int kind, const void* x, const void* block, const void* gate,
                               long gate_group, const void* post_w, const void* pre_w, const float* scale_dev, double scale,
                               double eps, void* y, void* h, float* stats, long rows, int D, void* stream) {
  int rc = check_norm(res_dtype, dtype, kind, x, block, gate, post_w, eps, rows, D, gate_group);
  if (rc || rows == 0) return rc;
  if (!h || (block && !y)) return kans_fail(KANS_ERR_ARG, "null output");
  std::lock_guard<std::mutex> lk(kans_mutex());
  if ((rc = kans_ensure_init())) return rc;
  NormArgs A{};
  A.x = x; A.block = block; A.gate = gate; A.post_w = post_w; A.pre_w = pre_w;
  A.scale_dev = scale_dev; A.scale = (float)scale; A.eps = (float)eps;
  A.y = y; A.h = h; A.stats = stats; A.rows = rows; A.gate_group = gate ? gate_group : rows; A.D = D;
  HIP_TRY(dispatch(res_dtype, dtype, kind, [&](auto tx, auto tb, auto layer) {
    return launch_fwd<decltype(tx), decltype(tb), decltype(layer)::value>(A, kans_caller_stream(stream));
  }));
  return 0;
}

long kans_residual_norm_workspace(long rows, int D, long gate_group) {
  if (rows <= 0 || D <= 0) return 0;
  const NormPlan p = plan_norm(rows, gate_group > 0 ? gate_group : rows);
  return p.chunks * (3L * D + 1) * (long)sizeof(float);
}

int kans_residual_norm_backward(int res_dtype, int dtype, int kind, const void* x, const void* block, const void* gate,
                                long gate_group, const void* post_w, const void* pre_w, const float* scale_dev, double scale,
                                double eps, const float* stats, const void* dy, const void* dh, void* dx, void* dblock,
                                void* dgate, int dgate_f32, void* dpost_w, void* dpre_w, float* dscale, long rows, int D,
                                void* workspace, long workspace_bytes, void* stream) {
  int rc = check_norm(res_dtype, dtype, kind, x, block, gate, post_w, eps, rows, D, gate_group);
  if (rc) return rc;
  if (rows == 0) return 0;
  if (!stats) return kans_fail(KANS_ERR_ARG, "null statistics");
  if ((dgate && !gate) || (dpost_w && !post_w) || (dpre_w && !pre_w) || (!block && (dblock || dscale)))
    return kans_fail(KANS_ERR_ARG, "gradient of an input that is not there");
  if (dgate_f32 && gate_group != 1) return kans_fail(KANS_ERR_ARG, "dgate_f32 needs a gate row for each row");
  const NormPlan p = plan_norm(rows, gate ? gate_group : rows);
  if (!workspace || workspace_bytes < p.chunks * (3L * D + 1) * (long)sizeof(float))
    return kans_fail(KANS_ERR_ARG, "workspace of %ld bytes, %ld needed", workspace ? workspace_bytes : 0,
                     p.chunks * (3L * D + 1) * (long)sizeof(float));
  std::lock_guard<std::mutex> lk(kans_mutex());
  if ((rc = kans_ensure_init())) return rc;
  hipStream_t st = kans_caller_stream(stream);
  NormArgs A{};
  A.x = x; A.block = block; A.gate = gate; A.post_w = post_w; A.pre_w = pre_w;
  A.scale_dev = scale_dev; A.scale = (float)scale; A.eps = (float)eps;
  A.stats = (float*)stats; A.rows = rows; A.D = D;
  A.gate_group = gate ? gate_group : rows;
  A.dy = dy; A.dh = dh; A.dx = dx; A.dblock = dblock; A.dgate = dgate;
  A.part_scale = (float*)workspace;
  A.part = (float*)workspace + p.chunks;
  A.span = p.span;
  A.per_chunk = p.per_chunk;
  A.chunks_per_group = p.chunks_per_group;
  A.at_pre = dpre_w ? A.parts++ : -1;
  A.at_post = dpost_w ? A.parts++ : -1;
  A.at_gate = dgate && gate_group > 1 ? A.parts++ : -1;
  A.want_scale = dscale != nullptr;
  A.gate_f32 = dgate_f32;
  HIP_TRY(dispatch(res_dtype, dtype, kind, [&](auto tx, auto tb, auto layer) {
    return launch_bwd<decltype(tx), decltype(tb), decltype(layer)::value>(A, p.chunks, st);
  }));
  if (A.parts == 0 && !dscale) return 0;
  ReduceArgs R{};
  R.part = A.part; R.part_scale = A.part_scale;
  R.dpre = dpre_w; R.dpost = dpost_w; R.dgate = dgate; R.dscale = dscale;
  R.chunks = p.chunks; R.chunks_per_group = p.chunks_per_group;
  R.D = D; R.parts = A.parts; R.at_pre = A.at_pre; R.at_post = A.at_post; R.at_gate = A.at_gate;
  R.col_tiles = (D + 63) / 64;
  R.groups = p.groups;
  const long outs = (A.at_pre >= 0) + (A.at_post >= 0) + (A.at_gate >= 0 ? p.groups : 0);
  const dim3 grid((unsigned)std::min(outs * R.col_tiles + (dscale ? 1 : 0), 1L << 16));
  auto* reduce = dtype == DT_F16 ? k_resnorm_reduce<_Float16> : dtype == DT_BF16 ? k_resnorm_reduce<__bf16> : k_resnorm_reduce<float>;
  hipLaunchKernelGGL(reduce, grid, dim3(1024), 0, st, R);
  HIP_TRY(hipGetLastError());
  return 0;
}

}  // extern "C"
