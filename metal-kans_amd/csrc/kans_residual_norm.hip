// Norms before and after a block, fused with its gate and residual scale (gfx950).
//
//   b^ = N(block),  u = post_w b^,  y = x + scale gate u,  h = pre_w N(y)
//   rms:   N(a) = a / sqrt(mean(a^2) + eps)
//   layer: N(a) = (a - mean(a)) / sqrt(var(a) + eps)
//
// Backward, from dy and dh (y^ = N(y), r = the reciprocal in N, q = pre_w dh; means over the row):
//   T = dy + r_y (q - y^ mean(q y^) [- mean(q)])           layer terms in brackets
//   dx = T,  dpre_w = sum dh y^,  dgate = sum scale T u
//   du = scale gate T,  dpost_w = sum du b^,  p = post_w du
//   dblock = r_b (p - b^ mean(p b^) [- mean(p)]),  dscale = sum T gate u = sum p b^ / scale
//
// All of it is bound by memory: the forward reads x, block (and a full gate) and
// writes y and h once; the backward reads x, block, dy, dh and writes dx and dblock.
// It takes y from x and block again (fp32, never rounded) instead of reading the
// stored one: the same bytes, and no rounding of y enters the gradients.  Rows
// live in registers, 8 elements a thread; the forward's statistics are kept
// (fp32, 2 or 4 a row) so that the backward needs two row sums.
//
// Sums over rows (weights, a shared gate, the scale): a workgroup takes a run
// of rows that share their gate row, adds up in fp32 registers and writes one partial row; a
// second kernel adds the partial rows in a fixed order.  Where few rows share a gate row a run is several whole
// groups of them: it writes each group's gradient itself and one partial row of the rest.  No atomics: the same bits on
// every run.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kans_api_internal.h"
#include "kans_wave.h"

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
  float* part_scale;       // [chunks] doubles at 4-byte addresses
  long span, groups, per_chunk, chunks_per_group, whole;  // the runs of rows: NormPlan
  int parts, at_pre, at_post, at_gate;  // rows of a chunk's partials, -1: not asked for
  int want_scale, gate_f32;  // gate_f32: dgate of a gate row for each row in fp32
};

constexpr int V = 8;  // elements of a thread: one 16-byte access in 16 bits, two in fp32

// V elements as they lie in memory (16-bit ones stay packed in their registers).
template <typename T> struct Raw { unsigned w[V * sizeof(T) / 4]; };

template <typename T>
__device__ __forceinline__ float get(const Raw<T>& r, int e) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[e]);
  else if constexpr (std::is_same_v<T, __bf16>) return __uint_as_float(e & 1 ? r.w[e / 2] & 0xffff0000u : r.w[e / 2] << 16);
  else return (float)__builtin_bit_cast(_Float16, (unsigned short)(r.w[e / 2] >> (16 * (e & 1))));
}

// Makes the compiler take the packed values anew from here on, instead of keeping what it
// has unpacked or computed from them before: a few instructions for many registers.
template <typename T>
__device__ __forceinline__ void repack(Raw<T>& r) {
#pragma unroll
  for (int i = 0; i < (int)(V * sizeof(T) / 4); ++i) asm volatile("" : "+v"(r.w[i]));
}

template <typename T>
__device__ __forceinline__ Raw<T> fill_raw(float v) {
  Raw<T> r;
  const T t = from_f32<T>(v);
#pragma unroll
  for (int i = 0; i < (int)(V * sizeof(T) / 4); ++i) {
    if constexpr (sizeof(T) == 4) r.w[i] = __builtin_bit_cast(unsigned, t);
    else r.w[i] = __builtin_bit_cast(unsigned short, t) * 0x10001u;
  }
  return r;
}

// V elements of a row of D from p on, of which `left` exist (maybe none), 0 for the others.  Rows start at any element:
// the device takes wide accesses at any address.
template <typename T>
__device__ __forceinline__ Raw<T> load_part(const T* p, int left) {
  Raw<T> r;
  if (left >= V) {
    __builtin_memcpy(&r, p, sizeof(r));
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < V; ++e) r.w[e] = e < left ? ((const unsigned*)p)[e] : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const unsigned short* q = (const unsigned short*)p;
      r.w[i] = (2 * i < left ? q[2 * i] : 0u) | (2 * i + 1 < left ? (unsigned)q[2 * i + 1] << 16 : 0u);
    }
  }
  return r;
}
// The same in two steps: load_raw asks for the values, settle makes them usable.  In 16 bits the narrow loads at the end of
// a row are put together at once, which waits for them, and with them for all loads that are under way.  So there (kShift) a
// thread at the end of the row reads its last V elements instead, in the one access that all make, and settle moves them to
// their places: 30000 x 2047 bf16, forward 143 -> 94 us, both directions 589 -> 309; 10000 x 7000: 125 -> 122, 443 -> 360.  (fp32,
// with nothing to put together, is 5 - 10 % slower so.)  `here` elements exist from p on, `left` of them count: all, or
// none in a row that is not there (p is then another row's).
template <typename T> constexpr bool shifts() { return sizeof(T) == 2; }
template <bool kShift, typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* p, int here, int left, int D) {
  if constexpr (!kShift) return load_part(p, left);
  if (D < V) return load_part(p, here);
  Raw<T> r;
  __builtin_memcpy(&r, p - max(V - here, 0), sizeof(r));
  return r;
}
template <bool kShift, typename T>
__device__ __forceinline__ void settle(Raw<T>& r, int left, int D) {
  if constexpr (kShift) {
    const int back = min(max(V - left, 0), V);
    if (!__builtin_amdgcn_ballot_w64(back != 0)) return;
    if (D >= V) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) r.w[i] = back & 1 ? r.w[i] >> 16 | (i + 1 < V / 2 ? r.w[i + 1] << 16 : 0u) : r.w[i];
#pragma unroll
      for (int by = 1; by < V / 2; by *= 2)
#pragma unroll
        for (int i = 0; i < V / 2; ++i) r.w[i] = back & 2 * by ? (i + by < V / 2 ? r.w[i + by] : 0u) : r.w[i];
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.w[i] = back == V ? 0u : r.w[i];
  }
}
template <typename T>
__device__ __forceinline__ Raw<T> load_or_one(const T* p, long at, int left) {
  return p ? load_part(p + at, left) : fill_raw<T>(1.0f);
}
// Results leave nontemporal: lines that are written whole need not be read or kept.  y and h of 2048 x 4096 bf16: 12.1 us
// (plain stores 16.4), of 16384 x 4096: 80 (112); with an operation behind them that reads both: 23.5 (26.5) and 161 (185).
// (Nontemporal loads as well: 14.7 and 94 us, as what a caller has just written is no longer found in a cache.)
template <typename T> using Wide = unsigned __attribute__((ext_vector_type(4), aligned(sizeof(T))));
template <typename T>
__device__ __forceinline__ void store_vec(T* p, int left, const float* o) {
  T v[V];
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = from_f32<T>(o[e]);
  if (left >= V) {
    Wide<T> w[sizeof(v) / 16];
    __builtin_memcpy(w, v, sizeof(v));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(v) / 16); ++i) __builtin_nontemporal_store(w[i], (Wide<T>*)p + i);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < left) p[e] = v[e];
  }
}

// Sums of a and b over the TPR threads of a row, in each of them.  `slot` (0 or 1)
// alternates between consecutive calls: the barrier of a call then also separates the reads of the
// call before from the writes of the next.
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float (*lds)[2][16], int slot) {
  a = wave_sum(a);
  b = wave_sum(b);
  if constexpr (TPR > 64) {
    const int wave = threadIdx.x >> 6, first = threadIdx.x / TPR * (TPR / 64);
    if ((threadIdx.x & 63) == 0) {
      lds[slot][0][wave] = a;
      lds[slot][1][wave] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) {
      a += lds[slot][0][first + w];
      b += lds[slot][1][first + w];
    }
  }
}

// Mean (layer) and reciprocal size of a row, of which this thread holds `left` elements in v (zeros behind them).
template <bool kLayer, int TPR>
__device__ __forceinline__ void row_stats(const float (&v)[V], int left, int D, float eps, float (*lds)[2][16], int& slot,
                                          float& mean, float& r) {
  float s = 0.0f, none = 0.0f;
  mean = 0.0f;
  if constexpr (kLayer) {
#pragma unroll
    for (int e = 0; e < V; ++e) s += v[e];
    row_sum2<TPR>(s, none, lds, slot);
    slot ^= 1;
    mean = s / (float)D;
    s = none = 0.0f;
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float c = e < left ? v[e] - mean : 0.0f;
    s += c * c;
  }
  row_sum2<TPR>(s, none, lds, slot);
  slot ^= 1;
  r = 1.0f / __builtin_sqrtf(s / (float)D + eps);
}

// Threads of a workgroup, and the rows that it takes at a time.
template <int TPR> constexpr int threads_of() { return TPR > 512 ? TPR : 512; }
template <int TPR> constexpr int rows_of() { return threads_of<TPR>() / TPR; }

// Bound by HBM: 16384 x 4096 bf16 (537 MB) in 80 us where the inputs are partly in a cache (6.7 TB/s), 90 - 105 cold.  One row's worth of threads
// a row with 8 elements each: two vectors a thread (half the threads) took 137 us.  A single row of 4096 is 8 waves and two
// barriers; its call is bound by the launch.
template <typename TX, typename TB, bool kLayer, int TPR>
__global__ __launch_bounds__(threads_of<TPR>()) void k_resnorm_fwd(const NormArgs A) {
  __shared__ float lds[2][2][16];
  const long row = (long)blockIdx.x * rows_of<TPR>() + threadIdx.x / TPR;
  const int at = threadIdx.x % TPR * V, D = A.D, here = D - at, left = row < A.rows ? here : 0;  // elements of this thread
  const long there = min(row, A.rows - 1), base = there * D + at;  // (a row that is not there reads the last)
  constexpr bool kx = shifts<TX>(), kb = shifts<TB>();
  Raw<TX> x = load_raw<kx>((const TX*)A.x + base, here, left, D);
  int slot = 0;
  float y[V], mean_b = 0.0f, r_b = 0.0f;
  auto load_or_one = [&](const void* p, long from) {
    return p ? load_raw<kb>((const TB*)p + from, here, left, D) : fill_raw<TB>(1.0f);
  };
  Raw<TB> nw = load_or_one(A.pre_w, at);
  if (A.block) {
    Raw<TB> bv = load_raw<kb>((const TB*)A.block + base, here, left, D);
    Raw<TB> g = load_or_one(A.gate, there / A.gate_group * D + at), pw = load_or_one(A.post_w, at);
    settle<kb>(bv, left, D);
    settle<kx>(x, left, D);
    settle<kb>(g, left, D);
    settle<kb>(pw, left, D);
    const float scale = A.scale_dev ? *A.scale_dev : A.scale;
    float b[V];
#pragma unroll
    for (int e = 0; e < V; ++e) b[e] = get(bv, e);
    row_stats<kLayer, TPR>(b, left, D, A.eps, lds, slot, mean_b, r_b);
#pragma unroll
    for (int e = 0; e < V; ++e)
      y[e] = e < left ? get(x, e) + scale * get(g, e) * ((b[e] - mean_b) * r_b * get(pw, e)) : 0.0f;
    store_vec((TX*)A.y + base, left, y);
  } else {
    settle<kx>(x, left, D);
#pragma unroll
    for (int e = 0; e < V; ++e) y[e] = get(x, e);
  }
  settle<kb>(nw, left, D);
  float mean_y, r_y, h[V];
  row_stats<kLayer, TPR>(y, left, D, A.eps, lds, slot, mean_y, r_y);
#pragma unroll
  for (int e = 0; e < V; ++e) h[e] = (y[e] - mean_y) * r_y * get(nw, e);
  store_vec((TB*)A.h + base, left, h);
  if (A.stats && at == 0 && row < A.rows) {
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
template <typename TX, typename TB>
struct RowIn {
  Raw<TX> x, dy;
  Raw<TB> b, dh, g;
  float r_b, r_y, mean_b, mean_y;
};

// Asks for row `row`, and with gate_at >= 0 for the gate's elements from there on; a row behind `last` is not there, and its
// values are zeros, which add nothing to any sum.
template <typename TX, typename TB, bool kLayer>
__device__ __forceinline__ void load_row(RowIn<TX, TB>& in, const NormArgs& A, long row, long last, int at, long gate_at) {
  constexpr bool kx = shifts<TX>(), kb = shifts<TB>();
  const bool there = row <= last;
  const int D = A.D, here = D - at, left = there ? here : 0;
  row = min(row, last);
  const long base = row * D + at;
  in.x = load_raw<kx>((const TX*)A.x + base, here, left, D);
  if (A.dy) in.dy = load_raw<kx>((const TX*)A.dy + base, here, left, D);
  if (A.dh) in.dh = load_raw<kb>((const TB*)A.dh + base, here, left, D);
  if (A.block) in.b = load_raw<kb>((const TB*)A.block + base, here, left, D);
  if (gate_at >= 0) in.g = load_raw<kb>((const TB*)A.gate + gate_at, here, left, D);
  const float* s = A.stats + row * (kLayer ? 4 : 2);
  in.r_b = there ? s[0] : 0.0f;
  in.r_y = there ? s[1] : 0.0f;
  in.mean_b = kLayer && there ? s[2] : 0.0f;
  in.mean_y = kLayer && there ? s[3] : 0.0f;
}

// One workgroup takes the rows of a run, rows_of<TPR>() at a time, with the next ones' loads in flight (at
// 1024 threads the 128 registers that a thread may have do not hold them too).  Two workgroups a CU, with
// up to 256 registers: held to 128 the kernel spills, and 16384 x 4096 bf16 (805 MB) take 600 us instead of 155 - 190
// (4.2 - 5.2 TB/s).  whole: the run is several whole gate groups (a kernel of its own: the rows' bookkeeping in all of them
// spilled at 1024 threads, 8192 x 8192 fp32 both directions 580 -> 628 us).
template <typename TX, typename TB, bool kLayer, int TPR, bool whole>
__global__ __launch_bounds__(threads_of<TPR>(), TPR > 512 ? 4 : 2) void k_resnorm_bwd(const NormArgs A) {
  constexpr int ROWS = rows_of<TPR>();
  __shared__ float lds[2][2][16];
  constexpr bool kAhead = TPR <= 512;
  __shared__ float sums[ROWS > 1 ? TPR * V : 1];
  __shared__ float4 kept[kAhead ? 1 : 3 * V / 4 * TPR];
  __shared__ double sum_scale[ROWS];  // of the rows that each `sub` has done
  const int at = threadIdx.x % TPR * V, sub = threadIdx.x / TPR;
  const int D = A.D, left = D - at;
  const long chunk = blockIdx.x;
  const bool gate_rows = !whole && A.gate && A.gate_group == 1;
  // the rows at a time, one for each `sub`: consecutive ones of the run from row0 on, or row in_group of ROWS consecutive
  // groups from group0 on
  long row0 = 0, end, group0;
  int in_group = 0;
  if constexpr (whole) {
    group0 = chunk * A.whole;
    end = min(group0 + A.whole, A.groups);  // in groups
  } else {
    group0 = chunk / A.chunks_per_group;
    row0 = group0 * A.span + (chunk - group0 * A.chunks_per_group) * A.per_chunk;
    end = min(min(row0 + A.per_chunk, (group0 + 1) * A.span), A.rows);
  }
  const long last = (whole ? end * A.span : end) - 1;
  const float scale = A.scale_dev ? *A.scale_dev : A.scale;
  Raw<TB> pw = load_or_one((const TB*)A.post_w, at, left), nw = load_or_one((const TB*)A.pre_w, at, left);
  RowIn<TX, TB> next{};
  if (!gate_rows && !whole) next.g = load_or_one((const TB*)A.gate, group0 * D + at, left);
  auto ask = [&](long r, long g, int in) {  // for the rows at a time from row r on, or row `in` of the groups from g on
    const long row = whole ? (g + sub) * A.span + in : r + sub;
    const long own = gate_rows ? min(row, last) : whole && in == 0 ? min(g + sub, end - 1) : -1;
    load_row<TX, TB, kLayer>(next, A, row, last, at, own < 0 ? -1L : own * D + at);
  };
  // sums of this thread's columns over the run's rows: pre_w, post_w, gate.  At 1024 threads a row they lie in LDS, each
  // thread its own, so that the rest fits in 128 registers: 8192 x 8192 bf16, both directions, 382 -> 310 us, fp32 780 -> 585.
  float s[kAhead ? 3 : 1][V];
  auto kept_at = [&](int k, int i) { return &kept[(k * (V / 4) + i) * TPR + threadIdx.x]; };
  auto add_up = [&](int k, const float(&v)[V]) {
    if constexpr (kAhead) {
#pragma unroll
      for (int e = 0; e < V; ++e) s[k][e] += v[e];
    } else {
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        float4 o = *kept_at(k, i);
        o.x += v[4 * i]; o.y += v[4 * i + 1]; o.z += v[4 * i + 2]; o.w += v[4 * i + 3];
        *kept_at(k, i) = o;
      }
    }
  };
#pragma unroll
  for (int k = 0; k < 3; ++k)
    if constexpr (kAhead) {
#pragma unroll
      for (int e = 0; e < V; ++e) s[k][e] = 0.0f;
    } else {
#pragma unroll
      for (int i = 0; i < V / 4; ++i) *kept_at(k, i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
  if (at == 0) sum_scale[sub] = 0.0;
  const float inv_d = 1.0f / (float)D;
  if (kAhead) ask(row0, group0, 0);
  while (whole ? group0 < end : row0 < end) {
    if (!kAhead) ask(row0, group0, in_group);
    RowIn<TX, TB> in = next;
    const int then_in = whole && in_group + 1 < A.span ? in_group + 1 : 0;
    const long then_group = whole && then_in == 0 ? group0 + ROWS : group0, then_row = row0 + ROWS;
    if (kAhead && (whole ? then_group < end : then_row < end)) ask(then_row, then_group, then_in);
    const long group = group0 + sub, row = whole ? group * A.span + in_group : row0 + sub;
    const long base = row * D + at;
    const int out = row <= last ? left : 0;
    constexpr bool kx = shifts<TX>(), kb = shifts<TB>();
    settle<kx>(in.x, out, D);
    settle<kx>(in.dy, out, D);
    settle<kb>(in.dh, out, D);
    settle<kb>(in.b, out, D);
    if (gate_rows || (whole && in_group == 0)) settle<kb>(in.g, out, D);
    if (whole && in_group == 0) next.g = in.g;  // (two rows at least share it)
    auto bn = [&](int e) { return e < left ? (get(in.b, e) - in.mean_b) * in.r_b : 0.0f; };
    auto yn = [&](int e) {
      const float y = get(in.x, e) + scale * get(in.g, e) * (bn(e) * get(pw, e));
      return e < left ? (y - in.mean_y) * in.r_y : 0.0f;
    };
    float t[V], add[V], sa = 0.0f, sb = 0.0f;
    repack(pw);
    repack(nw);
    repack(in.g);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float dh = get(in.dh, e), q = get(nw, e) * dh, n = yn(e);
      add[e] = dh * n;
      sa += q * n;
      sb += q;
    }
    add_up(0, add);
    row_sum2<TPR>(sa, sb, lds, 0);
    sa *= inv_d;
    sb = kLayer ? sb * inv_d : 0.0f;
    float pa = 0.0f, pb = 0.0f, dg[V];  // means of p b^ and p without the scale, so that the first sums up to its gradient too
    repack(in.x);
    repack(in.b);
    repack(in.dh);
    repack(in.g);
    repack(pw);
    repack(nw);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float q = get(nw, e) * get(in.dh, e), g = get(in.g, e), b = bn(e), u = b * get(pw, e);
      t[e] = get(in.dy, e) + in.r_y * (q - yn(e) * sa - sb);
      dg[e] = scale * t[e] * u;
      const float du = g * t[e], p = du * get(pw, e);
      add[e] = scale * du * b;
      pa += p * b;
      pb += e < left ? p : 0.0f;
    }
    add_up(1, add);
    add_up(2, dg);
    if (whole && A.dgate && then_in == 0) {  // the group's last row
      float v[V];
      if constexpr (kAhead) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          v[e] = s[2][e];
          s[2][e] = 0.0f;
        }
      } else {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
          __builtin_memcpy(v + 4 * i, kept_at(2, i), 16);
          *kept_at(2, i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
      }
      store_vec((TB*)A.dgate + group * D + at, out, v);
    }
    if (A.dx) store_vec((TX*)A.dx + base, out, t);
    if (gate_rows && A.dgate) {
      if (A.gate_f32) store_vec((float*)A.dgate + base, out, dg);
      else store_vec((TB*)A.dgate + base, out, dg);
    }
    row_sum2<TPR>(pa, pb, lds, 1);
    if (at == 0 && row <= last) sum_scale[sub] += (double)pa;
    if (A.dblock) {
      pa *= scale * inv_d;
      pb = kLayer ? pb * (scale * inv_d) : 0.0f;
      float db[V];
      repack(in.b);
      repack(in.g);
      repack(pw);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float p = scale * get(in.g, e) * t[e] * get(pw, e);
        db[e] = in.r_b * (p - bn(e) * pa - pb);
      }
      store_vec((TB*)A.dblock + base, out, db);
    }
    row0 = then_row;
    group0 = then_group;
    in_group = then_in;
  }
  // the run's partial rows; where several rows go at a time, those of the same columns one after the other
  float* part = A.part + chunk * A.parts * D;
  auto put = [&](int at_part, int k) {
    if (at_part < 0) return;
    float* o = part + (long)at_part * D;
    if constexpr (!kAhead) {
      float v[V];
#pragma unroll
      for (int i = 0; i < V / 4; ++i) __builtin_memcpy(v + 4 * i, kept_at(k, i), 16);
      store_vec(o + at, left, v);
    } else if constexpr (ROWS == 1) {
      store_vec(o + at, left, s[k]);
    } else {
      for (int w = 0; w < ROWS; ++w) {
        if (sub == w) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            float* c = &sums[e * TPR + threadIdx.x % TPR];
            *c = w == 0 ? s[k][e] : *c + s[k][e];
          }
        }
        __syncthreads();
      }
      for (int j = threadIdx.x; j < D; j += threads_of<TPR>()) o[j] = sums[j % V * TPR + j / V];
      __syncthreads();
    }
  };
  put(A.at_pre, 0);
  put(A.at_post, 1);
  put(A.at_gate, 2);
  if (A.want_scale) {
    __syncthreads();
    if (threadIdx.x == 0) {
      double all = sum_scale[0];
      for (int w = 1; w < ROWS; ++w) all += sum_scale[w];
      __builtin_memcpy(A.part_scale + 2 * chunk, &all, sizeof(all));
    }
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

// A chunk's rows one after the other; the partial rows are added up in memory, each column by one thread (of whole groups the
// gate's row is that of the group under way).
template <typename TX, typename TB, bool kLayer>
__global__ __launch_bounds__(kWide) void k_resnorm_wide_bwd(const NormArgs A) {
  __shared__ float lds[2][2][16];
  const int D = A.D;
  const long chunk = blockIdx.x, group = A.whole ? chunk * A.whole : chunk / A.chunks_per_group;
  const long first = A.whole ? group * A.span : group * A.span + (chunk - group * A.chunks_per_group) * A.per_chunk;
  const long end = min(A.whole ? (group + A.whole) * A.span : min(first + A.per_chunk, (group + 1) * A.span), A.rows);
  const TB *pw = (const TB*)A.post_w, *nw = (const TB*)A.pre_w;
  const float scale = A.scale_dev ? *A.scale_dev : A.scale, inv_d = 1.0f / (float)D;
  float* part = A.part + chunk * A.parts * D;
  for (int j = threadIdx.x; j < D; j += kWide)
    for (int k = 0; k < A.parts; ++k) part[(long)k * D + j] = 0.0f;
  double s_scale = 0.0;
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
      const float t = T(j), n = bn(j), u = n * post(j), du = gt(j) * t, p = du * post(j);
      if (A.dx) ((TX*)A.dx)[row * D + j] = from_f32<TX>(t);
      if (A.dgate && A.gate_group == 1) {
        if (A.gate_f32) ((float*)A.dgate)[row * D + j] = scale * t * u;
        else ((TB*)A.dgate)[row * D + j] = from_f32<TB>(scale * t * u);
      }
      if (A.at_pre >= 0 && dh) part[(long)A.at_pre * D + j] += to_f32(dh[j]) * yn(j);
      if (A.at_post >= 0) part[(long)A.at_post * D + j] += scale * du * n;
      if (A.at_gate >= 0) part[(long)A.at_gate * D + j] += scale * t * u;
      pa += p * n;
      pb += p;
    }
    row_sum2<kWide>(pa, pb, lds, 1);
    s_scale += (double)pa;
    pa *= scale * inv_d;
    pb = kLayer ? pb * (scale * inv_d) : 0.0f;
    if (A.whole && A.at_gate >= 0 && (row + 1) % A.span == 0)
      for (int j = threadIdx.x; j < D; j += kWide) {
        float* sum = part + (long)A.at_gate * D + j;
        ((TB*)A.dgate)[row / A.span * D + j] = from_f32<TB>(*sum);
        *sum = 0.0f;
      }
    if (A.block && A.dblock)
      for (int j = threadIdx.x; j < D; j += kWide) {
        const float p = scale * gt(j) * T(j) * post(j);
        ((TB*)A.dblock)[row * D + j] = from_f32<TB>(r_b * (p - bn(j) * pa - pb));
      }
  }
  if (A.want_scale && threadIdx.x == 0) __builtin_memcpy(A.part_scale + 2 * chunk, &s_scale, sizeof(s_scale));
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

// Sum over a workgroup in 64 bits, in its first thread.  The scale's gradient is one number of terms of both signs; all else
// here is a sum along one row or column.
__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
  if (threadIdx.x == 0)
    for (int w = 0; w < (int)blockDim.x / 64; ++w) v += lds[w];
  return v;
}

// 16384 x 4096: 512 partial rows of 3 x 4096 in 7 us (25 MB, mostly from the last-level cache).
// A workgroup adds 64 columns of one output row at a time: 16 runs of partial rows, joined in a fixed order.
// Work by column tile and output row: dpre, dpost, then dgate's groups, and last the scale.
template <typename TB>
__global__ __launch_bounds__(1024) void k_resnorm_reduce(const ReduceArgs A) {
  __shared__ alignas(8) float lds[16][64];
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
#pragma unroll 8
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
    double s = 0.0;
    for (long c = threadIdx.x; c < A.chunks; c += 1024) {
      double of_chunk;
      __builtin_memcpy(&of_chunk, A.part_scale + 2 * c, sizeof(of_chunk));
      s += of_chunk;
    }
    s = block_sum(s, (double*)&lds[0][0]);
    if (threadIdx.x == 0) *A.dscale = (float)s;
  }
}

// ---- launches ---------------------------------------------------------------------------------------
// Calls go(threads a row) with the fewest threads that hold a row, or 0 where no workgroup does.
template <typename F>
void by_width(int D, F go) {
  const int vecs = (D + V - 1) / V;
  if (vecs <= 64) go(std::integral_constant<int, 64>{});
  else if (vecs <= 128) go(std::integral_constant<int, 128>{});
  else if (vecs <= 256) go(std::integral_constant<int, 256>{});
  else if (vecs <= 512) go(std::integral_constant<int, 512>{});
  else if (vecs <= 1024) go(std::integral_constant<int, 1024>{});
  else go(std::integral_constant<int, 0>{});
}

template <typename TX, typename TB, bool kLayer>
hipError_t launch_fwd(const NormArgs& A, hipStream_t st) {
  by_width(A.D, [&](auto width) {
    constexpr int TPR = decltype(width)::value;
    if constexpr (TPR == 0)
      hipLaunchKernelGGL((k_resnorm_wide_fwd<TX, TB, kLayer>), dim3((unsigned)A.rows), dim3(kWide), 0, st, A);
    else
      hipLaunchKernelGGL((k_resnorm_fwd<TX, TB, kLayer, TPR>), dim3((unsigned)((A.rows + rows_of<TPR>() - 1) / rows_of<TPR>())),
                         dim3(threads_of<TPR>()), 0, st, A);
  });
  return hipGetLastError();
}

template <typename TX, typename TB, bool kLayer>
hipError_t launch_bwd(const NormArgs& A, long chunks, hipStream_t st) {
  by_width(A.D, [&](auto width) {
    constexpr int TPR = decltype(width)::value;
    if constexpr (TPR == 0)
      hipLaunchKernelGGL((k_resnorm_wide_bwd<TX, TB, kLayer>), dim3((unsigned)chunks), dim3(kWide), 0, st, A);
    else
      hipLaunchKernelGGL((A.whole ? k_resnorm_bwd<TX, TB, kLayer, TPR, true> : k_resnorm_bwd<TX, TB, kLayer, TPR, false>),
                         dim3((unsigned)chunks), dim3(threads_of<TPR>()), 0, st, A);
  });
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
// there are that many, so that the partial rows stay a small part of the traffic.  Groups of fewer rows than such a run
// go several to a run, a number that its rows at a time share evenly (16384 x 4096 in groups of 2, bf16: 512 runs,
// 25 MB of partial rows; a run for each group was 8192 and 403 MB, three times x).
struct NormPlan {
  long span, groups;                 // rows that share a gate row (all of them where none is shared), and how many such
  long per_chunk, chunks_per_group;  // rows of a run, runs of a span
  long whole;                        // or whole groups of a run (0: a run lies in one)
  long chunks;
};
constexpr long kNormChunks = 512, kMinRows = 8;
NormPlan plan_norm(long rows, int D, long gate_group) {
  NormPlan p{};
  const long span = p.span = gate_group == 1 ? rows : gate_group;  // (a gate row for each row is not summed)
  p.groups = (rows + span - 1) / span;
  const long run = std::max(kMinRows, (rows + kNormChunks - 1) / kNormChunks);
  if (p.groups > 1 && span < run) {
    long at_a_time = 1;
    by_width(D, [&](auto width) {
      if constexpr (decltype(width)::value != 0) at_a_time = rows_of<decltype(width)::value>();
    });
    p.whole = (run / span + at_a_time - 1) / at_a_time * at_a_time;
    p.chunks = (p.groups + p.whole - 1) / p.whole;
    return p;
  }
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
  const NormPlan p = plan_norm(rows, D, gate_group > 0 ? gate_group : rows);
  return p.chunks * (3L * D + 2) * (long)sizeof(float);
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
  const NormPlan p = plan_norm(rows, D, gate ? gate_group : rows);
  if (!workspace || workspace_bytes < p.chunks * (3L * D + 2) * (long)sizeof(float))
    return kans_fail(KANS_ERR_ARG, "workspace of %ld bytes, %ld needed", workspace ? workspace_bytes : 0,
                     p.chunks * (3L * D + 2) * (long)sizeof(float));
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
  A.part = (float*)workspace + 2 * p.chunks;
  A.span = p.span;
  A.groups = p.groups;
  A.whole = p.whole;
  A.per_chunk = p.per_chunk;
  A.chunks_per_group = p.chunks_per_group;
  A.at_pre = dpre_w ? A.parts++ : -1;
  A.at_post = dpost_w ? A.parts++ : -1;
  const bool kept = p.whole && D <= 1024 * V;  // (the groups' sums stay in the registers of a workgroup)
  A.at_gate = dgate && gate_group > 1 && !kept ? A.parts++ : -1;
  A.want_scale = dscale != nullptr;
  A.gate_f32 = dgate_f32;
  HIP_TRY(dispatch(res_dtype, dtype, kind, [&](auto tx, auto tb, auto layer) {
    return launch_bwd<decltype(tx), decltype(tb), decltype(layer)::value>(A, p.chunks, st);
  }));
  if (!dpre_w && !dpost_w && !dscale && (A.at_gate < 0 || p.whole)) return 0;
  ReduceArgs R{};
  R.part = A.part; R.part_scale = A.part_scale;
  R.dpre = dpre_w; R.dpost = dpost_w; R.dgate = dgate; R.dscale = dscale;
  R.chunks = p.chunks; R.chunks_per_group = p.chunks_per_group;
  R.D = D; R.parts = A.parts; R.at_pre = A.at_pre; R.at_post = A.at_post; R.at_gate = p.whole ? -1 : A.at_gate;
  R.col_tiles = (D + 63) / 64;
  R.groups = p.groups;
  const long outs = (R.at_pre >= 0) + (R.at_post >= 0) + (R.at_gate >= 0 ? p.groups : 0);
  const dim3 grid((unsigned)std::min(outs * R.col_tiles + (dscale ? 1 : 0), 1L << 16));
  auto* reduce = dtype == DT_F16 ? k_resnorm_reduce<_Float16> : dtype == DT_BF16 ? k_resnorm_reduce<__bf16> : k_resnorm_reduce<float>;
  hipLaunchKernelGGL(reduce, grid, dim3(1024), 0, st, R);
  HIP_TRY(hipGetLastError());
  return 0;
}

}  // extern "C"
