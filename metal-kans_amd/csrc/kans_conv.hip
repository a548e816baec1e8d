// Short causal convolution along the sequence, channel by channel, with its activation (gfx950).
//
//   u[t] = bias + sum_j w[j] x[t - W + 1 + j],   y[t] = u[t] sigmoid(u[t])  (or u[t])
//   du[t] = dy[t] y'(u[t]),   dx[t] = sum_j w[j] du[t + W - 1 - j],   dw[j] = sum_t du[t] x[t - W + 1 + j],   dbias = sum_t du[t]
//
// Inputs before the first step are the state (zeros without one); steps behind a sequence's length count as zeros.
//
// Bound by memory: the forward reads x and writes y, the backward reads x and dy and writes dx (u is computed again).
// Channels lie side by side, so a thread takes a few neighbouring ones and walks a tile of steps with the last W - 1
// inputs in registers; a tile reads W - 1 steps of its neighbour again.  Sums over steps and sequences: a tile writes
// one partial row for each tap and the bias, and a second kernel adds the rows in a fixed order.  The inputs of the next 8
// (backward 4) steps are under way while those before are computed; with one step at a time the kernels waited for memory.
// bf16 8 x 2048 x 4096, 4 taps: forward 55 us (268 MB, 4.9 TB/s), with single steps 100; backward 80 (455 MB, 5.7 TB/s) and
// 143, its reduction 7.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kans_api_internal.h"

namespace kans {
namespace {

constexpr int kMaxTaps = 8;

struct ConvArgs {
  const void *x, *w, *bias, *dy;
  void *y, *state, *dx;
  const int64_t* lengths;
  float* part;                 // [tiles of all sequences][W + 1][D]
  long x_batch, x_row;         // elements between sequences and between steps of x
  int B, L, D, tile, tiles;    // tile: steps of a thread, tiles: of a sequence
  int vecs;                    // threads beside each other along the channels
  int silu;
};

// V neighbouring channels as they lie in memory, at any address (the device takes wide accesses anywhere).
template <typename T, int V> struct Vec { T v[V]; };
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
  Vec<T, V> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void load(float (&o)[V], const T* p) {
  const Vec<T, V> v = load_vec<T, V>(p);
#pragma unroll
  for (int e = 0; e < V; ++e) o[e] = to_f32(v.v[e]);
}
// Without the first `skip` channels.  Results leave nontemporal: lines that are written whole need not be read or kept.
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&o)[V], int skip) {
  typedef unsigned Wide __attribute__((ext_vector_type(V * sizeof(T) >= 4 ? V * sizeof(T) / 4 : 1), aligned(sizeof(T))));
  Vec<T, V> v;
#pragma unroll
  for (int e = 0; e < V; ++e) v.v[e] = from_f32<T>(o[e]);
  if constexpr (V > 1) {
    if (skip == 0) {
      __builtin_nontemporal_store(__builtin_bit_cast(Wide, v), (Wide*)p);
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (e >= skip) p[e] = v.v[e];
}

__device__ __forceinline__ float sigmoid(float u) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(u * -1.44269504f)); }

// The place of a thread: channels [c, c + V) of which the first `skip` are its neighbour's (the last access of a row ends
// with it), steps [t0, t1) of sequence b, of which `len` count.
struct Place {
  int b, tile, c, skip, t0, t1, len;
};
template <int V>
__device__ __forceinline__ bool place(const ConvArgs& A, Place& p) {
  const long id = (long)blockIdx.x * 256 + threadIdx.x, row = id / A.vecs;
  if (row >= (long)A.B * A.tiles) return false;
  p.b = (int)(row / A.tiles);
  p.tile = (int)(row - (long)p.b * A.tiles);
  const int c = (int)(id - row * A.vecs) * V;
  p.c = min(c, A.D - V);
  p.skip = c - p.c;
  p.t0 = p.tile * A.tile;
  p.t1 = min(p.t0 + A.tile, A.L);
  p.len = A.lengths ? (int)min(max(A.lengths[p.b], (int64_t)0), (int64_t)A.L) : A.L;
  return true;
}

// The inputs of kSteps steps from t >= 0 on; steps behind the last are the last one's (their results are not kept).
template <typename T, int V, int kSteps>
__device__ __forceinline__ void read(Vec<T, V> (&v)[kSteps], const T* p, long row, int t, int L) {
#pragma unroll
  for (int g = 0; g < kSteps; ++g) v[g] = load_vec<T, V>(p + min(t + g, L - 1) * row);
}

template <typename T, int W, int V>
__global__ __launch_bounds__(256) void k_conv_fwd(const ConvArgs A) {
  constexpr int G = 8;  // steps whose inputs are under way together
  Place p;
  if (!place<V>(A, p)) return;
  const T* x = (const T*)A.x + p.b * A.x_batch + p.c;
  T* y = (T*)A.y + ((long)p.b * A.L + p.t0) * A.D + p.c;
  T* state = A.state ? (T*)A.state + (long)p.b * (W - 1) * A.D + p.c : nullptr;
  Vec<T, V> next[G];
  read(next, x, A.x_row, p.t0, A.L);
  float w[W][V], bias[V] = {}, in[W - 1 + G][V];  // in: the W - 1 inputs before a group of steps, and theirs
#pragma unroll
  for (int e = 0; e < V; ++e)
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][e] = to_f32(((const T*)A.w)[(long)(p.c + e) * W + j]);
  if (A.bias) load(bias, (const T*)A.bias + p.c);
  auto input = [&](float (&o)[V], int t) {  // the input of step t >= -(W - 1)
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = 0.0f;
    if (t >= 0 && t < p.len) load(o, x + (long)t * A.x_row);
    else if (t < 0 && state) load(o, state + (long)(t + W - 1) * A.D);
  };
#pragma unroll
  for (int j = 0; j < W - 1; ++j) input(in[j], p.t0 - (W - 1) + j);
  // The new state: the last W - 1 inputs of the sequence.  The first tile writes it, which alone reads the old one; the
  // thread's own channels, so that no other reads what it has written.
  float last[W][V];
  if (state && p.tile == 0)
#pragma unroll
    for (int j = 0; j < W - 1; ++j) input(last[j], p.len - (W - 1) + j);
  for (int t = p.t0; t < p.t1; t += G) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int e = 0; e < V; ++e) in[W - 1 + g][e] = t + g < p.len ? to_f32(next[g].v[e]) : 0.0f;
    read(next, x, A.x_row, t + G, A.L);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float u = bias[e];
#pragma unroll
        for (int j = 0; j < W; ++j) u += w[j][e] * in[g + j][e];
        o[e] = t + g >= p.len ? 0.0f : A.silu ? u * sigmoid(u) : u;
      }
      if (t + g < p.t1) store(y, o, p.skip);
      y += A.D;
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) in[j][e] = in[G + j][e];
  }
  if (state && p.tile == 0)
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store(state + (long)j * A.D, last[j], p.skip);
}

template <typename T, int W, int V>
__global__ __launch_bounds__(256) void k_conv_bwd(const ConvArgs A) {
  constexpr int G = 4;
  Place p;
  if (!place<V>(A, p)) return;
  const T* x = (const T*)A.x + p.b * A.x_batch + p.c;
  const T* dy = (const T*)A.dy + (long)p.b * A.L * A.D + p.c;
  T* dx = A.dx ? (T*)A.dx + (long)p.b * A.L * A.D + p.c : nullptr;
  Vec<T, V> next_x[G], next_dy[G];
  read(next_x, x, A.x_row, p.t0, A.L);
  read(next_dy, dy, A.D, p.t0, A.L);
  // in, du: those of a group of steps behind those of the W - 1 steps before it
  float w[W][V], bias[V] = {}, in[W - 1 + G][V] = {}, du[W - 1 + G][V] = {}, dw[W][V] = {}, dbias[V] = {};
#pragma unroll
  for (int e = 0; e < V; ++e)
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][e] = to_f32(((const T*)A.w)[(long)(p.c + e) * W + j]);
  if (A.bias) load(bias, (const T*)A.bias + p.c);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    const int t = p.t0 - (W - 1) + j;
    if (t >= 0 && t < p.len) load(in[j], x + (long)t * A.x_row);
  }
  // dx[t] needs du up to t + W - 1: the walk goes W - 1 steps beyond the tile, whose du the next tile adds up
  for (int t = p.t0; t < p.t1 + W - 1; t += G) {
    float d[G][V];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        in[W - 1 + g][e] = t + g < p.len ? to_f32(next_x[g].v[e]) : 0.0f;
        d[g][e] = t + g < p.len ? to_f32(next_dy[g].v[e]) : 0.0f;
      }
    read(next_x, x, A.x_row, t + G, A.L);
    read(next_dy, dy, A.D, t + G, A.L);
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float u = bias[e], slope = 1.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) u += w[j][e] * in[g + j][e];
        if (A.silu) {
          const float s = sigmoid(u);
          slope = s * (1.0f + u * (1.0f - s));
        }
        du[W - 1 + g][e] = t + g < p.len ? d[g][e] * slope : 0.0f;
      }
      if (t + g < min(p.t1, p.len)) {  // (not by zeros: the next tile's inputs may be infinite)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float v = du[W - 1 + g][e];
          dbias[e] += v;
#pragma unroll
          for (int j = 0; j < W; ++j) dw[j][e] += v * in[g + j][e];
        }
      }
      const int to = t + g - (W - 1);  // du[g + j] is that of step to + j
      if (dx && to >= p.t0 && to < p.t1) {
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          o[e] = 0.0f;
#pragma unroll
          for (int j = 0; j < W; ++j) o[e] += w[W - 1 - j][e] * du[g + j][e];
          if (to >= p.len) o[e] = 0.0f;
        }
        store(dx + (long)to * A.D, o, p.skip);
      }
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        in[j][e] = in[G + j][e];
        du[j][e] = du[G + j][e];
      }
  }
  if (!A.part) return;
  float* part = A.part + ((long)p.b * A.tiles + p.tile) * (W + 1) * A.D + p.c;
#pragma unroll
  for (int j = 0; j < W; ++j) store(part + (long)j * A.D, dw[j], p.skip);
  store(part + (long)W * A.D, dbias, p.skip);
}

// Partial rows [rows][taps][D] to dw [D][W] and dbias [D], 64 channels a workgroup: 16 runs of rows, joined in order.
template <typename T>
__global__ __launch_bounds__(1024) void k_conv_reduce(const float* part, long rows, int D, int W, T* dw, T* dbias) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, run = threadIdx.x >> 6, c = blockIdx.x * 64 + lane, tap = blockIdx.y;
  float s = 0.0f;
  if (c < D)
#pragma unroll 8
    for (long r = run; r < rows; r += 16) s += part[(r * (W + 1) + tap) * D + c];
  lds[run][lane] = s;
  __syncthreads();
  if (run != 0 || c >= D) return;
#pragma unroll
  for (int r = 1; r < 16; ++r) s += lds[r][lane];
  if (tap < W) {
    if (dw) dw[(long)c * W + tap] = from_f32<T>(s);
  } else if (dbias) {
    dbias[c] = from_f32<T>(s);
  }
}

// ---- launches -----------------------------------------------------------------------------------------
struct ConvPlan {
  int tile, tiles, v, vecs;
  long threads;
};
constexpr int kTile = 64;
// v: channels of a thread.
ConvPlan plan_conv(int B, int L, int D) {
  ConvPlan p{};
  p.v = D < 4 ? 1 : 4;
  p.vecs = (D + p.v - 1) / p.v;
  p.tile = kTile;
  while (p.tile > 8 && (long)B * ((L + p.tile - 1) / p.tile) * p.vecs < 256L * 256) p.tile /= 2;
  p.tiles = (L + p.tile - 1) / p.tile;
  p.threads = (long)B * p.tiles * p.vecs;
  return p;
}

int check_conv(int dtype, int B, int L, int D, int W, long x_batch = 0, long x_row = 0) {
  if (dtype != DT_F32 && dtype != DT_F16 && dtype != DT_BF16) return kans_fail(KANS_ERR_ARG, "dtype %d", dtype);
  if (B < 0 || L < 0 || D <= 0) return kans_fail(KANS_ERR_ARG, "bad dims B=%d L=%d D=%d", B, L, D);
  if (x_batch < 0 || x_row < 0) return kans_fail(KANS_ERR_ARG, "negative strides");
  if (W < 1 || W > kMaxTaps) return kans_fail(KANS_ERR_UNSUPPORTED, "%d taps, 1 to %d", W, kMaxTaps);
  // (a grid holds fewer than 2^32 threads along x; the sums' has 1024 for 64 channels.  Tiles are shorter than kTile only where
  // there are few threads.  By division: the product may pass 64 bits.)
  const long rows = (long)B * ((L + (long)kTile - 1) / kTile), vecs = D < 4 ? D : (D + 3L) / 4;
  if (L > (1 << 30) || D > (1 << 27) || rows > ((1L << 31) - 1) / vecs)
    return kans_fail(KANS_ERR_UNSUPPORTED, "B=%d L=%d D=%d fit no grid", B, L, D);
  return 0;
}

template <typename F>
hipError_t by_conv(int dtype, int W, int v, F f) {
  hipError_t rc = hipErrorInvalidValue;
  auto taps = [&](auto t, auto vec) {
    auto go = [&](auto w) { rc = f(t, w, vec); };
    switch (W) {
      case 1: go(std::integral_constant<int, 1>{}); break;
      case 2: go(std::integral_constant<int, 2>{}); break;
      case 3: go(std::integral_constant<int, 3>{}); break;
      case 4: go(std::integral_constant<int, 4>{}); break;
      case 5: go(std::integral_constant<int, 5>{}); break;
      case 6: go(std::integral_constant<int, 6>{}); break;
      case 7: go(std::integral_constant<int, 7>{}); break;
      case 8: go(std::integral_constant<int, 8>{}); break;
    }
  };
  auto widths = [&](auto t) {
    if (v == 1) taps(t, std::integral_constant<int, 1>{});
    else taps(t, std::integral_constant<int, 4>{});
  };
  if (dtype == DT_F32) widths(0.0f);
  else if (dtype == DT_F16) widths((_Float16)0.0f);
  else widths((__bf16)0.0f);
  return rc;
}

}  // namespace
}  // namespace kans

using namespace kans;

extern "C" {

int kans_causal_conv_forward(int dtype, const void* x, long x_batch, long x_row, const void* w, const void* bias, void* state,
                             const int64_t* lengths, int silu, void* y, int B, int L, int D, int W, void* stream) {
  int rc = check_conv(dtype, B, L, D, W, x_batch, x_row);
  if (rc || B == 0 || L == 0) return rc;
  if (!x || !w || !y) return kans_fail(KANS_ERR_ARG, "null argument");
  std::lock_guard<std::mutex> lk(kans_mutex());
  if ((rc = kans_ensure_init())) return rc;
  const ConvPlan p = plan_conv(B, L, D);
  ConvArgs A{};
  A.x = x; A.w = w; A.bias = bias; A.y = y; A.state = W > 1 ? state : nullptr; A.lengths = lengths; A.silu = silu;
  A.x_batch = x_batch; A.x_row = x_row; A.B = B; A.L = L; A.D = D; A.tile = p.tile; A.tiles = p.tiles; A.vecs = p.vecs;
  HIP_TRY(by_conv(dtype, W, p.v, [&](auto t, auto taps, auto vec) {
    hipLaunchKernelGGL((k_conv_fwd<decltype(t), decltype(taps)::value, decltype(vec)::value>), dim3((unsigned)((p.threads + 255) / 256)),
                       dim3(256), 0, kans_caller_stream(stream), A);
    return hipGetLastError();
  }));
  return 0;
}

long kans_causal_conv_workspace(int dtype, int B, int L, int D, int W) {
  const int rc = check_conv(dtype, B, L, D, W);
  if (rc) return rc;
  const ConvPlan p = plan_conv(B, L, D);
  return (long)B * p.tiles * (W + 1) * D * (long)sizeof(float);
}

int kans_causal_conv_backward(int dtype, const void* x, long x_batch, long x_row, const void* w, const void* bias,
                              const int64_t* lengths, int silu, const void* dy, void* dx, void* dw, void* dbias, int B, int L, int D,
                              int W, void* workspace, long workspace_bytes, void* stream) {
  int rc = check_conv(dtype, B, L, D, W, x_batch, x_row);
  if (rc) return rc;
  const bool any = B > 0 && L > 0;
  if (any && (!x || !w || !dy)) return kans_fail(KANS_ERR_ARG, "null argument");
  if (dbias && !bias) return kans_fail(KANS_ERR_ARG, "gradient of an input that is not there");
  const ConvPlan p = plan_conv(B, L, D);
  const long rows = (long)B * p.tiles, need = rows * (W + 1) * D * (long)sizeof(float);
  const bool sums = dw || dbias;
  if (sums && need && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need))
    return kans_fail(KANS_ERR_ARG, "workspace of %ld bytes, %ld at a multiple of 16 needed", workspace ? workspace_bytes : 0, need);
  std::lock_guard<std::mutex> lk(kans_mutex());
  if ((rc = kans_ensure_init())) return rc;
  hipStream_t st = kans_caller_stream(stream);
  if (any) {
    ConvArgs A{};
    A.x = x; A.w = w; A.bias = bias; A.dy = dy; A.dx = dx; A.lengths = lengths; A.silu = silu;
    A.part = sums ? (float*)workspace : nullptr;
    A.x_batch = x_batch; A.x_row = x_row; A.B = B; A.L = L; A.D = D; A.tile = p.tile; A.tiles = p.tiles; A.vecs = p.vecs;
    HIP_TRY(by_conv(dtype, W, p.v, [&](auto t, auto taps, auto vec) {
      hipLaunchKernelGGL((k_conv_bwd<decltype(t), decltype(taps)::value, decltype(vec)::value>), dim3((unsigned)((p.threads + 255) / 256)),
                           dim3(256), 0, st, A);
      return hipGetLastError();
    }));
  }
  if (!sums) return 0;
  const dim3 grid((D + 63) / 64, W + 1);
  auto reduce = [&](auto t) {
    typedef decltype(t) T;
    hipLaunchKernelGGL(k_conv_reduce<T>, grid, dim3(1024), 0, st, (const float*)workspace, any ? rows : 0, D, W, (T*)dw, (T*)dbias);
  };
  if (dtype == DT_F32) reduce(0.0f);
  else if (dtype == DT_F16) reduce((_Float16)0.0f);
  else reduce((__bf16)0.0f);
  HIP_TRY(hipGetLastError());
  return 0;
}

}  // extern "C"
