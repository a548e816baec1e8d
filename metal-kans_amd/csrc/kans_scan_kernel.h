// Kernels of the selective scan (gfx950); the mathematics, the split and the measurements are in kans_scan.hip.
//
// Four lanes (a quad) hold a channel's states, kRegs each; a wave has 16 channels, a workgroup of four waves 64.  Lane q of
// a quad reads x, dt and z of the steps 4 m + q, so that what belongs to a step and channel is computed once; the step's
// turn takes it from its lane by a quad permute, which is part of the instruction that uses it.  B and C of a tile of
// steps lie in LDS in fp32, a lane reads its own states' there.  Sums over the states go through the quad, four steps at
// a time, so that lane q ends with the sum of step 4 m + q.
#pragma once
#include "kans_scan.h"
#include "kans_tile.h"

namespace kans {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// v of lane K of the quad
template <int K>
__device__ __forceinline__ float of_lane(float v) { return dpp<K * 0x55>(v); }

__device__ __forceinline__ float quad_sum(float v) {
  v += dpp<0xb1>(v);
  return v + dpp<0x4e>(v);
}
// Lane q of the quad gets the quad's sum of v[q].
__device__ __forceinline__ float quad_sums(const float (&v)[4]) {
  const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
  const float v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3];
  const float a = (odd ? v1 : v0) + dpp<0xb1>(odd ? v0 : v1);
  const float b = (odd ? v3 : v2) + dpp<0xb1>(odd ? v2 : v3);
  return (high ? b : a) + dpp<0x4e>(high ? a : b);
}
// Lane l gets the sum of v[l / 4] over the 16 lanes with its place in the quad.
typedef unsigned Pair __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float sum_of(Pair v) {
  const unsigned a = v.x, b = v.y;  // (a bit cast of v.y itself takes v.x)
  return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float wave_sums(float (&v)[16]) {
  auto bits = [](float f) { return __builtin_bit_cast(unsigned, f); };
#pragma unroll
  for (int i = 0; i < 8; ++i)
    v[i] = sum_of(__builtin_bit_cast(Pair, __builtin_amdgcn_permlane32_swap(bits(v[i]), bits(v[i + 8]), false, false)));
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = sum_of(__builtin_bit_cast(Pair, __builtin_amdgcn_permlane16_swap(bits(v[i]), bits(v[i + 4]), false, false)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] += dpp<0x128>(v[i]);  // 8 lanes on in the row
    v[i] += dpp<0x124>(v[i]);  // 4 lanes on
  }
  const bool b2 = threadIdx.x & 4, b3 = threadIdx.x & 8;
  const float v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3], low = b2 ? v1 : v0, high = b2 ? v3 : v2;
  return b3 ? high : low;
}

__device__ __forceinline__ float exp_neg(float v) { return __builtin_amdgcn_exp2f(v * -kLog2e); }
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.0f + exp_neg(v)); }

// log(1 + exp(v)) = max(v, 0) + log(1 + e), e = exp(-|v|) in [0, 1].  log(1 + e) / e by a polynomial of degree 9 (least largest
// relative error, 5e-9 before its coefficients are rounded): the usual small step sizes keep all their digits, which a
// logarithm of the rounded 1 + e would not.
__device__ __forceinline__ float softplus(float v) {
  const float e = exp_neg(fabsf(v));
  float p = -0.0032440251670777798f;
  p = p * e + 0.01985146477818489f;
  p = p * e - 0.056959547102451324f;
  p = p * e + 0.10603656619787216f;
  p = p * e - 0.15305593609809875f;
  p = p * e + 0.1967594027519226f;
  p = p * e - 0.24954134225845337f;
  p = p * e + 0.3332996368408203f;
  p = p * e - 0.4999990165233612f;
  p = p * e + 1.0f;
  return (v < 0.0f ? 0.0f : v) + p * e;  // (NaN stays NaN)
}

template <int kRegs> struct Shape {
  static constexpr int kPad = 4 * kRegs;                 // states, rounded up
  static constexpr int kTile = 16;                       // steps of a forward tile
  static constexpr int kInterval = scan_interval(kRegs); // steps of a backward tile
};

// Where a lane stands.
struct Lane {
  int b, chunk, c, q, len, t0, t1;  // c: its channel (maybe behind the last), steps [t0, t1) of the chunk, len of the sequence
  bool on;                          // the channel exists
  long row;                         // the channel, or the last one
};
__device__ __forceinline__ Lane lane_of(const ScanArgs& A) {
  Lane l;
  const int blocks = (A.D + kScanChannels - 1) / kScanChannels;
  const int id = blockIdx.x / blocks, block = blockIdx.x - id * blocks;
  l.b = id / A.chunks;
  l.chunk = id - l.b * A.chunks;
  l.c = block * kScanChannels + (int)threadIdx.x / 4;
  l.q = threadIdx.x & 3;
  l.on = l.c < A.D;
  l.row = min(l.c, A.D - 1);
  l.len = A.lengths ? (int)min(max(A.lengths[l.b], (int64_t)0), (int64_t)A.L) : A.L;
  l.t0 = l.chunk * A.chunk;
  l.t1 = min(l.t0 + A.chunk, A.L);
  return l;
}

// B and C of kSteps steps, on their way from memory to LDS.  Steps and states that are not there are zeros.
template <typename T, int kRegs, int kSteps>
struct Rows {
  static constexpr int kPad = 4 * kRegs, kEach = kSteps * 2 * kPad, kPer = (kEach + kThreads - 1) / kThreads;
  T v[kPer];
  __device__ __forceinline__ void read(const ScanArgs& A, int b, int first, int len) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int at = i * kThreads + threadIdx.x, step = at / (2 * kPad), n = at % kPad, t = first + step;
      const bool is_c = at / kPad & 1, there = at < kEach && t < len && n < A.N;
      const T* from = is_c ? (const T*)A.Cm + b * A.c_batch + (long)t * A.c_row : (const T*)A.Bm + b * A.b_batch + (long)t * A.b_row;
      v[i] = there ? from[n] : from_f32<T>(0.0f);
    }
  }
  __device__ __forceinline__ void write(float* lds) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int at = i * kThreads + threadIdx.x;
      if (kEach % kThreads == 0 || at < kEach) lds[at] = to_f32(v[i]);
    }
  }
};

template <int kRegs>
__device__ __forceinline__ void read_states(float (&o)[kRegs], const float* lds) {
#pragma unroll
  for (int i = 0; i < kRegs; ++i) o[i] = lds[i];
}

// A lane's states in memory (those from N on are not there).
template <int kRegs>
__device__ __forceinline__ void load_states(float (&h)[kRegs], const float* p, int q, int N, bool on) {
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const int n = q * kRegs + i;
    h[i] = on && n < N ? p[n] : 0.0f;
  }
}
template <int kRegs>
__device__ __forceinline__ void store_states(const float (&h)[kRegs], float* p, int q, int N, bool on) {
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const int n = q * kRegs + i;
    if (on && n < N) p[n] = h[i];
  }
}

// A lane's values of an input at the steps first + 4 m + q.
template <typename T, int kCount>
__device__ __forceinline__ void read_steps(T (&v)[kCount], const T* p, long row, int first, int q, int L) {
#pragma unroll
  for (int m = 0; m < kCount; ++m) v[m] = p[(long)min(first + 4 * m + q, L - 1) * row];
}

// ---- forward ------------------------------------------------------------------------------------------
// kEdges: of each chunk alone, from a state of zeros, its last state and the sum of its step sizes.
template <typename T, int kRegs, bool kEdges>
__global__ __launch_bounds__(kThreads) void k_scan_fwd(const ScanArgs A) {
  constexpr int kPad = Shape<kRegs>::kPad, kTile = Shape<kRegs>::kTile, kInterval = Shape<kRegs>::kInterval, kM = kTile / 4;
  __shared__ float bc[2][kTile * 2 * kPad];
  const Lane l = lane_of(A);
  const T* x = (const T*)A.x + l.b * A.x_batch + l.row;
  const T* dt = (const T*)A.dt + l.b * A.dt_batch + l.row;
  const T* z = A.z ? (const T*)A.z + l.b * A.z_batch + l.row : nullptr;
  const float bias = A.bias ? A.bias[l.row] : 0.0f, skip = A.skip ? A.skip[l.row] : 0.0f;
  float a2[kRegs], h[kRegs];
  load_states<kRegs>(a2, A.A + l.row * A.N, l.q, A.N, true);
#pragma unroll
  for (int i = 0; i < kRegs; ++i) a2[i] *= kLog2e;
  const long place = (long)l.b * A.chunks + l.chunk;
  if (kEdges) {
#pragma unroll
    for (int i = 0; i < kRegs; ++i) h[i] = 0.0f;
  } else if (A.chunks > 1) {
    load_states<kRegs>(h, A.edge + (place * A.D + l.row) * A.N, l.q, A.N, true);
  } else {
    load_states<kRegs>(h, A.state + ((long)l.b * A.D + l.row) * A.N, l.q, A.N, A.state != nullptr);
  }
  float total = 0.0f;
  const int intervals = (A.L + kInterval - 1) / kInterval;

  T xv[kM], dv[kM], zv[kM];
  Rows<T, kRegs, kTile> rows;
  read_steps(xv, x, A.x_row, l.t0, l.q, A.L);
  read_steps(dv, dt, A.dt_row, l.t0, l.q, A.L);
  if (!kEdges && z) read_steps(zv, z, A.z_row, l.t0, l.q, A.L);
  rows.read(A, l.b, l.t0, l.len);
  rows.write(bc[0]);
  __syncthreads();
  for (int t = l.t0, turn = 0; t < l.t1; t += kTile, turn ^= 1) {
    float s[kM], u[kM], xs[kM], zs[kM];
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      const bool counts = t + 4 * m + l.q < l.len;
      const float v = to_f32(dv[m]) + bias;
      s[m] = counts ? (A.softplus ? softplus(v) : v) : 0.0f;
      xs[m] = counts ? to_f32(xv[m]) : 0.0f;
      u[m] = s[m] * xs[m];
      if (kEdges) total += s[m];
      else if (z) zs[m] = to_f32(zv[m]);
    }
    const bool more = t + kTile < l.t1;
    if (more) {
      read_steps(xv, x, A.x_row, t + kTile, l.q, A.L);
      read_steps(dv, dt, A.dt_row, t + kTile, l.q, A.L);
      if (!kEdges && z) read_steps(zv, z, A.z_row, t + kTile, l.q, A.L);
      rows.read(A, l.b, t + kTile, l.len);
    }
    const float* mine = bc[turn] + l.q * kRegs;
    static_for<0, kM>([&](auto m_) {
      constexpr int m = decltype(m_)::value;
      float y[4];
      static_for<0, 4>([&](auto k_) {
        constexpr int k = decltype(k_)::value, j = 4 * m + k;
        if (!kEdges && j % kInterval == 0 && A.saved && t + j < A.L)
          store_states<kRegs>(h, A.saved + (((long)l.b * intervals + (t + j) / kInterval) * A.D + l.row) * A.N, l.q, A.N, l.on);
        float Bv[kRegs], Cv[kRegs];
        read_states<kRegs>(Bv, mine + j * 2 * kPad);
        if (!kEdges) read_states<kRegs>(Cv, mine + j * 2 * kPad + kPad);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kRegs; ++i) {
          h[i] = __builtin_amdgcn_exp2f(of_lane<k>(s[m]) * a2[i]) * h[i] + of_lane<k>(u[m]) * Bv[i];
          if (!kEdges) sum += h[i] * Cv[i];
        }
        y[k] = sum;
      });
      if (!kEdges) {
        const int at = t + 4 * m + l.q;
        float o = quad_sums(y) + skip * xs[m];
        if (z) o *= zs[m] * sigmoid(zs[m]);
        if (l.on && at < A.L) ((T*)A.out)[((long)l.b * A.L + at) * A.D + l.c] = from_f32<T>(at < l.len ? o : 0.0f);
      }
    });
    if (more) rows.write(bc[turn ^ 1]);
    __syncthreads();
  }
  if (kEdges) {
    store_states<kRegs>(h, A.edge + (place * A.D + l.row) * A.N, l.q, A.N, l.on);
    total = quad_sum(total);
    if (l.on && l.q == 0) A.sums[place * A.D + l.c] = total;
  } else if (A.state && l.chunk == A.chunks - 1) {
    store_states<kRegs>(h, A.state + ((long)l.b * A.D + l.row) * A.N, l.q, A.N, l.on);
  }
}

// ---- backward -----------------------------------------------------------------------------------------
// kEdges: of each chunk alone, without a gradient from behind it, the gradient of its first state, and the sum of its step sizes.
template <typename T, int kRegs, bool kEdges>
__global__ __launch_bounds__(kThreads) void k_scan_bwd(const ScanArgs A) {
  constexpr int kPad = Shape<kRegs>::kPad, kTile = Shape<kRegs>::kInterval, kM = kTile / 4, kGroups = kTile * 2 * kRegs / 16;
  __shared__ float bc[2][kTile * 2 * kPad];
  __shared__ float red[kEdges ? 1 : 2][4][kEdges ? 1 : kGroups * 64];
  const Lane l = lane_of(A);
  const T* x = (const T*)A.x + l.b * A.x_batch + l.row;
  const T* dt = (const T*)A.dt + l.b * A.dt_batch + l.row;
  const T* z = A.z ? (const T*)A.z + l.b * A.z_batch + l.row : nullptr;
  const T* dout = (const T*)A.dout + (long)l.b * A.L * A.D + l.row;
  const float bias = A.bias ? A.bias[l.row] : 0.0f, skip = A.skip ? A.skip[l.row] : 0.0f;
  float a2[kRegs], carry[kRegs], dA[kRegs] = {}, dskip = 0.0f, dbias = 0.0f, total = 0.0f;
  load_states<kRegs>(a2, A.A + l.row * A.N, l.q, A.N, true);
#pragma unroll
  for (int i = 0; i < kRegs; ++i) a2[i] *= kLog2e;
  const long place = (long)l.b * A.chunks + l.chunk;
  load_states<kRegs>(carry, A.edge + (place * A.D + l.row) * A.N, l.q, A.N, !kEdges && A.chunks > 1 && l.on);
  const int intervals = (A.L + kTile - 1) / kTile;
  const float* saved = A.saved + ((long)l.b * intervals * A.D + l.row) * A.N;

  const int tiles = (l.t1 - l.t0 + kTile - 1) / kTile;
  T xv[kM], dv[kM], zv[kM], gv[kM];
  float first[kRegs];
  Rows<T, kRegs, kTile> rows;
  auto read = [&](int t) {
    read_steps(xv, x, A.x_row, t, l.q, A.L);
    read_steps(dv, dt, A.dt_row, t, l.q, A.L);
    read_steps(gv, dout, A.D, t, l.q, A.L);
    if (z) read_steps(zv, z, A.z_row, t, l.q, A.L);
    rows.read(A, l.b, t, l.len);
    if (!kEdges) load_states<kRegs>(first, saved + (long)(t / kTile) * A.D * A.N, l.q, A.N, true);
  };
  read(l.t0 + (tiles - 1) * kTile);
  rows.write(bc[0]);
  __syncthreads();
  for (int tile = tiles - 1, turn = 0; tile >= 0; --tile, turn ^= 1) {
    const int t = l.t0 + tile * kTile;
    float s[kM], u[kM], xs[kM], dy[kM], vs[kM], zs[kM], ds[kM], h[kRegs];
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      const bool counts = l.on && t + 4 * m + l.q < l.len;
      vs[m] = to_f32(dv[m]) + bias;
      s[m] = counts ? (A.softplus ? softplus(vs[m]) : vs[m]) : 0.0f;
      xs[m] = counts ? to_f32(xv[m]) : 0.0f;
      u[m] = s[m] * xs[m];
      ds[m] = counts ? to_f32(gv[m]) : 0.0f;  // (dout)
      zs[m] = z && counts ? to_f32(zv[m]) : 0.0f;
      dy[m] = z ? ds[m] * (zs[m] * sigmoid(zs[m])) : ds[m];
      if (kEdges) total += s[m];
    }
#pragma unroll
    for (int i = 0; i < kRegs; ++i) h[i] = first[i];
    if (tile > 0) read(t - kTile);
    const float* mine = bc[turn] + l.q * kRegs;
    // the states of the tile again: before each step, and what the step leaves of them
    float before[kEdges ? 1 : kTile][kRegs], left[kTile][kRegs], ys[kM];
    static_for<0, kM>([&](auto m_) {
      constexpr int m = decltype(m_)::value;
      float y[4];
      static_for<0, 4>([&](auto k_) {
        constexpr int k = decltype(k_)::value, j = 4 * m + k;
        float Bv[kRegs], Cv[kRegs], sum = 0.0f;
        if (!kEdges) read_states<kRegs>(Bv, mine + j * 2 * kPad);
        if (!kEdges && z) read_states<kRegs>(Cv, mine + j * 2 * kPad + kPad);
#pragma unroll
        for (int i = 0; i < kRegs; ++i) {
          left[j][i] = __builtin_amdgcn_exp2f(of_lane<k>(s[m]) * a2[i]);
          if (kEdges) continue;
          before[kEdges ? 0 : j][i] = h[i];
          h[i] = left[j][i] * h[i] + of_lane<k>(u[m]) * Bv[i];
          if (z) sum += h[i] * Cv[i];
        }
        y[k] = sum;
      });
      ys[m] = !kEdges && z ? quad_sums(y) + skip * xs[m] : 0.0f;
    });
    float vals[16], dA_tile[kRegs] = {};
    static_for<0, kM>([&](auto m_) {
      constexpr int m = kM - 1 - decltype(m_)::value;
      float yB[4], yA[4];
      static_for<0, 4>([&](auto k_) {
        constexpr int k = 3 - decltype(k_)::value, j = 4 * m + k;
        float Bv[kRegs], Cv[kRegs], g[kRegs], sB = 0.0f, sA = 0.0f;
        if (!kEdges) read_states<kRegs>(Bv, mine + j * 2 * kPad);
        read_states<kRegs>(Cv, mine + j * 2 * kPad + kPad);
#pragma unroll
        for (int i = 0; i < kRegs; ++i) {
          g[i] = Cv[i] * of_lane<k>(dy[m]) + carry[i];
          carry[i] = g[i] * left[j][i];
          if (kEdges) continue;
          sB += g[i] * Bv[i];
          const float w = carry[i] * before[kEdges ? 0 : j][i];
          sA += w * a2[i];
          dA_tile[i] += w * of_lane<k>(s[m]);
        }
        if (kEdges) return;
        yB[k] = sB;
        yA[k] = sA;
        static_for<0, 2 * kRegs>([&](auto i_) {
          constexpr int i = decltype(i_)::value, value = (kTile - 1 - j) * 2 * kRegs + i;
          vals[value % 16] = i < kRegs ? g[i % kRegs] * of_lane<k>(u[m]) : h[i % kRegs] * of_lane<k>(dy[m]);
          if (value % 16 == 15) red[turn][threadIdx.x >> 6][value / 16 * 64 + (threadIdx.x & 63)] = wave_sums(vals);
        });
#pragma unroll
        for (int i = 0; i < kRegs; ++i) h[i] = before[kEdges ? 0 : j][i];
      });
      if (!kEdges) {
        const float gB = quad_sums(yB), gA = quad_sums(yA) * kLn2;
        const int at = t + 4 * m + l.q;
        const bool counts = l.on && at < l.len;
        const float dstep = xs[m] * gB + gA;
        const float ddt = counts ? (A.softplus ? dstep * sigmoid(vs[m]) : dstep) : 0.0f;
        const float dxv = counts ? s[m] * gB + skip * dy[m] : 0.0f;
        dskip += dy[m] * xs[m];
        dbias += ddt;
        if (l.on && at < A.L) {
          const long to = ((long)l.b * A.L + at) * A.D + l.c;
          ((T*)A.dx)[to] = from_f32<T>(dxv);
          ((T*)A.ddt)[to] = from_f32<T>(ddt);
          if (z) {
            const float sg = sigmoid(zs[m]);
            ((T*)A.dz)[to] = from_f32<T>(counts ? ds[m] * ys[m] * (sg * (1.0f + zs[m] * (1.0f - sg))) : 0.0f);
          }
        }
      }
    });
#pragma unroll
    for (int i = 0; i < kRegs; ++i) dA[i] += dA_tile[i];
    if (tile > 0) rows.write(bc[turn ^ 1]);
    __syncthreads();
    if (!kEdges) {
      // the sums over this workgroup's channels: [step][B or C][state]
      const int block = (int)(blockIdx.x % ((A.D + kScanChannels - 1) / kScanChannels));
      float* part = A.part_bc + (((long)block * A.B + l.b) * A.L + t) * 2 * kPad;
      const int there = min(kTile, A.L - t) * 2 * kPad;
#pragma unroll
      for (int i = 0; i < (kTile * 2 * kPad + kThreads - 1) / kThreads; ++i) {
        const int at = i * kThreads + (int)threadIdx.x;
        if (at >= there) break;
        const int j = at / (2 * kPad), which = at / kPad & 1, n = at % kPad;
        const int value = (kTile - 1 - j) * 2 * kRegs + which * kRegs + n % kRegs, from = value / 16 * 64 + value % 16 * 4 + n / kRegs;
        part[at] = (red[turn][0][from] + red[turn][1][from]) + (red[turn][2][from] + red[turn][3][from]);
      }
    }
  }
  if (kEdges) {
    store_states<kRegs>(carry, A.edge + (place * A.D + l.row) * A.N, l.q, A.N, l.on);
    total = quad_sum(total);
    if (l.on && l.q == 0) A.sums[place * A.D + l.c] = total;
    return;
  }
  float* par = A.part_par + (place * A.D + l.row) * (A.N + 2);
  store_states<kRegs>(dA, par, l.q, A.N, l.on);
  dskip = quad_sum(dskip);
  dbias = quad_sum(dbias);
  if (l.on && l.q == 0) {
    par[A.N] = dskip;
    par[A.N + 1] = dbias;
  }
}

// ---- one step -----------------------------------------------------------------------------------------
// A single token: the state read and written once.  A quad goes through a channel's states, 4 x 4 at a time.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_scan_step(const ScanArgs A) {
  const long at = ((long)blockIdx.x * kThreads + threadIdx.x) / 4, all = (long)A.B * A.D;
  const long row = min(at, all - 1);
  const int b = (int)(row / A.D), c = (int)(row - (long)b * A.D), q = threadIdx.x & 3;
  const bool counts = !A.lengths || A.lengths[b] > 0;
  const float x = to_f32(((const T*)A.x)[b * A.x_batch + c]);
  float s = to_f32(((const T*)A.dt)[b * A.dt_batch + c]) + (A.bias ? A.bias[c] : 0.0f);
  if (A.softplus) s = softplus(s);
  const float u = s * x;
  const T *Bm = (const T*)A.Bm + b * A.b_batch, *Cm = (const T*)A.Cm + b * A.c_batch;
  float* h = A.state + row * A.N;
  const float* a = A.A + (long)c * A.N;
  float y = 0.0f;
  if (A.N % 4 == 0) {  // (the state and A start at multiples of 16 bytes)
    for (int n = 4 * q; n < A.N; n += 16) {
      float4 hv = *(const float4*)(h + n);
      const float4 av = *(const float4*)(a + n);
      float hs[4] = {hv.x, hv.y, hv.z, hv.w}, as[4] = {av.x, av.y, av.z, av.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        hs[i] = __builtin_amdgcn_exp2f(s * (as[i] * kLog2e)) * hs[i] + u * to_f32(Bm[n + i]);
        y += hs[i] * to_f32(Cm[n + i]);
      }
      if (counts && at < all) *(float4*)(h + n) = make_float4(hs[0], hs[1], hs[2], hs[3]);
    }
  } else {
    for (int n = q; n < A.N; n += 4) {
      const float v = __builtin_amdgcn_exp2f(s * (a[n] * kLog2e)) * h[n] + u * to_f32(Bm[n]);
      y += v * to_f32(Cm[n]);
      if (counts && at < all) h[n] = v;
    }
  }
  y = quad_sum(y);
  if (q != 0 || at >= all) return;
  y += (A.skip ? A.skip[c] : 0.0f) * x;
  if (A.z) {
    const float z = to_f32(((const T*)A.z)[b * A.z_batch + c]);
    y *= z * sigmoid(z);
  }
  ((T*)A.out)[row] = from_f32<T>(counts ? y : 0.0f);
}

// ---- sums of the partial rows --------------------------------------------------------------------------
// dB and dC: [blocks][rows][2][padded] to [rows][N] twice.
template <typename T>
__global__ __launch_bounds__(256) void k_scan_reduce(const float* part, int blocks, long rows, int padded, int N, T* dB, T* dC) {
  const long at = (long)blockIdx.x * 256 + threadIdx.x, all = rows * 2 * padded;
  if (at >= all) return;
  float s = 0.0f;
#pragma unroll 8
  for (int k = 0; k < blocks; ++k) s += part[k * all + at];
  const int n = (int)(at % padded);
  if (n >= N) return;
  T* to = at / padded & 1 ? dC : dB;
  if (to) to[at / (2 * padded) * N + n] = from_f32<T>(s);
}

template <typename T, int kRegs>
hipError_t launch(ScanPass pass, const ScanArgs& A, hipStream_t st) {
  const dim3 grid((unsigned)((long)A.B * A.chunks * ((A.D + kScanChannels - 1) / kScanChannels)));
  switch (pass) {
    case ScanPass::kForward: hipLaunchKernelGGL((k_scan_fwd<T, kRegs, false>), grid, dim3(kThreads), 0, st, A); break;
    case ScanPass::kEdges: hipLaunchKernelGGL((k_scan_fwd<T, kRegs, true>), grid, dim3(kThreads), 0, st, A); break;
    case ScanPass::kBackward: hipLaunchKernelGGL((k_scan_bwd<T, kRegs, false>), grid, dim3(kThreads), 0, st, A); break;
    case ScanPass::kBackwardEdges: hipLaunchKernelGGL((k_scan_bwd<T, kRegs, true>), grid, dim3(kThreads), 0, st, A); break;
    case ScanPass::kStep: break;
  }
  return hipGetLastError();
}

template <typename T>
hipError_t launch_scan(ScanPass pass, const ScanArgs& A, hipStream_t st) {
  if (pass == ScanPass::kStep) {
    hipLaunchKernelGGL(k_scan_step<T>, dim3((unsigned)(((long)A.B * A.D * 4 + kThreads - 1) / kThreads)), dim3(kThreads), 0, st, A);
    return hipGetLastError();
  }
  switch (scan_regs(A.N)) {
    case 1: return launch<T, 1>(pass, A, st);
    case 2: return launch<T, 2>(pass, A, st);
    case 4: return launch<T, 4>(pass, A, st);
    case 6: return launch<T, 6>(pass, A, st);
    case 8: return launch<T, 8>(pass, A, st);
    case 16: return launch<T, 16>(pass, A, st);
  }
  return hipErrorInvalidValue;
}

template <typename T>
hipError_t reduce_scan(const ScanArgs& A, int padded, void* dB, void* dC, hipStream_t st) {
  const long rows = (long)A.B * A.L;
  hipLaunchKernelGGL(k_scan_reduce<T>, dim3((unsigned)((rows * 2 * padded + 255) / 256)), dim3(256), 0, st, A.part_bc,
                     (A.D + kScanChannels - 1) / kScanChannels, rows, padded, A.N, (T*)dB, (T*)dC);
  return hipGetLastError();
}

}  // namespace
}  // namespace kans
