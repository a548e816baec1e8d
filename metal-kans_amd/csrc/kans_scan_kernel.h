// Kernels of the selective scan (gfx950); the mathematics, the split and the measurements are in kans_scan.hip.
//
// Four lanes (a quad) hold a channel's states, kRegs each; a wave has 16 channels, a workgroup of four waves 64.  Lane q of
// a quad reads x, dt and z of the steps 4 m + q, so that what belongs to a step and channel is computed once; the step's
// turn takes it from its lane by a quad permute, which is part of the instruction that uses it.  B and C of a tile of
// steps lie in LDS in fp32, a lane reads its own states' there.  Sums over the states go through the quad, four steps at
// a time, so that lane q ends with the sum of step 4 m + q.
#pragma once
#include <algorithm>

#include "kans_scan.h"
#include "kans_tile.h"

namespace kans {
namespace {

constexpr int kThreads = 256;

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
// Lane q of the quad gets the quad's sum of v[q].  (By selections: 4 x 4 x 1 products with unit columns on the matrix pipe take 3 vector
// instructions instead of 9, but their waits made the kernels 5 - 7 % slower, and 0 times infinity would carry one step's
// infinity to the three beside it.)
__device__ __forceinline__ float quad_sums(const float (&v)[4]) {
  const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
  const float v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3];
  const float a = (odd ? v1 : v0) + dpp<0xb1>(odd ? v0 : v1);
  const float b = (odd ? v3 : v2) + dpp<0xb1>(odd ? v2 : v3);
  return (high ? b : a) + dpp<0x4e>(high ? a : b);
}

// The backward's lanes hold their states in mirrored order in every other quad: lane q of an odd one those of 3 - q, so that a lane's
// partner in a mirrored row, or half of a row, holds the same states.
__device__ __forceinline__ int states_of(int lane) { return lane & 4 ? 3 - (lane & 3) : lane & 3; }

// The sums of 16 values over the 16 lanes with the same states: lane l gets that of value 8 b3 + 4 b2 + 2 b4 + b5, b its bits.
// Half of the lanes that are added take one value of a pair, half the other: sums with the mirrored row (and half row) are
// written to some banks of four lanes only, two instructions a pair; the rows meet by swaps.  33 issue slots for 16 values, 47
// by swaps and selections alone (a swap takes two).  On the matrix pipe, 16 products of 16 x 16 x 4 in a chain, the
// backward took twice as long.
typedef unsigned Pair __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float sum_of(Pair v) {
  const unsigned a = v.x, b = v.y;  // (a bit cast of v.y itself takes v.x)
  return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float wave_sums(float (&v)[16]) {
  // (A lane permute reads what is at least two instructions old, and five behind a change of the lanes that are on.  Results are
  // written while others are still to be read.)
  asm("s_nop 4\n"
      "v_add_f32_dpp %0, %0, %0 row_mirror row_mask:0xf bank_mask:0xf\n"
      "v_add_f32_dpp %1, %1, %1 row_mirror row_mask:0xf bank_mask:0xf\n"
      "v_add_f32_dpp %2, %2, %2 row_mirror row_mask:0xf bank_mask:0xf\n"
      "v_add_f32_dpp %3, %3, %3 row_mirror row_mask:0xf bank_mask:0xf\n"
      "v_add_f32_dpp %4, %4, %4 row_mirror row_mask:0xf bank_mask:0xf\n"
      "v_add_f32_dpp %5, %5, %5 row_mirror row_mask:0xf bank_mask:0xf\n"
      "v_add_f32_dpp %6, %6, %6 row_mirror row_mask:0xf bank_mask:0xf\n"
      "v_add_f32_dpp %7, %7, %7 row_mirror row_mask:0xf bank_mask:0xf\n"
      "v_add_f32_dpp %0, %8, %8 row_mirror row_mask:0xf bank_mask:0xc\n"
      "v_add_f32_dpp %1, %9, %9 row_mirror row_mask:0xf bank_mask:0xc\n"
      "v_add_f32_dpp %2, %10, %10 row_mirror row_mask:0xf bank_mask:0xc\n"
      "v_add_f32_dpp %3, %11, %11 row_mirror row_mask:0xf bank_mask:0xc\n"
      "v_add_f32_dpp %4, %12, %12 row_mirror row_mask:0xf bank_mask:0xc\n"
      "v_add_f32_dpp %5, %13, %13 row_mirror row_mask:0xf bank_mask:0xc\n"
      "v_add_f32_dpp %6, %14, %14 row_mirror row_mask:0xf bank_mask:0xc\n"
      "v_add_f32_dpp %7, %15, %15 row_mirror row_mask:0xf bank_mask:0xc\n"
      "v_add_f32_dpp %0, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n"
      "v_add_f32_dpp %1, %1, %1 row_half_mirror row_mask:0xf bank_mask:0xf\n"
      "v_add_f32_dpp %2, %2, %2 row_half_mirror row_mask:0xf bank_mask:0xf\n"
      "v_add_f32_dpp %3, %3, %3 row_half_mirror row_mask:0xf bank_mask:0xf\n"
      "v_add_f32_dpp %0, %4, %4 row_half_mirror row_mask:0xf bank_mask:0xa\n"
      "v_add_f32_dpp %1, %5, %5 row_half_mirror row_mask:0xf bank_mask:0xa\n"
      "v_add_f32_dpp %2, %6, %6 row_half_mirror row_mask:0xf bank_mask:0xa\n"
      "v_add_f32_dpp %3, %7, %7 row_half_mirror row_mask:0xf bank_mask:0xa\n"
      "s_nop 1"
      : "+&v"(v[0]), "+&v"(v[1]), "+&v"(v[2]), "+&v"(v[3]), "+&v"(v[4]), "+&v"(v[5]), "+&v"(v[6]), "+&v"(v[7])
      : "v"(v[8]), "v"(v[9]), "v"(v[10]), "v"(v[11]), "v"(v[12]), "v"(v[13]), "v"(v[14]), "v"(v[15]));
  auto bits = [](float f) { return __builtin_bit_cast(unsigned, f); };
#pragma unroll
  for (int i = 0; i < 2; ++i)
    v[i] = sum_of(__builtin_bit_cast(Pair, __builtin_amdgcn_permlane16_swap(bits(v[i]), bits(v[i + 2]), false, false)));
  return sum_of(__builtin_bit_cast(Pair, __builtin_amdgcn_permlane32_swap(bits(v[0]), bits(v[1]), false, false)));
}

__device__ __forceinline__ float exp_neg(float v) { return __builtin_amdgcn_exp2f(v * -kLog2e); }
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.0f + exp_neg(v)); }

// log(1 + exp(v)) = max(v, 0) + log(1 + e), e = exp(-|v|) in [0, 1].  log(1 + e) / e by a polynomial of degree 9 (least largest
// relative error, 5e-9 before its coefficients are rounded): the usual small step sizes keep all their digits, which a
// logarithm of the rounded 1 + e would not.
// slope: sigmoid(v), from the same exponential.
__device__ __forceinline__ float softplus(float v, float& slope) {
  const float e = exp_neg(fabsf(v)), r = __builtin_amdgcn_rcpf(1.0f + e);
  slope = v < 0.0f ? e * r : r;
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
__device__ __forceinline__ float softplus(float v) {
  float slope;
  return softplus(v, slope);
}

template <int kRegs> struct Shape {
  static constexpr int kPad = 4 * kRegs;                 // states, rounded up
  static constexpr int kTile = 16;                       // steps of a forward tile
  static constexpr int kInterval = scan_interval(kRegs); // steps of a backward tile
  // steps whose B and C are read from LDS together, forward and (with fewer registers to spare) backward
  static constexpr int kAhead = kRegs <= 4 ? 4 : kRegs <= 8 ? 2 : 1, kAheadBack = kRegs <= 2 ? 4 : 1;
};

// ---- memory -------------------------------------------------------------------------------------------
// Buffers with an end: what lies behind it reads as zero and is not written, so that the last steps, the last channels and
// absent tensors need no branch (a branch ends what the compiler can move: the loads of the next steps).
typedef __amdgpu_buffer_rsrc_t Buffer;
constexpr unsigned kNowhere = 0x80000000u;  // an offset behind every end (none reaches 2^30), also with 16 steps added
__device__ __forceinline__ Buffer buffer(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00027000);
}
template <typename T>
__device__ __forceinline__ T fetch(Buffer b, unsigned offset) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(b, (int)offset, 0, 0));
  else return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(b, (int)offset, 0, 0));
}
template <typename T>
__device__ __forceinline__ void put(Buffer b, unsigned offset, T v) {
  if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), b, (int)offset, 0, 0);
  else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, v), b, (int)offset, 0, 0);
}
// A lane's states in the padded layouts of saved and edge.
template <int kRegs>
__device__ __forceinline__ void fetch_states(float (&h)[kRegs], Buffer b, unsigned offset) {
  typedef unsigned Two __attribute__((ext_vector_type(2)));
  typedef unsigned Four __attribute__((ext_vector_type(4)));
  if constexpr (kRegs == 1) {
    h[0] = fetch<float>(b, offset);
  } else if constexpr (kRegs % 4 == 0) {
#pragma unroll
    for (int i = 0; i < kRegs; i += 4) {
      const Four v = __builtin_amdgcn_raw_buffer_load_b128(b, (int)(offset + 4 * i), 0, 0);
      __builtin_memcpy(h + i, &v, 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kRegs; i += 2) {
      const Two v = __builtin_amdgcn_raw_buffer_load_b64(b, (int)(offset + 4 * i), 0, 0);
      __builtin_memcpy(h + i, &v, 8);
    }
  }
}
template <int kRegs>
__device__ __forceinline__ void put_states(const float (&h)[kRegs], Buffer b, unsigned offset) {
  typedef unsigned Two __attribute__((ext_vector_type(2)));
  typedef unsigned Four __attribute__((ext_vector_type(4)));
  if constexpr (kRegs == 1) {
    put(b, offset, h[0]);
  } else if constexpr (kRegs % 4 == 0) {
#pragma unroll
    for (int i = 0; i < kRegs; i += 4) {
      Four v;
      __builtin_memcpy(&v, h + i, 16);
      __builtin_amdgcn_raw_buffer_store_b128(v, b, (int)(offset + 4 * i), 0, 0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kRegs; i += 2) {
      Two v;
      __builtin_memcpy(&v, h + i, 8);
      __builtin_amdgcn_raw_buffer_store_b64(v, b, (int)(offset + 4 * i), 0, 0);
    }
  }
}

// Where a lane stands.
struct Lane {
  int b, chunk, block, c0, c, q, len, t0, t1;  // c: its channel (maybe behind the last), c0: the workgroup's first; steps [t0, t1)
                                               // of the chunk, len of the sequence
  bool on;                                     // the channel exists
  int row;                                     // the channel, or the last one
  int in;                                      // the channel in the workgroup
};
__device__ __forceinline__ Lane lane_of(const ScanArgs& A) {
  Lane l;
  const int blocks = (A.D + kScanChannels - 1) / kScanChannels;
  const int id = blockIdx.x / blocks;
  l.block = blockIdx.x - id * blocks;
  l.b = id / A.chunks;
  l.chunk = id - l.b * A.chunks;
  l.in = threadIdx.x / 4;
  l.c0 = l.block * kScanChannels;
  l.c = l.c0 + l.in;
  l.q = threadIdx.x & 3;
  l.on = l.c < A.D;
  l.row = min(l.c, A.D - 1);
  l.len = A.lengths ? (int)min(max(A.lengths[l.b], (int64_t)0), (int64_t)A.L) : A.L;
  l.t0 = l.chunk * A.chunk;
  l.t1 = min(l.t0 + A.chunk, A.L);
  return l;
}

// A [B][L][channels] tensor, seen from a workgroup: lane q's values of the steps t + 4 m + q of a tile of kTile steps, zeros
// behind the sequence's length and the last channel, whatever memory holds there.  The tile's buffer is made of a pointer that
// moves with it and the steps left, by the same few scalar instructions for all.
template <typename T, int kTile>
struct Steps {
  const char* tile;     // the sequence's and workgroup's first channel in the tile's first step
  int row, width;       // bytes of a step, and of the channels from the first one on
  unsigned at;          // the lane's place in four steps
  __device__ __forceinline__ Steps(const void* p, long batch, long row_, const Lane& l, int t, int D)
      : tile((const char*)p + (l.b * batch + l.c0 + t * row_) * (long)sizeof(T)), row((int)row_ * (int)sizeof(T)),
        width((D - l.c0) * (int)sizeof(T)),
        at(!l.on ? kNowhere : (unsigned)l.q * (unsigned)row + (unsigned)(l.in * (int)sizeof(T))) {}
  __device__ __forceinline__ void move(int tiles) { tile += (long)tiles * kTile * row; }
  __device__ __forceinline__ Buffer steps(int left) const {  // left: of the tensor from the tile's first step on
    const int there = min(left, kTile);
    return buffer(tile, ((there - 1) * row + width) & (there > 0 ? -1 : 0));
  }
  __device__ __forceinline__ unsigned four(int m) const { return at + (unsigned)(4 * m * row); }
  template <int kCount>
  __device__ __forceinline__ void read(T (&v)[kCount], int left) const {
    const Buffer from = steps(left);
#pragma unroll
    for (int m = 0; m < kCount; ++m) v[m] = fetch<T>(from, four(m));
  }
  __device__ __forceinline__ void write(Buffer to, int m, float v) const { put(to, four(m), from_f32<T>(v)); }
  // Zeros in `steps` steps from the tile on (to the end of one), `left` as above.
  __device__ __forceinline__ void clear(int left, int steps) {
    for (; steps > 0; steps -= kTile, left -= kTile) {
      const Buffer to = this->steps(left);
#pragma unroll
      for (int m = 0; m < kTile / 4; ++m) write(to, m, 0.0f);
      move(1);
    }
  }
};

// The states of the workgroup's channels at a place of the padded layouts.
template <int kRegs>
__device__ __forceinline__ Buffer states_at(const float* base, long place, const Lane& l, int D, bool there) {
  constexpr int kPad = 4 * kRegs;
  return buffer(base + (place * D + l.c0) * kPad, (min(D - l.c0, kScanChannels) * kPad * 4) & (there ? -1 : 0));
}

// B and C of kSteps steps, on their way from memory to LDS.  Steps and states that are not there are zeros.
template <typename T, int kRegs, int kSteps>
struct Rows {
  static constexpr int kPad = 4 * kRegs, kEach = kSteps * kPad, kPer = (kEach + kThreads - 1) / kThreads;
  const char* tile[2];
  int row[2], width;
  T v[2][kPer];
  unsigned at[2][kPer];
  __device__ __forceinline__ Rows(const ScanArgs& A, int b, int t) {
    tile[0] = (const char*)A.Bm + (b * A.b_batch + t * A.b_row) * (long)sizeof(T);
    tile[1] = (const char*)A.Cm + (b * A.c_batch + t * A.c_row) * (long)sizeof(T);
    row[0] = (int)A.b_row * (int)sizeof(T);
    row[1] = (int)A.c_row * (int)sizeof(T);
    width = A.N * (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = i * kThreads + threadIdx.x, step = e / kPad, n = e % kPad;
#pragma unroll
      for (int w = 0; w < 2; ++w)
        at[w][i] = e < kEach && n < A.N ? (unsigned)step * (unsigned)row[w] + (unsigned)(n * (int)sizeof(T)) : kNowhere;
    }
  }
  __device__ __forceinline__ void move(int tiles) {
#pragma unroll
    for (int w = 0; w < 2; ++w) tile[w] += (long)tiles * kSteps * row[w];
  }
  __device__ __forceinline__ void read(int left) {  // left: steps of the sequence from the tile's first on
    const int there = min(left, kSteps);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const Buffer from = buffer(tile[w], ((there - 1) * row[w] + width) & (there > 0 ? -1 : 0));
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[w][i] = fetch<T>(from, at[w][i]);
    }
  }
  // [step][B, then C][state]
  __device__ __forceinline__ void write(float* lds) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = i * kThreads + threadIdx.x;
      if (kEach % kThreads == 0 || e < kEach) {
        float* to = lds + e / kPad * 2 * kPad + e % kPad;
        to[0] = to_f32(v[0][i]);
        to[kPad] = to_f32(v[1][i]);
      }
    }
  }
};

// B and C of kAhead steps, read while the steps before are computed.
template <int kRegs, int kAhead, bool kB, bool kC>
struct Ahead {
  static constexpr int kPad = 4 * kRegs;
  float B[kAhead][kRegs], C[kAhead][kRegs];
  __device__ __forceinline__ void read(const float* lds, int first) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
#pragma unroll
      for (int i = 0; i < kRegs; ++i) {
        if (kB) B[k][i] = lds[(first + k) * 2 * kPad + i];
        if (kC) C[k][i] = lds[(first + k) * 2 * kPad + kPad + i];
      }
  }
};

// The states that are there (kFull: all).  Others stay zeros: what multiplies them is zero too, but may meet infinity.
template <int kRegs, bool kFull>
struct There {
  bool is[kRegs];
  __device__ __forceinline__ There(const ScanArgs& A, int group) {
#pragma unroll
    for (int i = 0; i < kRegs; ++i) is[i] = kFull || group * kRegs + i < A.N;
  }
  __device__ __forceinline__ float operator()(int i, float v) const { return kFull || is[i] ? v : 0.0f; }
};

// A lane's A.
template <int kRegs>
__device__ __forceinline__ void load_decays(float (&a)[kRegs], const ScanArgs& A, const Lane& l, int group) {
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const int n = group * kRegs + i;
    a[i] = n < A.N ? decay_of(A.A[(long)l.row * A.N + n]) : 0.0f;
  }
}

// Keeps a value from being computed in a branch of its own.
__device__ __forceinline__ float here(float v) {
  asm volatile("" : "+v"(v));
  return v;
}

// Where a grid has no more than two workgroups a CU, the two waves of a SIMD come first by turns.  The older one always came first,
// was done early and left the other alone, which cannot use all cycles: forward of bf16 8 x 2048 x 4096 386 -> 359 us then.
// Workgroups go over the card's 256 CUs in order.  bf16, 1024 steps of 4096 channels, 16 states, us, without turns | with them:
//   sequences  4 (256 workgroups)  5 (320)    8 (512)    9 (576)    16 (1024)
//   forward    112 | 132           156 | 156  158 | 158  221 | 211  282 | 268
//   both ways  396 | 423           592 | 566  616 | 583  880 | 876  1158 | 1125
// (The border is that of the case measured first; those that these figures ask for are not drawn yet.)
__device__ __forceinline__ void take_turns(int tile) {
  if (gridDim.x > 512) return;
  if ((tile ^ (int)(blockIdx.x >> 8)) & 1) __builtin_amdgcn_s_setprio(1);
  else __builtin_amdgcn_s_setprio(0);
}

// ---- forward ------------------------------------------------------------------------------------------
// kEdges: of each chunk alone, from a state of zeros, its last state and the sum of its step sizes.
template <typename T, int kRegs, bool kFull, bool kEdges, bool kGated>
__global__ __launch_bounds__(kThreads) void k_scan_fwd(const ScanArgs A) {
  constexpr int kPad = Shape<kRegs>::kPad, kTile = Shape<kRegs>::kTile, kInterval = Shape<kRegs>::kInterval, kM = kTile / 4;
  constexpr int kAhead = Shape<kRegs>::kAhead;
  __shared__ float bc[2][kTile * 2 * kPad];
  const Lane l = lane_of(A);
  Steps<T, kTile> x(A.x, A.x_batch, A.x_row, l, l.t0, A.D), dt(A.dt, A.dt_batch, A.dt_row, l, l.t0, A.D);
  Steps<T, kTile> z(A.z, A.z_batch, A.z_row, l, l.t0, A.D), out(A.out, (long)A.L * A.D, A.D, l, l.t0, A.D);
  const float bias = A.bias ? A.bias[l.row] : 0.0f, skip = A.skip ? A.skip[l.row] : 0.0f;
  const unsigned mine = (unsigned)(l.in * kPad + l.q * kRegs) * 4;
  float a[kRegs], h[kRegs];
  const There<kRegs, kFull> there(A, l.q);
  load_decays<kRegs>(a, A, l, l.q);
  const long place = (long)l.b * A.chunks + l.chunk;
  float* state = A.state ? A.state + ((long)l.b * A.D + l.row) * A.N : nullptr;
#pragma unroll
  for (int i = 0; i < kRegs; ++i) h[i] = 0.0f;
  if (!kEdges && A.chunks > 1) fetch_states<kRegs>(h, states_at<kRegs>(A.edge, place, l, A.D, true), mine);
  else if (!kEdges && state)
#pragma unroll
    for (int i = 0; i < kRegs; ++i)
      if (l.q * kRegs + i < A.N) h[i] = state[l.q * kRegs + i];
  float total = 0.0f;
  const float* saved = A.saved + ((l.b * (long)((A.L + kInterval - 1) / kInterval) + l.t0 / kInterval) * A.D + l.c0) * kPad;
  const int saved_bytes = A.saved ? min(A.D - l.c0, kScanChannels) * kPad * 4 : 0;

  T xv[kM], dv[kM], zv[kM];
  Rows<T, kRegs, kTile> rows(A, l.b, l.t0);
  auto read = [&](int t) {
    x.read(xv, l.len - t);
    dt.read(dv, l.len - t);
    if (kGated) z.read(zv, l.len - t);
    rows.read(l.len - t);
    x.move(1);
    dt.move(1);
    if (kGated) z.move(1);
    rows.move(1);
  };
  read(l.t0);
  rows.write(bc[0]);
  __syncthreads();
  int t = l.t0;
  for (int turn = 0; t < min(l.t1, l.len); t += kTile, turn ^= 1) {
    take_turns(t / kTile);
    float s2[kM], u[kM], xs[kM], gate[kM];  // s2: the step size times log2(e)
    const int left = l.len - t - l.q;
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      const bool counts = 4 * m < left;
      const float v = to_f32(dv[m]) + bias, soft = here(softplus(v));
      const float s = counts ? (A.softplus ? soft : v) : 0.0f;  // (no step: the state stays)
      s2[m] = s * kLog2e;
      xs[m] = to_f32(xv[m]);
      u[m] = s * xs[m];
      gate[m] = 1.0f;
      if (kEdges) total += s;
      else if (kGated) gate[m] = to_f32(zv[m]) * sigmoid(to_f32(zv[m]));
    }
    // (behind the chunk's last tile the reads are another chunk's, or nothing)
    read(t + kTile);
    const Buffer to = out.steps(A.L - t);
    const float* lds = bc[turn] + l.q * kRegs;
    Ahead<kRegs, kAhead, true, !kEdges> ahead;
    ahead.read(lds, 0);
    float y[4];
    static_for<0, kTile / kAhead>([&](auto g_) {
      constexpr int g = decltype(g_)::value;
      const Ahead<kRegs, kAhead, true, !kEdges> now = ahead;
      if constexpr (g + 1 < kTile / kAhead) ahead.read(lds, (g + 1) * kAhead);
      static_for<0, kAhead>([&](auto k_) {
        constexpr int j = g * kAhead + decltype(k_)::value, m = j / 4, k = j % 4;
        if constexpr (!kEdges && j % kInterval == 0) {
          put_states<kRegs>(h, buffer(saved, saved_bytes & (t + j < A.L ? -1 : 0)), mine);
          saved += (long)A.D * kPad;
        }
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kRegs; ++i) {
          h[i] = there(i, __builtin_amdgcn_exp2f(of_lane<k>(s2[m]) * a[i]) * h[i] + of_lane<k>(u[m]) * now.B[j - g * kAhead][i]);
          if (!kEdges) sum += h[i] * now.C[j - g * kAhead][i];
        }
        y[k] = sum;
        if constexpr (!kEdges && k == 3) {
          const float o = (quad_sums(y) + skip * xs[m]) * gate[m];  // (outside the condition: all lanes of the quad take part)
          out.write(to, m, 4 * m < left ? o : 0.0f);
        }
      });
    });
    out.move(1);
    rows.write(bc[turn ^ 1]);
    __syncthreads();
  }
  if (!kEdges) out.clear(A.L - t, l.t1 - t);  // (the states stay as they are; the backward does not ask for them)
  if (kEdges) {
    put_states<kRegs>(h, states_at<kRegs>(A.edge, place, l, A.D, true), mine);
    total = quad_sum(total);
    if (l.on && l.q == 0) A.sums[place * A.D + l.c] = total;
  } else if (state && l.on && l.chunk == A.chunks - 1) {
#pragma unroll
    for (int i = 0; i < kRegs; ++i)
      if (l.q * kRegs + i < A.N) state[l.q * kRegs + i] = h[i];
  }
}

// ---- backward -----------------------------------------------------------------------------------------
// kEdges: of each chunk alone, without a gradient from behind it, the gradient of its first state, and the sum of its step sizes.
// (At most 256 registers: two waves a SIMD, where one leaves a third of its cycles unused; 64 states need more.)
// kWhole: all steps of all tiles count.  Otherwise the state that stays behind a sequence's end may be infinite or NaN, and times no
// gradient it would be NaN in dA: it is selected away.  8 x 2047 x 2048 with 16 states, fp16, both directions: 705 us without the
// selection, 723 with it (bf16 8 x 2048 x 4096: 1159 and 1165).  A branch a step costs as much; a second copy of the tile spills.
template <typename T, int kRegs, bool kFull, bool kEdges, bool kGated, bool kWhole>
__global__ __launch_bounds__(kThreads, kRegs <= 8 ? 2 : 1) void k_scan_bwd(const ScanArgs A) {
  constexpr int kPad = Shape<kRegs>::kPad, kTile = Shape<kRegs>::kInterval, kM = kTile / 4, kGroups = kTile * 2 * kRegs / 16;
  constexpr int kAhead = Shape<kRegs>::kAheadBack;
  __shared__ float bc[2][kTile * 2 * kPad];
  __shared__ float red[kEdges ? 1 : 2][4][kEdges ? 1 : kGroups * 64];
  const Lane l = lane_of(A);
  // the chunk's tiles, and the last one that the sequence reaches: behind it all gradients are zeros
  const int all = (l.t1 - l.t0 + kTile - 1) / kTile, tiles = max(0, (min(l.t1, l.len) - l.t0 + kTile - 1) / kTile);
  const int last = l.t0 + (tiles - 1) * kTile;
  const long full = (long)A.L * A.D;
  Steps<T, kTile> x(A.x, A.x_batch, A.x_row, l, last, A.D), dt(A.dt, A.dt_batch, A.dt_row, l, last, A.D);
  Steps<T, kTile> z(A.z, A.z_batch, A.z_row, l, last, A.D), dout(A.dout, full, A.D, l, last, A.D);
  Steps<T, kTile> dx(A.dx, full, A.D, l, last, A.D), ddt(A.ddt, full, A.D, l, last, A.D), dz(A.dz, full, A.D, l, last, A.D);
  const float bias = A.bias ? A.bias[l.row] : 0.0f, skip = A.skip ? A.skip[l.row] : 0.0f;
  const int group = states_of(threadIdx.x);  // of the lane's states
  const unsigned mine = (unsigned)(l.in * kPad + group * kRegs) * 4;
  float a[kRegs], carry[kRegs], dA[kRegs] = {}, dskip = 0.0f, dbias = 0.0f, total = 0.0f;
  const There<kRegs, kFull> is_there(A, group);
  load_decays<kRegs>(a, A, l, group);
  const long place = (long)l.b * A.chunks + l.chunk;
#pragma unroll
  for (int i = 0; i < kRegs; ++i) carry[i] = 0.0f;
  if (!kEdges && A.chunks > 1) fetch_states<kRegs>(carry, states_at<kRegs>(A.edge, place, l, A.D, true), mine);
  const float* saved = A.saved + ((l.b * (long)((A.L + kTile - 1) / kTile) + last / kTile) * A.D + l.c0) * kPad;
  const int saved_bytes = min(A.D - l.c0, kScanChannels) * kPad * 4;

  T xv[kM], dv[kM], zv[kM], gv[kM];
  float first[kRegs];
  Rows<T, kRegs, kTile> rows(A, l.b, last);
  auto read = [&](int t, bool there) {  // (before the chunk's first tile nothing is)
    const int left = there ? l.len - t : 0;
    x.read(xv, left);
    dt.read(dv, left);
    dout.read(gv, left);
    if (kGated) z.read(zv, left);
    rows.read(left);
    if (!kEdges) fetch_states<kRegs>(first, buffer(saved, saved_bytes & (there ? -1 : 0)), mine);
    x.move(-1);
    dt.move(-1);
    dout.move(-1);
    if (kGated) z.move(-1);
    rows.move(-1);
    saved -= (long)A.D * kPad;
  };
  if (!kEdges && tiles < all) {
    Steps<T, kTile> behind[3] = {dx, ddt, dz};
#pragma unroll
    for (int i = 0; i < (kGated ? 3 : 2); ++i) {
      behind[i].move(1);
      behind[i].clear(A.L - last - kTile, (all - tiles) * kTile);
    }
  }
  read(last, tiles > 0);
  rows.write(bc[0]);
  __syncthreads();
  for (int tile = tiles - 1, turn = 0; tile >= 0; --tile, turn ^= 1) {
    const int t = l.t0 + tile * kTile;
    take_turns(tile);
    // dzs: dout times silu's slope, slope: the step size's
    float s[kM], s2[kM], u[kM], xs[kM], dy[kM], dzs[kM], slope[kM], h[kRegs];
    const int left = l.len - t - l.q;
#pragma unroll
    for (int m = 0; m < kM; ++m) {
      const bool counts = 4 * m < left;
      const float v = to_f32(dv[m]) + bias;
      float sig;
      const float soft = here(softplus(v, sig));
      s[m] = counts ? (A.softplus ? soft : v) : 0.0f;
      s2[m] = s[m] * kLog2e;
      slope[m] = A.softplus ? here(sig) : 1.0f;  // (of the length's end on it meets zeros)
      xs[m] = to_f32(xv[m]);
      u[m] = s[m] * xs[m];
      dy[m] = to_f32(gv[m]);
      dzs[m] = 0.0f;
      if (kGated) {
        const float zf = to_f32(zv[m]), sg = sigmoid(zf);
        dzs[m] = dy[m] * (sg * (1.0f + zf * (1.0f - sg)));
        dy[m] *= zf * sg;
      }
      if (kEdges) total += s[m];
    }
#pragma unroll
    for (int i = 0; i < kRegs; ++i) h[i] = first[i];
    const Buffer to_dx = dx.steps(A.L - t), to_ddt = ddt.steps(A.L - t), to_dz = dz.steps(A.L - t);
    const float* lds = bc[turn] + group * kRegs;
    // the states of the tile again: before each step, and what the step leaves of them
    float before[kEdges ? 1 : kTile][kRegs], stay[kTile][kRegs];
    {
      Ahead<kRegs, kAhead, !kEdges, !kEdges && kGated> ahead;
      ahead.read(lds, 0);
      float y[4];
      static_for<0, kTile / kAhead>([&](auto g_) {
        constexpr int g = decltype(g_)::value;
        const Ahead<kRegs, kAhead, !kEdges, !kEdges && kGated> now = ahead;
        if constexpr (g + 1 < kTile / kAhead) ahead.read(lds, (g + 1) * kAhead);
        static_for<0, kAhead>([&](auto k_) {
          constexpr int j = g * kAhead + decltype(k_)::value, m = j / 4, k = j % 4;
          float sum = 0.0f;
#pragma unroll
          for (int i = 0; i < kRegs; ++i) {
            stay[j][i] = __builtin_amdgcn_exp2f(of_lane<k>(s2[m]) * a[i]);
            if constexpr (!kEdges) {
              before[j][i] = h[i];
              h[i] = is_there(i, stay[j][i] * h[i] + of_lane<k>(u[m]) * now.B[j - g * kAhead][i]);
              if (kGated) sum += h[i] * now.C[j - g * kAhead][i];
            }
          }
          y[k] = sum;
          if constexpr (!kEdges && k == 3) __builtin_amdgcn_sched_barrier(0);  // (nothing moves over four steps: no registers for it)
          if constexpr (!kEdges && kGated && k == 3) {
            const float o = dzs[m] * (quad_sums(y) + skip * xs[m]);
            dz.write(to_dz, m, 4 * m < left ? o : 0.0f);
          }
        });
      });
    }
    float vals[16], dA_tile[kRegs] = {}, of_b[4], of_a[4];
    Ahead<kRegs, kAhead, !kEdges, true> ahead;
    ahead.read(lds, kTile - kAhead);
    static_for<0, kTile / kAhead>([&](auto g_) {
      constexpr int g = kTile / kAhead - 1 - decltype(g_)::value;
      const Ahead<kRegs, kAhead, !kEdges, true> now = ahead;
      if constexpr (g > 0) ahead.read(lds, (g - 1) * kAhead);
      static_for<0, kAhead>([&](auto k_) {
        constexpr int j = g * kAhead + kAhead - 1 - decltype(k_)::value, m = j / 4, k = j % 4;
        // the tile before, once the first of its successor's states are done with (their registers hold it)
        if constexpr (j == kTile * 3 / 4 - 1) read(t - kTile, tile > 0);
        float gr[kRegs], sB = 0.0f, sA = 0.0f;
#pragma unroll
        for (int i = 0; i < kRegs; ++i) {
          gr[i] = is_there(i, now.C[j - g * kAhead][i] * of_lane<k>(dy[m]) + carry[i]);
          carry[i] = gr[i] * stay[j][i];
          if constexpr (!kEdges) {
            sB += gr[i] * now.B[j - g * kAhead][i];
            const float w = kWhole || j < l.len - t ? carry[i] * before[j][i] : 0.0f;
            sA += w * a[i];
            dA_tile[i] += w * of_lane<k>(s[m]);
          }
        }
        if constexpr (!kEdges) {
          of_b[k] = sB;
          of_a[k] = sA;
          static_for<0, 2 * kRegs>([&](auto i_) {
            constexpr int i = decltype(i_)::value, value = (kTile - 1 - j) * 2 * kRegs + i;
            vals[value % 16] = i < kRegs ? gr[i % kRegs] * of_lane<k>(u[m]) : h[i % kRegs] * of_lane<k>(dy[m]);
            if (value % 16 == 15) red[turn][threadIdx.x >> 6][value / 16 * 64 + (threadIdx.x & 63)] = wave_sums(vals);
          });
#pragma unroll
          for (int i = 0; i < kRegs; ++i) h[i] = before[j][i];
          if constexpr (k == 0) __builtin_amdgcn_sched_barrier(0);
          if constexpr (k == 0) {
            const float gB = quad_sums(of_b), gA = quad_sums(of_a);
            const bool counts = 4 * m < left;
            const float ddtv = counts ? (xs[m] * gB + gA) * slope[m] : 0.0f;
            dskip += dy[m] * xs[m];
            dbias += ddtv;
            dx.write(to_dx, m, counts ? s[m] * gB + skip * dy[m] : 0.0f);
            ddt.write(to_ddt, m, ddtv);
          }
        }
      });
    });
#pragma unroll
    for (int i = 0; i < kRegs; ++i) dA[i] += dA_tile[i];
    dx.move(-1);
    ddt.move(-1);
    if (kGated) dz.move(-1);
    rows.write(bc[turn ^ 1]);
    __syncthreads();
    if (!kEdges) {
      // the sums over this workgroup's channels: [step][B or C][state]
      float* part = A.part_bc + (((long)l.block * A.B + l.b) * A.L + t) * 2 * kPad;
      const int there = min(kTile, l.len - t) * 2 * kPad;  // (no others are added up)
#pragma unroll
      for (int i = 0; i < (kTile * 2 * kPad + kThreads - 1) / kThreads; ++i) {
        const int at = i * kThreads + (int)threadIdx.x;
        if (at >= there) break;
        const int j = at / (2 * kPad), which = at / kPad & 1, n = at % kPad;
        const int value = (kTile - 1 - j) * 2 * kRegs + which * kRegs + n % kRegs, v = value % 16, odd = v >> 2 & 1;
        // (where wave_sums leaves it)
        const int lane = (v & 8) + (v & 4) + (v & 2) * 8 + (v & 1) * 32 + (odd ? 3 - n / kRegs : n / kRegs), from = value / 16 * 64 + lane;
        part[at] = (red[turn][0][from] + red[turn][1][from]) + (red[turn][2][from] + red[turn][3][from]);
      }
    }
  }
  if (kEdges) {
    put_states<kRegs>(carry, states_at<kRegs>(A.edge, place, l, A.D, true), mine);
    total = quad_sum(total);
    if (l.on && l.q == 0) A.sums[place * A.D + l.c] = total;
    return;
  }
  float* par = A.part_par + (place * A.D + l.row) * (A.N + 2);
  dskip = quad_sum(dskip);
  dbias = quad_sum(dbias);
  if (!l.on) return;
#pragma unroll
  for (int i = 0; i < kRegs; ++i)
    if (group * kRegs + i < A.N) par[group * kRegs + i] = dA[i];
  if (l.q == 0) {
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
  const float u = s * x, s2 = s * kLog2e;
  const T *Bm = (const T*)A.Bm + b * A.b_batch, *Cm = (const T*)A.Cm + b * A.c_batch;
  float* h = A.state + row * A.N;
  const float* a = A.A + (long)c * A.N;
  float y = 0.0f;
  if (A.N % 4 == 0 && (((uintptr_t)A.state | (uintptr_t)A.A) & 15) == 0) {
    for (int n = 4 * q; n < A.N; n += 16) {
      const float4 hv = *(const float4*)(h + n), av = *(const float4*)(a + n);
      float hs[4] = {hv.x, hv.y, hv.z, hv.w}, as[4] = {av.x, av.y, av.z, av.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        hs[i] = fmaf(__builtin_amdgcn_exp2f(s2 * decay_of(as[i])), hs[i], u * to_f32(Bm[n + i]));
        y = fmaf(hs[i], to_f32(Cm[n + i]), y);
      }
      if (counts && at < all) *(float4*)(h + n) = make_float4(hs[0], hs[1], hs[2], hs[3]);
    }
  } else {  // (the same operations in the same order)
    for (int first = 4 * q; first < A.N; first += 16)
      for (int n = first; n < min(first + 4, A.N); ++n) {
        const float v = fmaf(__builtin_amdgcn_exp2f(s2 * decay_of(a[n])), h[n], u * to_f32(Bm[n]));
        y = fmaf(v, to_f32(Cm[n]), y);
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
// dB and dC: [blocks][B][L][2][padded] to [B][L][N] twice, zeros behind a sequence's length.  (Every kReduceBlocks workgroups: a
// grid holds fewer than 2^32 threads.)
constexpr long kReduceBlocks = 1 << 20;
template <typename T>
__global__ __launch_bounds__(256) void k_scan_reduce(const float* part, int blocks, long rows, int padded, int N, int L, const int64_t* lengths,
                                                     T* dB, T* dC) {
  const long all = rows * 2 * padded;
  for (long at = (long)blockIdx.x * 256 + threadIdx.x; at < all; at += kReduceBlocks * 256) {
    const int n = (int)(at % padded);
    if (n >= N) continue;
    const long row = at / (2 * padded);
    float s = 0.0f;
    if (!lengths || row % L < lengths[row / L])
#pragma unroll 8
      for (int k = 0; k < blocks; ++k) s += part[k * all + at];
    T* to = at / padded & 1 ? dC : dB;
    if (to) to[row * N + n] = from_f32<T>(s);
  }
}

template <typename T, int kRegs, bool kFull>
hipError_t launch(ScanPass pass, const ScanArgs& A, hipStream_t st) {
  const dim3 grid((unsigned)((long)A.B * A.chunks * ((A.D + kScanChannels - 1) / kScanChannels)));
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, st, A);
    return hipGetLastError();
  };
  switch (pass) {
    case ScanPass::kForward: return A.z ? go(k_scan_fwd<T, kRegs, kFull, false, true>) : go(k_scan_fwd<T, kRegs, kFull, false, false>);
    case ScanPass::kEdges: return go(k_scan_fwd<T, kRegs, kFull, true, false>);
    case ScanPass::kBackward:
      if (!A.lengths && A.L % scan_interval(kRegs) == 0)
        return A.z ? go(k_scan_bwd<T, kRegs, kFull, false, true, true>) : go(k_scan_bwd<T, kRegs, kFull, false, false, true>);
      return A.z ? go(k_scan_bwd<T, kRegs, kFull, false, true, false>) : go(k_scan_bwd<T, kRegs, kFull, false, false, false>);
    case ScanPass::kBackwardEdges:  // (dA is not among its sums)
      return A.z ? go(k_scan_bwd<T, kRegs, kFull, true, true, true>) : go(k_scan_bwd<T, kRegs, kFull, true, false, true>);
    case ScanPass::kStep: break;
  }
  return hipErrorInvalidValue;
}

template <typename T>
hipError_t launch_scan(ScanPass pass, const ScanArgs& A, hipStream_t st) {
  if (pass == ScanPass::kStep) {
    hipLaunchKernelGGL(k_scan_step<T>, dim3((unsigned)(((long)A.B * A.D * 4 + kThreads - 1) / kThreads)), dim3(kThreads), 0, st, A);
    return hipGetLastError();
  }
  switch (scan_regs(A.N)) {
    case 1: return A.N == 4 * 1 ? launch<T, 1, true>(pass, A, st) : launch<T, 1, false>(pass, A, st);
    case 2: return A.N == 4 * 2 ? launch<T, 2, true>(pass, A, st) : launch<T, 2, false>(pass, A, st);
    case 4: return A.N == 4 * 4 ? launch<T, 4, true>(pass, A, st) : launch<T, 4, false>(pass, A, st);
    case 6: return A.N == 4 * 6 ? launch<T, 6, true>(pass, A, st) : launch<T, 6, false>(pass, A, st);
    case 8: return A.N == 4 * 8 ? launch<T, 8, true>(pass, A, st) : launch<T, 8, false>(pass, A, st);
    case 16: return A.N == 4 * 16 ? launch<T, 16, true>(pass, A, st) : launch<T, 16, false>(pass, A, st);
  }
  return hipErrorInvalidValue;
}

template <typename T>
hipError_t reduce_scan(const ScanArgs& A, int padded, void* dB, void* dC, hipStream_t st) {
  const long rows = (long)A.B * A.L;
  hipLaunchKernelGGL(k_scan_reduce<T>, dim3((unsigned)std::min(kReduceBlocks, (rows * 2 * padded + 255) / 256)), dim3(256), 0, st, A.part_bc,
                     (A.D + kScanChannels - 1) / kScanChannels, rows, padded, A.N, A.L, A.lengths, (T*)dB, (T*)dC);
  return hipGetLastError();
}

}  // namespace
}  // namespace kans
