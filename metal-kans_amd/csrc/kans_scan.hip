// Selective state space scan: entry points, and what joins a sequence's chunks (gfx950).  The kernels are in kans_scan_kernel.h.
//
//   s[t] = softplus(dt[t] + bias),  h[t] = exp(s[t] A) h[t-1] + s[t] x[t] B[t],  y[t] = C[t] . h[t] + skip x[t],  out = y z sigmoid(z)
//
// for each channel, with a state h of N numbers; B and C are shared by a sequence's channels.  Backward, with dy = dout z sigmoid(z):
//   g[t] = C[t] dy[t] + exp(s[t+1] A) g[t+1]                       (the gradient of h[t])
//   dC[t] = sum dy h[t],  dB[t] = sum g[t] s x                     (over the channels)
//   k[t] = g[t] exp(s[t] A) h[t-1]
//   dx = s (g . B) + skip dy,  ds = x (g . B) + k . A,  dA = sum k s,  dskip = sum dy x,  ddt = ds softplus'(dt + bias)
//
// All of it in fp32; h does not leave the registers but for every 16th step (8th or 4th for many states), where the forward of a
// training step keeps it: the backward runs through the 16 steps again and then back.
//
// The vector units bound it, not memory: a step of 16 channels and 16 states takes a wave 32 instructions forward (20 of them
// the recurrence's own: product, exponential, product and two sums for each four states) and 93 backward (24 for the states again,
// 32 for the gradients, 17 for the sums of dB and dC over the channels).  Four lanes share a channel: with one, a
// wave would have 64 channels and there would be too few waves; with 16, sums over the states would cost as much as the
// recurrence.  bf16 8 x 2048 x 4096, 16 states: forward 327 - 332 us, backward 858 - 877 (84 and 86 % of the issue slots taken, at 2.2 GHz),
// of which the bytes alone take 160 and 280; 1 x 8192 x 1024 fp16 forward 44 us and 32 for the chunks' edges.  What lies
// behind a sequence's end is cleared, not computed.
// A batch of B sequences and D channels has B D / 16 waves.  Where those are too few for the card the sequence is cut in chunks: a
// first pass runs each from a state of zeros for its last state (the decay over a chunk is exp(A sum s)), k_scan_join adds
// these up to the state before each chunk, and the scan runs the chunks beside each other.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <initializer_list>

#include "kans_scan.h"

namespace kans {
namespace {

// Per chunk in order (backward: from the last), edge becomes what comes into it: H, then H exp(A sum s) + edge.
__global__ __launch_bounds__(64) void k_scan_join(const ScanArgs A, int padded, bool backward) {
  const long at = (long)blockIdx.x * 64 + threadIdx.x, states = (long)A.D * padded;
  if (at >= A.B * states) return;
  const long b = at / states, to = at - b * states, d = to / padded;
  const int n = (int)(to - d * padded);
  if (n >= A.N) return;  // (zeros throughout)
  const float a = decay_of(A.A[d * A.N + n]);
  float h = !backward && A.state ? A.state[(b * A.D + d) * A.N + n] : 0.0f;
  constexpr int kAhead = 16;  // chunks whose values are under way together
  for (int first = 0; first < A.chunks; first += kAhead) {
    float e[kAhead], s[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int in_order = min(first + i, A.chunks - 1);
      const long place = b * A.chunks + (backward ? A.chunks - 1 - in_order : in_order);
      e[i] = A.edge[place * A.D * padded + to];
      s[i] = A.sums[place * A.D + d];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (first + i >= A.chunks) break;
      const long place = b * A.chunks + (backward ? A.chunks - 1 - first - i : first + i);
      A.edge[place * A.D * padded + to] = h;
      // (in two halves: a chunk may let a small state grow by more than fp32 holds; and nothing times that is nothing)
      const float half = __builtin_amdgcn_exp2f(0.5f * kLog2e * s[i] * a), grown = half * (half * h);
      h = (h == 0.0f ? 0.0f : grown) + e[i];
    }
  }
}

// Sums of the parameters' partial rows, [rows][D][N + 2].
__global__ __launch_bounds__(256) void k_scan_params(const float* part, long rows, int D, int N, float* dA, float* dskip, float* dbias) {
  const long at = (long)blockIdx.x * 256 + threadIdx.x, all = (long)D * (N + 2);
  if (at >= all) return;
  float s = 0.0f;
#pragma unroll 4
  for (long r = 0; r < rows; ++r) s += part[r * all + at];
  const long d = at / (N + 2);
  const int n = (int)(at - d * (N + 2));
  if (n < N) {
    if (dA) dA[d * N + n] = s;
  } else if (n == N) {
    if (dskip) dskip[d] = s;
  } else if (dbias) {
    dbias[d] = s;
  }
}

hipError_t launch(int dtype, ScanPass pass, const ScanArgs& A, hipStream_t st) {
  return dtype == DT_F32 ? scan_launch_f32(pass, A, st) : dtype == DT_F16 ? scan_launch_f16(pass, A, st) : scan_launch_bf16(pass, A, st);
}

constexpr int kMaxStates = 64, kMinChunk = 64;
constexpr long kEnoughWaves = 1024, kWantedWaves = 4096;

// Chunks of a sequence where its waves do not give every SIMD one: four for each, eight if the chunks keep 128 steps.  us, bf16,
// 16 states, forward and both directions, one chunk | two | four | eight waves a SIMD:
//   1 x 8192 x 1024   869  3276 |  94 290 |  88 275 |  96 294
//   2 x 8192 x 4096   978  3484 |         | 502 1735 | 471 1661
//   3 x 777 x 1300    140   455 |  71 213 |  63 185 |  62 183  (24 states)
//   16 x 1000 x 1500  158   660 |         | 201  720 | 186  686  (1536 waves: whole)
struct ScanPlan {
  int blocks, chunk, chunks, interval, padded;
  long edges;                        // floats of the chunks' edges and sums
  long part_bc, part_par, saved;     // floats
};
ScanPlan plan_scan(int B, int L, int D, int N) {
  ScanPlan p{};
  const int regs = scan_regs(N);
  p.interval = scan_interval(regs);
  p.padded = 4 * regs;
  p.blocks = (D + kScanChannels - 1) / kScanChannels;
  const long waves = 4L * p.blocks * std::max(B, 1);
  p.chunk = std::max(L, 1);
  if (waves < kEnoughWaves && L >= 2 * kMinChunk) {
    const long four = (kWantedWaves + waves - 1) / waves;
    const long want = std::min(std::max(four, std::min(2 * four, (long)L / (2 * kMinChunk))), (long)L / kMinChunk);
    p.chunk = (int)(((L + want - 1) / want + 15) & ~15L);
  }
  p.chunks = std::max(1, (L + p.chunk - 1) / p.chunk);
  p.edges = p.chunks > 1 ? (long)B * p.chunks * D * (p.padded + 1) : 0;
  p.edges = (p.edges + 3) & ~3L;
  p.part_bc = (long)p.blocks * B * L * 2 * p.padded;
  p.part_par = (long)B * p.chunks * D * (N + 2);
  p.saved = (long)B * ((L + p.interval - 1) / p.interval) * D * p.padded;
  return p;
}

int check_scan(int dtype, int B, int L, int D, int N) {
  if (dtype != DT_F32 && dtype != DT_F16 && dtype != DT_BF16) return kans_fail(KANS_ERR_ARG, "dtype %d", dtype);
  if (B < 0 || L < 0 || D <= 0 || N <= 0) return kans_fail(KANS_ERR_ARG, "bad dims B=%d L=%d D=%d N=%d", B, L, D, N);
  if (N > kMaxStates) return kans_fail(KANS_ERR_UNSUPPORTED, "%d states, up to %d", N, kMaxStates);
  // (a grid holds fewer than 2^32 threads along x, a channel four; the kernels reach 16 steps by offsets below 2^30 and the
  // outputs have D elements a step)
  const long blocks = ((long)D + kScanChannels - 1) / kScanChannels;
  if (L > (1 << 30) || D >= 1 << 23 || (long)B * blocks >= 1L << 22 || (long)B * L * 2 * kMaxStates >= 1L << 38)
    return kans_fail(KANS_ERR_UNSUPPORTED, "B=%d L=%d D=%d fit no grid", B, L, D);
  return 0;
}

// Elements between sequences and between the L steps of `width` channels or states.  (Steps in each other's memory would be read
// behind a length, where a buffer's end is to give zeros.)
struct Rows {
  long batch, row;
  int width;
};
int check_rows(int L, std::initializer_list<Rows> tensors) {
  for (const Rows& t : tensors) {
    if (t.batch < 0) return kans_fail(KANS_ERR_ARG, "%ld elements between sequences", t.batch);
    if (t.row < 0 || t.row >= 1L << 23) return kans_fail(KANS_ERR_UNSUPPORTED, "%ld elements between steps, fewer than 2^23", t.row);
    if (L > 1 && t.row > 0 && t.row < t.width)
      return kans_fail(KANS_ERR_UNSUPPORTED, "%ld elements between steps of %d: 0, or at least these", t.row, t.width);
  }
  return 0;
}

int check_workspace(const void* workspace, long bytes, long need) {
  if (need && (!workspace || (uintptr_t)workspace % 16 || bytes < need))
    return kans_fail(KANS_ERR_ARG, "workspace of %ld bytes, %ld at a multiple of 16 needed", workspace ? bytes : 0, need);
  return 0;
}

}  // namespace
}  // namespace kans

using namespace kans;

extern "C" {

long kans_selective_scan_saved(int B, int L, int D, int N) {
  const int rc = check_scan(DT_F32, B, L, D, N);
  return rc ? rc : plan_scan(B, L, D, N).saved * (long)sizeof(float);
}

long kans_selective_scan_workspace(int B, int L, int D, int N, int backward) {
  const int rc = check_scan(DT_F32, B, L, D, N);
  if (rc) return rc;
  const ScanPlan p = plan_scan(B, L, D, N);
  return (p.edges + (backward ? p.part_bc + p.part_par : 0)) * (long)sizeof(float);
}

int kans_selective_scan_forward(int dtype, const void* x, long x_batch, long x_row, const void* dt, long dt_batch, long dt_row,
                                const float* A, const void* Bm, long b_batch, long b_row, const void* Cm, long c_batch, long c_row,
                                const float* skip, const void* z, long z_batch, long z_row, const float* dt_bias, int softplus,
                                float* state, const int64_t* lengths, void* out, float* saved, int B, int L, int D, int N,
                                void* workspace, long workspace_bytes, void* stream) {
  int rc = check_scan(dtype, B, L, D, N);
  if (rc || B == 0 || L == 0) return rc;
  if (!x || !dt || !A || !Bm || !Cm || !out) return kans_fail(KANS_ERR_ARG, "null argument");
  if ((rc = check_rows(L, {{x_batch, x_row, D}, {dt_batch, dt_row, D}, {b_batch, b_row, N}, {c_batch, c_row, N},
                          {z ? z_batch : 0, z ? z_row : 0, D}}))) return rc;
  const ScanPlan p = plan_scan(B, L, D, N);
  if ((rc = check_workspace(workspace, workspace_bytes, p.edges * (long)sizeof(float)))) return rc;
  std::lock_guard<std::mutex> lk(kans_mutex());
  if ((rc = kans_ensure_init())) return rc;
  hipStream_t st = kans_caller_stream(stream);
  ScanArgs S{};
  S.x = x; S.dt = dt; S.Bm = Bm; S.Cm = Cm; S.z = z; S.A = A; S.skip = skip; S.bias = dt_bias;
  S.x_batch = x_batch; S.x_row = x_row; S.dt_batch = dt_batch; S.dt_row = dt_row; S.b_batch = b_batch; S.b_row = b_row;
  S.c_batch = c_batch; S.c_row = c_row; S.z_batch = z_batch; S.z_row = z_row;
  S.state = state; S.lengths = lengths; S.out = out; S.saved = saved;
  S.B = B; S.L = L; S.D = D; S.N = N; S.softplus = softplus; S.chunk = p.chunk; S.chunks = p.chunks;
  if (L == 1 && state && !saved) {
    HIP_TRY(launch(dtype, ScanPass::kStep, S, st));
    return 0;
  }
  if (p.chunks > 1) {
    S.edge = (float*)workspace;
    S.sums = S.edge + (long)B * p.chunks * D * p.padded;
    HIP_TRY(launch(dtype, ScanPass::kEdges, S, st));
    hipLaunchKernelGGL(k_scan_join, dim3((unsigned)(((long)B * D * p.padded + 63) / 64)), dim3(64), 0, st, S, p.padded, false);
    HIP_TRY(hipGetLastError());
  }
  HIP_TRY(launch(dtype, ScanPass::kForward, S, st));
  return 0;
}

int kans_selective_scan_backward(int dtype, const void* x, long x_batch, long x_row, const void* dt, long dt_batch, long dt_row,
                                 const float* A, const void* Bm, long b_batch, long b_row, const void* Cm, long c_batch, long c_row,
                                 const float* skip, const void* z, long z_batch, long z_row, const float* dt_bias, int softplus,
                                 const int64_t* lengths, const float* saved, const void* dout, void* dx, void* ddt, float* dA, void* dB,
                                 void* dC, float* dskip, void* dz, float* ddt_bias, int B, int L, int D, int N, void* workspace,
                                 long workspace_bytes, void* stream) {
  int rc = check_scan(dtype, B, L, D, N);
  if (rc) return rc;
  const bool any = B > 0 && L > 0;
  if (any && (!x || !dt || !A || !Bm || !Cm || !saved || !dout || !dx || !ddt || (z && !dz))) return kans_fail(KANS_ERR_ARG, "null argument");
  if ((dskip && !skip) || (dz && !z) || (ddt_bias && !dt_bias)) return kans_fail(KANS_ERR_ARG, "gradient of an input that is not there");
  if (any && (rc = check_rows(L, {{x_batch, x_row, D}, {dt_batch, dt_row, D}, {b_batch, b_row, N}, {c_batch, c_row, N},
                          {z ? z_batch : 0, z ? z_row : 0, D}}))) return rc;
  const ScanPlan p = plan_scan(B, L, D, N);
  if ((rc = check_workspace(workspace, workspace_bytes, (p.edges + p.part_bc + p.part_par) * (long)sizeof(float)))) return rc;
  std::lock_guard<std::mutex> lk(kans_mutex());
  if ((rc = kans_ensure_init())) return rc;
  hipStream_t st = kans_caller_stream(stream);
  ScanArgs S{};
  S.x = x; S.dt = dt; S.Bm = Bm; S.Cm = Cm; S.z = z; S.A = A; S.skip = skip; S.bias = dt_bias; S.dout = dout;
  S.x_batch = x_batch; S.x_row = x_row; S.dt_batch = dt_batch; S.dt_row = dt_row; S.b_batch = b_batch; S.b_row = b_row;
  S.c_batch = c_batch; S.c_row = c_row; S.z_batch = z_batch; S.z_row = z_row;
  S.lengths = lengths; S.saved = (float*)saved; S.dx = dx; S.ddt = ddt; S.dz = dz;
  S.B = B; S.L = L; S.D = D; S.N = N; S.softplus = softplus; S.chunk = p.chunk; S.chunks = p.chunks;
  S.edge = (float*)workspace;
  S.sums = S.edge + (long)B * p.chunks * D * p.padded;
  S.part_bc = (float*)workspace + p.edges;
  S.part_par = S.part_bc + p.part_bc;
  if (any) {
    if (p.chunks > 1) {
      HIP_TRY(launch(dtype, ScanPass::kBackwardEdges, S, st));
      hipLaunchKernelGGL(k_scan_join, dim3((unsigned)(((long)B * D * p.padded + 63) / 64)), dim3(64), 0, st, S, p.padded, true);
      HIP_TRY(hipGetLastError());
    }
    HIP_TRY(launch(dtype, ScanPass::kBackward, S, st));
    if (dB || dC)
      HIP_TRY(dtype == DT_F32 ? scan_reduce_f32(S, p.padded, dB, dC, st) : dtype == DT_F16 ? scan_reduce_f16(S, p.padded, dB, dC, st)
                                                                                           : scan_reduce_bf16(S, p.padded, dB, dC, st));
  }
  if (dA || dskip || ddt_bias) {
    hipLaunchKernelGGL(k_scan_params, dim3((unsigned)(((long)D * (N + 2) + 255) / 256)), dim3(256), 0, st, S.part_par,
                       any ? (long)B * p.chunks : 0L, D, N, dA, dskip, ddt_bias);
    HIP_TRY(hipGetLastError());
  }
  return 0;
}

}  // extern "C"
