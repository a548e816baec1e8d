// The selective scan's arguments and launches, shared by its entry points (kans_scan.hip) and its kernels, one translation
// unit for each element type (kans_scan_{f32,f16,bf16}.hip around kans_scan_kernel.h).
#pragma once
#include <hip/hip_runtime.h>

#include <cfloat>

#include "kans_api_internal.h"

namespace kans {

struct ScanArgs {
  const void *x, *dt, *Bm, *Cm, *z, *dout;
  const float *A, *skip, *bias;
  float* state;               // [B][D][N], read and written; or null
  const int64_t* lengths;
  void* out;
  float* saved;               // [B][ceil(L / interval)][D][padded N]: the states before every `interval` steps
  // Elements between sequences and between steps of the inputs, whose channels and states lie side by side.
  long x_batch, x_row, dt_batch, dt_row, b_batch, b_row, c_batch, c_row, z_batch, z_row;
  int B, L, D, N;
  int softplus;
  // Where a sequence is cut in chunks (chunks > 1): of `chunk` steps each, their first states [B][chunks][D][padded N] (or,
  // backward, the gradients behind their last), and the sums of the step sizes [B][chunks][D].
  int chunk, chunks;
  float *edge, *sums;
  // backward
  void *dx, *ddt, *dz;
  float* part_bc;             // [channel blocks][B][L][2][padded N]
  float* part_par;            // [B][chunks][D][N + 2]: dA, dskip, dbias
};

constexpr int kScanChannels = 64;  // of a workgroup

// exp(s A) is the hardware's exponential of (s log2(e)) A: A log2(e) would overflow for the largest A, and a step of size zero must
// leave the state as it is.  Minus infinity counts as the lowest number for the same reason.
__device__ __forceinline__ float decay_of(float a) { return a == -__builtin_inff() ? -FLT_MAX : a; }

// Registers of a lane for the states, four lanes a channel; steps between two saved states.
inline int scan_regs(int N) {
  for (int r : {1, 2, 4, 6, 8, 16})
    if (N <= 4 * r) return r;
  return 0;
}
constexpr int scan_interval(int regs) { return regs <= 4 ? 16 : regs <= 6 ? 8 : 4; }

enum class ScanPass { kForward, kEdges, kBackward, kBackwardEdges, kStep };
hipError_t scan_launch_f32(ScanPass pass, const ScanArgs& A, hipStream_t st);
hipError_t scan_launch_f16(ScanPass pass, const ScanArgs& A, hipStream_t st);
hipError_t scan_launch_bf16(ScanPass pass, const ScanArgs& A, hipStream_t st);
// dB, dC [B][L][N] of their type from part_bc
hipError_t scan_reduce_f32(const ScanArgs& A, int padded, void* dB, void* dC, hipStream_t st);
hipError_t scan_reduce_f16(const ScanArgs& A, int padded, void* dB, void* dC, hipStream_t st);
hipError_t scan_reduce_bf16(const ScanArgs& A, int padded, void* dB, void* dC, hipStream_t st);

}  // namespace kans
