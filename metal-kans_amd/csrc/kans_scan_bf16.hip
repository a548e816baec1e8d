// The selective scan on bf16 tensors.
#include "kans_scan_kernel.h"

namespace kans {
hipError_t scan_launch_bf16(ScanPass pass, const ScanArgs& A, hipStream_t st) { return launch_scan<__bf16>(pass, A, st); }
hipError_t scan_reduce_bf16(const ScanArgs& A, int padded, void* dB, void* dC, hipStream_t st) {
  return reduce_scan<__bf16>(A, padded, dB, dC, st);
}
}  // namespace kans
