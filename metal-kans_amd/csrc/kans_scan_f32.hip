// The selective scan on fp32 tensors.
#include "kans_scan_kernel.h"

namespace kans {
hipError_t scan_launch_f32(ScanPass pass, const ScanArgs& A, hipStream_t st) { return launch_scan<float>(pass, A, st); }
hipError_t scan_reduce_f32(const ScanArgs& A, int padded, void* dB, void* dC, hipStream_t st) {
  return reduce_scan<float>(A, padded, dB, dC, st);
}
}  // namespace kans
