// The selective scan on fp16 tensors.
#include "kans_scan_kernel.h"

namespace kans {
hipError_t scan_launch_f16(ScanPass pass, const ScanArgs& A, hipStream_t st) { return launch_scan<_Float16>(pass, A, st); }
hipError_t scan_reduce_f16(const ScanArgs& A, int padded, void* dB, void* dC, hipStream_t st) {
  return reduce_scan<_Float16>(A, padded, dB, dC, st);
}
}  // namespace kans
