// Cross entropy kernels of bf16 inputs.
#include "kans_xent_kernel.h"

namespace kans {
template size_t xent_workspace<__bf16>(int, int, int, bool, bool);
template hipError_t xent_forward<__bf16>(const XentCall&, hipStream_t);
template hipError_t xent_backward<__bf16>(const XentCall&, hipStream_t);
}  // namespace kans
