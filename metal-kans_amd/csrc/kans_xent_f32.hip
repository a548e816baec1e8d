// Cross entropy kernels of fp32 (products of three bf16 terms) inputs.
#include "kans_xent_kernel.h"

namespace kans {
template size_t xent_workspace<float>(int, int, int, bool, bool);
template hipError_t xent_forward<float>(const XentCall&, hipStream_t);
template hipError_t xent_backward<float>(const XentCall&, hipStream_t);
}  // namespace kans
