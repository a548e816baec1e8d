// Cross entropy kernels of fp16 inputs.
#include "kans_xent_kernel.h"

namespace kans {
template size_t xent_workspace<_Float16>(int, int, int, bool, bool);
template hipError_t xent_forward<_Float16>(const XentCall&, hipStream_t);
template hipError_t xent_backward<_Float16>(const XentCall&, hipStream_t);
}  // namespace kans
