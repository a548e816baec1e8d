// Entry points of the cross entropy of a linear head (kans_xent.h); one unit per element type holds the kernels.
#include "kans_api_internal.h"
#include "kans_xent.h"

using namespace kans;

namespace {

int check_xent(int dtype, const void* H, const void* W, const void* target, int N, int D, int V, int reduction,
               const void* state) {
  if (dtype != DT_F32 && dtype != DT_F16 && dtype != DT_BF16) return kans_fail(KANS_ERR_ARG, "unknown dtype %d", dtype);
  if (N < 0 || D <= 0 || V <= 0) return kans_fail(KANS_ERR_ARG, "bad dims N=%d D=%d V=%d", N, D, V);
  if (reduction < 0 || reduction > 2) return kans_fail(KANS_ERR_ARG, "reduction %d, must be 0 (none), 1 (mean) or 2 (sum)", reduction);
  if (N > 0 && (!H || !W || !target || !state)) return kans_fail(KANS_ERR_ARG, "null hidden, weight, target or state");
  if (((uintptr_t)target & 7) || ((uintptr_t)state & 3)) return kans_fail(KANS_ERR_ARG, "misaligned target or state");
  // 32-bit places inside a tile and in a panel's grid
  if (N > (1 << 21) || V > (1 << 24) || D > (1 << 16))
    return kans_fail(KANS_ERR_UNSUPPORTED, "N=%d D=%d V=%d, at most 2^21, 2^16 and 2^24", N, D, V);
  return 0;
}

size_t workspace(int dtype, int N, int D, int V, bool backward, bool rows) {
  return dtype == DT_F16 ? xent_workspace<_Float16>(N, D, V, backward, rows)
         : dtype == DT_BF16 ? xent_workspace<__bf16>(N, D, V, backward, rows)
                            : xent_workspace<float>(N, D, V, backward, rows);
}

}  // namespace

extern "C" {

long kans_linear_xent_workspace(int dtype, int N, int D, int V, int backward) {
  const int rc = check_xent(dtype, (void*)8, (void*)8, (void*)8, N, D, V, 0, (void*)8);
  if (rc || N == 0) return rc;
  return (long)workspace(dtype, N, D, V, backward != 0, backward != 2);
}

int kans_linear_xent_forward(int dtype, const void* H, const void* W, const int64_t* target, int N, int D, int V,
                             int64_t ignore_index, int reduction, float* loss, int* state, void* workspace_p,
                             long workspace_bytes, void* stream) {
  int rc = check_xent(dtype, H, W, target, N, D, V, reduction, state);
  if (rc) return rc;
  if (N == 0) return 0;
  if (!loss) return kans_fail(KANS_ERR_ARG, "null loss");
  const size_t need = workspace(dtype, N, D, V, false, false);
  if (!workspace_p || ((uintptr_t)workspace_p & 15) || workspace_bytes < (long)need)
    return kans_fail(KANS_ERR_ARG, "workspace of %ld bytes (16-byte aligned), %zu needed", workspace_p ? workspace_bytes : 0, need);
  std::lock_guard<std::mutex> lk(kans_mutex());
  if ((rc = kans_ensure_init())) return rc;
  XentCall c{};
  c.H = H; c.W = W; c.target = target; c.N = N; c.D = D; c.V = V; c.ignore = ignore_index; c.reduction = reduction;
  c.loss = loss; c.state = state; c.ws = (char*)workspace_p;
  auto* go = dtype == DT_F16 ? xent_forward<_Float16> : dtype == DT_BF16 ? xent_forward<__bf16> : xent_forward<float>;
  HIP_TRY(go(c, kans_caller_stream(stream)));
  return 0;
}

int kans_linear_xent_backward(int dtype, const void* H, const void* W, const int64_t* target, int N, int D, int V,
                              int64_t ignore_index, int reduction, const int* state, const float* grad, void* dH, void* dW,
                              void* workspace_p, long workspace_bytes, void* stream) {
  int rc = check_xent(dtype, H, W, target, N, D, V, reduction, state);
  if (rc) return rc;
  if (N == 0 || (!dH && !dW)) return 0;
  if (!grad) return kans_fail(KANS_ERR_ARG, "null gradient");
  const size_t need = workspace(dtype, N, D, V, true, reduction == 0);
  if (!workspace_p || ((uintptr_t)workspace_p & 15) || workspace_bytes < (long)need)
    return kans_fail(KANS_ERR_ARG, "workspace of %ld bytes (16-byte aligned), %zu needed", workspace_p ? workspace_bytes : 0, need);
  std::lock_guard<std::mutex> lk(kans_mutex());
  if ((rc = kans_ensure_init())) return rc;
  XentCall c{};
  c.H = H; c.W = W; c.target = target; c.N = N; c.D = D; c.V = V; c.ignore = ignore_index; c.reduction = reduction;
  c.state = const_cast<int*>(state); c.grad = grad; c.dH = dH; c.dW = dW; c.ws = (char*)workspace_p;
  auto* go = dtype == DT_F16 ? xent_backward<_Float16> : dtype == DT_BF16 ? xent_backward<__bf16> : xent_backward<float>;
  HIP_TRY(go(c, kans_caller_stream(stream)));
  return 0;
}

}  // extern "C"
