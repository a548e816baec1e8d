// Softmax cross entropy of a linear head without its logits (gfx950): what the host entry points (kans_xent.hip)
// and the kernels of one element type (kans_xent_kernel.h, one unit per type) share.
//
//   l[n][v] = sum_d H[n][d] W[v][d],  top[n] = max_v l[n][v],  rest[n] = log sum_v exp(l[n][v] - top[n])
//   loss[n] = (top[n] - l[n][t_n]) + rest[n],  c_n = d(result)/d(loss[n])
//   G[n][v] = c_n (exp(l[n][v] - top[n] - rest[n]) - [v = t_n]),  dH = G W,  dW = G^T H
//
// Rows whose target is the ignored one are left out of everything: the rows that count are numbered anew
// ("compact" rows, in their order) on the device, and the products run over those alone.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace kans {

// Head of the state that the forward leaves for the backward: ints [4]: number of compact rows, -, -, -;
// then per compact row its row [N], its rest (fp32; until the sums are joined its target, -1: outside the
// vocabulary) [N] and its top (fp32) [N].
constexpr int kXentHead = 4;

struct XentCall {
  const void *H, *W;
  const int64_t* target;
  int N, D, V;
  int64_t ignore;
  int reduction;           // 0 none, 1 mean, 2 sum
  float* loss;             // forward: [N] or [1]
  int* state;
  const float* grad;       // backward: [N] or [1]
  void *dH, *dW;           // backward: either may be null
  char* ws;
};

// Bytes of workspace (rows: of a call without reduction too), and the calls, of one element type (launches are enqueued on st).
template <typename TO> size_t xent_workspace(int N, int D, int V, bool backward, bool rows);
template <typename TO> hipError_t xent_forward(const XentCall& c, hipStream_t st);
template <typename TO> hipError_t xent_backward(const XentCall& c, hipStream_t st);

}  // namespace kans
