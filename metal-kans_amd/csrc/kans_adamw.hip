// AdamW over many tensors at once (gfx950), states in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// everything in fp32, each operation rounded by itself (no contraction), so an
// elementwise fp32 restatement gives the same bits.  A 16-bit parameter has an
// fp32 master among the states and is its rounding.
//
// The states of a set of tensors lie in one buffer per kind, every tensor at a
// multiple of kAdamBlock elements.  In 8 bits the kAdamBlock consecutive elements
// of a block share one fp32 scale s per moment, the largest magnitude in it (at
// least 2^-126, so that 1 / s is finite):
//   m: code q = sign(m) rint(127 sqrt(|m| / s)), value s (q / 127) |q / 127|
//   v: code q = rint(255 (v / s)^(1/4)) and at least 1 where v > 0 (a v rounded to
//      zero would divide by eps alone), value s (q / 255)^4
// The powers spend the codes where the magnitudes lie: sqrt(v), which the step
// divides by, keeps a relative step of 2 / q.  A block that holds an infinity or a
// NaN gets the scale NaN: the failure stays visible.
#include <hip/hip_runtime.h>

#include <cmath>

#include "kans_api_internal.h"
#include "kans_wave.h"

namespace kans {
namespace {

constexpr int kAdamBlock = 256;    // elements of a block: one wave, 4 a lane
constexpr int kAdamThreads = 256;
constexpr int kAdamUnroll = 4;     // blocks of a wave
constexpr int kAdamTile = kAdamThreads * 4 * kAdamUnroll;  // elements of a workgroup
constexpr int kAdamTensors = 96;   // tensors of one launch: the table fits the 4 KB of kernel arguments
constexpr long kAdamMaxGrid = 1L << 22;

struct AdamwBatch {
  const void* g[kAdamTensors];
  void* p[kAdamTensors];
  long n[kAdamTensors];
  unsigned block[kAdamTensors];     // first block of the states
  unsigned first[kAdamTensors];     // first workgroup; unused entries 2^32 - 1
  float step_size[kAdamTensors];    // lr / (1 - b1^t)
  float root[kAdamTensors];         // 1 / sqrt(1 - b2^t)
  void *m, *v;
  float *m_scale, *v_scale, *master;
  float b1, c1, b2, c2, keep, eps;  // c = 1 - b, keep = 1 - lr wd
};
static_assert(sizeof(AdamwBatch) <= 4096, "kernel arguments");

// Four elements as they lie in memory.  Loads and stores bypass what they can of the caches: a step reads and
// writes everything once (126 M bf16 parameters: 681 us without, 614 with).
template <typename T> struct QuadOf;
template <> struct QuadOf<float> { typedef unsigned type __attribute__((ext_vector_type(4))); };
template <> struct QuadOf<_Float16> { typedef unsigned type __attribute__((ext_vector_type(2))); };
template <> struct QuadOf<__bf16> { typedef unsigned type __attribute__((ext_vector_type(2))); };

// Four consecutive elements of which `left` exist (all of them, aligned, where `vec`).
template <typename T>
__device__ __forceinline__ void load4(const T* p, long left, bool vec, float* o) {
  T e[4];
  if (vec && left >= 4) {
    const auto q = __builtin_nontemporal_load((const typename QuadOf<T>::type*)p);
    __builtin_memcpy(e, &q, sizeof(e));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = i < left ? p[i] : (T)0.0f;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = to_f32(e[i]);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, long left, bool vec, const float* o) {
  T e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(o[i]);
  if (vec && left >= 4) {
    typename QuadOf<T>::type q;
    __builtin_memcpy(&q, e, sizeof(e));
    __builtin_nontemporal_store(q, (typename QuadOf<T>::type*)p);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = e[i];
  }
}

#pragma clang fp contract(off)

__device__ __forceinline__ float avg_value(int q, float s) {
  const float t = (float)q * (float)(1.0 / 127.0);
  return s * (t * __builtin_fabsf(t));
}
__device__ __forceinline__ float sq_value(unsigned q, float s) {
  float t = (float)q * (float)(1.0 / 255.0);
  t = t * t;
  return s * (t * t);
}

// Scale of a wave's 256 magnitudes (4 a lane).
__device__ __forceinline__ float block_scale(const float* a) {
  float top = 0.0f;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    top = fmaxf(top, __builtin_fabsf(a[e]));
    bad |= !(__builtin_fabsf(a[e]) < __builtin_inff());
  }
  top = fmaxf(wave_max(top), 0x1p-126f);
  return __builtin_amdgcn_ballot_w64(bad) ? __builtin_nanf("") : top;
}

// rint(127 sqrt(a)) and rint(255 sqrt(sqrt(a))) of four magnitudes in [0, 1] or so, as if each root and product were
// rounded correctly.  The hardware's root is within an ulp, the product then within 8e-5 of the correct one: where no lane
// is that close to the middle between two codes (a wave in ten is) its rounding is the right one, at a quarter of the
// instructions.
template <int TOP>
__device__ __forceinline__ void codes_of(const float* a, float* code) {
  float edge = 1.0f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float r = __builtin_amdgcn_sqrtf(a[e]);
    if (TOP == 255) r = __builtin_amdgcn_sqrtf(r);
    r *= (float)TOP;
    code[e] = __builtin_rintf(r);
    edge = fminf(edge, 0.5f - __builtin_fabsf(r - code[e]));
  }
  if (__builtin_amdgcn_ballot_w64(!(edge > 3e-4f))) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float r = __builtin_sqrtf(a[e]);
      if (TOP == 255) r = __builtin_sqrtf(r);
      code[e] = __builtin_rintf((float)TOP * r);
    }
  }
}

// One wave takes a block of 256 elements a turn, 4 consecutive ones a lane, four turns with their loads together.  Bound
// by HBM in 32 bits (126 M bf16 parameters, 3.5 GB: 614 us, 5.7 TB/s); with 8-bit states by the roots and the quotient, all
// rounded correctly (97 M fp32 parameters, 1.56 GB: 348 us, 4.5 TB/s).
template <typename T, bool k8>
__global__ __launch_bounds__(kAdamThreads) void k_adamw(const AdamwBatch A) {
  // the tensor of this workgroup: the last whose first workgroup is not behind it
  const int lane = threadIdx.x & 63;
  int ti = __builtin_popcountll(__builtin_amdgcn_ballot_w64(A.first[lane] <= blockIdx.x));
  ti += __builtin_popcountll(
      __builtin_amdgcn_ballot_w64(lane < kAdamTensors - 64 && A.first[min(64 + lane, kAdamTensors - 1)] <= blockIdx.x));
  ti = __builtin_amdgcn_readfirstlane(ti - 1);
  const long n = A.n[ti];
  T* const p = (T*)A.p[ti];
  const T* const g = (const T*)A.g[ti];
  const bool vec = (((uintptr_t)p | (uintptr_t)g) & (4 * sizeof(T) - 1)) == 0;
  const long base = (long)(blockIdx.x - A.first[ti]) * kAdamTile + (threadIdx.x >> 6) * kAdamBlock;  // of the wave
  const long state0 = (long)A.block[ti] * kAdamBlock;
  const float step_size = A.step_size[ti], root = A.root[ti];

  float w[kAdamUnroll][4], gr[kAdamUnroll][4], m[kAdamUnroll][4], v[kAdamUnroll][4];
#pragma unroll
  for (int u = 0; u < kAdamUnroll; ++u) {
    const long at = base + u * kAdamThreads * 4 + lane * 4, left = n - at;
    load4(g + at, left, vec, gr[u]);
    if constexpr (sizeof(T) == 4) load4(p + at, left, vec, w[u]);
    else load4((const float*)A.master + state0 + at, left, true, w[u]);
    if constexpr (!k8) {
      load4((const float*)A.m + state0 + at, left, true, m[u]);
      load4((const float*)A.v + state0 + at, left, true, v[u]);
    } else if (base + u * kAdamThreads * 4 < n) {  // (codes behind the last element are part of the block: zeros)
      const unsigned mc = __builtin_nontemporal_load((const unsigned*)((const signed char*)A.m + state0 + at));
      const unsigned vc = __builtin_nontemporal_load((const unsigned*)((const unsigned char*)A.v + state0 + at));
      const float ms = A.m_scale[(state0 + at) / kAdamBlock], vs = A.v_scale[(state0 + at) / kAdamBlock];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        m[u][e] = avg_value((signed char)(mc >> (8 * e)), ms);
        v[u][e] = sq_value((vc >> (8 * e)) & 255, vs);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kAdamUnroll; ++u) {
    const long at = base + u * kAdamThreads * 4 + lane * 4, left = n - at;
    if (base + u * kAdamThreads * 4 >= n) break;  // uniform in the wave
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      m[u][e] = m[u][e] * A.b1 + gr[u][e] * A.c1;
      v[u][e] = v[u][e] * A.b2 + (gr[u][e] * gr[u][e]) * A.c2;
      w[u][e] = w[u][e] * A.keep - step_size * (m[u][e] / (__builtin_sqrtf(v[u][e]) * root + A.eps));
    }
    store4(p + at, left, vec, w[u]);
    if constexpr (sizeof(T) == 2) store4(A.master + state0 + at, left, true, w[u]);
    if constexpr (!k8) {
      store4((float*)A.m + state0 + at, left, true, m[u]);
      store4((float*)A.v + state0 + at, left, true, v[u]);
    } else {
      const float ms = block_scale(m[u]), vs = block_scale(v[u]);
      const float mi = 1.0f / ms, vi = 1.0f / vs;
      float am[4], av[4], qm[4], qv[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        am[e] = __builtin_fabsf(m[u][e]) * mi;
        av[e] = v[u][e] * vi;
      }
      codes_of<127>(am, qm);
      codes_of<255>(av, qv);
      unsigned mc = 0, vc = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // (min and max also turn the NaN of a block without a scale into a code)
        const int q = (int)__builtin_copysignf(fminf(qm[e], 127.0f), m[u][e]);
        const unsigned c = (unsigned)fmaxf(fminf(qv[e], 255.0f), v[u][e] > 0.0f ? 1.0f : 0.0f);
        mc |= (unsigned)(q & 255) << (8 * e);
        vc |= c << (8 * e);
      }
      __builtin_nontemporal_store(mc, (unsigned*)((signed char*)A.m + state0 + at));
      __builtin_nontemporal_store(vc, (unsigned*)((unsigned char*)A.v + state0 + at));
      if (lane == 0) {
        A.m_scale[(state0 + at) / kAdamBlock] = ms;
        A.v_scale[(state0 + at) / kAdamBlock] = vs;
      }
    }
  }
}

// The values of 8-bit states: a wave takes one block, 4 elements a lane (97 M of each moment, 970 MB: 170 - 190 us).
__global__ __launch_bounds__(256) void k_adamw_values(const unsigned* mc, const unsigned* vc, const float* ms,
                                                      const float* vs, float4* m, float4* v, long quads) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < quads; i += (long)gridDim.x * 256) {
    const float s = ms[i / 64], r = vs[i / 64];
    const unsigned a = mc[i], b = vc[i];
    const float mv[4] = {avg_value((signed char)a, s), avg_value((signed char)(a >> 8), s),
                         avg_value((signed char)(a >> 16), s), avg_value((signed char)(a >> 24), s)};
    const float vv[4] = {sq_value(b & 255, r), sq_value((b >> 8) & 255, r), sq_value((b >> 16) & 255, r), sq_value(b >> 24, r)};
    store4((float*)(m + i), 4, true, mv);
    store4((float*)(v + i), 4, true, vv);
  }
}

template <typename T>
hipError_t launch_adamw(const AdamwBatch& A, long wgs, bool k8, hipStream_t st) {
  if (k8) hipLaunchKernelGGL((k_adamw<T, true>), dim3(wgs), dim3(kAdamThreads), 0, st, A);
  else hipLaunchKernelGGL((k_adamw<T, false>), dim3(wgs), dim3(kAdamThreads), 0, st, A);
  return hipGetLastError();
}

bool rate(double v) { return v >= 0.0 && std::isfinite(v); }

}  // namespace
}  // namespace kans

using namespace kans;

extern "C" {

int kans_adamw_step(int dtype, int state_bits, int n_tensors, void* const* params, const void* const* grads,
                    const long* numel, const long* blocks, const long* steps, void* exp_avg, void* exp_avg_sq,
                    float* exp_avg_scale, float* exp_avg_sq_scale, float* master, double lr, double beta1, double beta2,
                    double eps, double weight_decay, void* stream) {
  if (dtype != DT_F32 && dtype != DT_F16 && dtype != DT_BF16) return kans_fail(KANS_ERR_ARG, "unknown dtype %d", dtype);
  if (state_bits != 8 && state_bits != 32) return kans_fail(KANS_ERR_ARG, "state_bits=%d, must be 8 or 32", state_bits);
  if (n_tensors < 0) return kans_fail(KANS_ERR_ARG, "n_tensors=%d", n_tensors);
  if (n_tensors == 0) return 0;
  if (!params || !grads || !numel || !blocks || !steps) return kans_fail(KANS_ERR_ARG, "null tensor table");
  if (!rate(lr) || !rate(eps) || !rate(weight_decay) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0))
    return kans_fail(KANS_ERR_ARG, "lr, eps and weight_decay must be finite and >= 0, the betas in [0, 1)");
  bool any = false;
  for (int i = 0; i < n_tensors; ++i) {
    if (numel[i] < 0 || blocks[i] < 0 || steps[i] < 1 || (numel[i] > 0 && (!params[i] || !grads[i])))
      return kans_fail(KANS_ERR_ARG, "tensor %d: null pointer, negative size or block, or step %ld < 1", i, steps[i]);
    if (numel[i] > kAdamMaxGrid * kAdamTile || blocks[i] > 0xffffffffL)
      return kans_fail(KANS_ERR_UNSUPPORTED, "tensor %d: %ld elements at block %ld exceed one launch", i, numel[i], blocks[i]);
    any |= numel[i] > 0;
  }
  if (!any) return 0;
  if (!exp_avg || !exp_avg_sq) return kans_fail(KANS_ERR_ARG, "null state");
  if (state_bits == 8 && (!exp_avg_scale || !exp_avg_sq_scale)) return kans_fail(KANS_ERR_ARG, "8-bit states need their scales");
  if (dtype != DT_F32 && !master) return kans_fail(KANS_ERR_ARG, "16-bit parameters need their fp32 masters");
  if (((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq | (uintptr_t)master) & 15)
    return kans_fail(KANS_ERR_ARG, "states must be 16-byte aligned");
  std::lock_guard<std::mutex> lk(kans_mutex());
  int rc = kans_ensure_init();
  if (rc) return rc;
  hipStream_t st = kans_caller_stream(stream);
  // a replayed step would keep the bias corrections of the step that was captured
  bool capturing = false;
  HIP_TRY(kans_capturing(st, &capturing));
  if (capturing) return kans_fail(KANS_ERR_STATE, "an AdamW step cannot be captured: its bias corrections change every step");
  AdamwBatch A;
  A.m = exp_avg; A.v = exp_avg_sq; A.m_scale = exp_avg_scale; A.v_scale = exp_avg_sq_scale; A.master = master;
  A.b1 = (float)beta1; A.c1 = (float)(1.0 - beta1);
  A.b2 = (float)beta2; A.c2 = (float)(1.0 - beta2);
  A.keep = (float)(1.0 - lr * weight_decay); A.eps = (float)eps;
  auto* launch = dtype == DT_F16 ? launch_adamw<_Float16> : dtype == DT_BF16 ? launch_adamw<__bf16> : launch_adamw<float>;
  int count = 0;
  long wgs = 0;
  auto flush = [&]() -> hipError_t {
    if (count == 0) return hipSuccess;
    for (int i = count; i < kAdamTensors; ++i) A.first[i] = 0xffffffffu;
    const hipError_t e = launch(A, wgs, state_bits == 8, st);
    count = 0;
    wgs = 0;
    return e;
  };
  for (int i = 0; i < n_tensors; ++i) {
    if (numel[i] == 0) continue;
    const long need = (numel[i] + kAdamTile - 1) / kAdamTile;
    if (count == kAdamTensors || wgs + need > kAdamMaxGrid) HIP_TRY(flush());
    A.p[count] = params[i];
    A.g[count] = grads[i];
    A.n[count] = numel[i];
    A.block[count] = (unsigned)blocks[i];
    A.first[count] = (unsigned)wgs;
    A.step_size[count] = (float)(lr / (1.0 - std::pow(beta1, (double)steps[i])));
    A.root[count] = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)steps[i])));
    wgs += need;
    ++count;
  }
  HIP_TRY(flush());
  return 0;
}

int kans_adamw_values(const void* exp_avg, const void* exp_avg_sq, const float* exp_avg_scale,
                      const float* exp_avg_sq_scale, float* avg_out, float* sq_out, long blocks, void* stream) {
  if (blocks < 0) return kans_fail(KANS_ERR_ARG, "blocks=%ld", blocks);
  if (blocks == 0) return 0;
  if (!exp_avg || !exp_avg_sq || !exp_avg_scale || !exp_avg_sq_scale || !avg_out || !sq_out)
    return kans_fail(KANS_ERR_ARG, "null argument");
  if (((uintptr_t)avg_out | (uintptr_t)sq_out) & 15 || ((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 3)
    return kans_fail(KANS_ERR_ARG, "outputs must be 16-byte aligned, codes 4-byte aligned");
  std::lock_guard<std::mutex> lk(kans_mutex());
  int rc = kans_ensure_init();
  if (rc) return rc;
  const long quads = blocks * (kAdamBlock / 4);
  hipLaunchKernelGGL(k_adamw_values, dim3((unsigned)std::min<long>((quads + 255) / 256, 16384)), dim3(256), 0,
                     kans_caller_stream(stream), (const unsigned*)exp_avg, (const unsigned*)exp_avg_sq, exp_avg_scale,
                     exp_avg_sq_scale, (float4*)avg_out, (float4*)sq_out, quads);
  HIP_TRY(hipGetLastError());
  return 0;
}

}  // extern "C"
