// Kernels and launches of the cross entropy for one element type TO (see kans_xent.h).
//
// The logits are computed twice: for the sums of the softmax, and again in the backward, a piece of the vocabulary
// at a time, where the epilogue turns them into G.  Only G of one piece is ever in memory (16-bit, or three
// bf16 terms for fp32; at most kXentPiece elements) and goes into the two products behind it.  H, G and a head whose
// rows are not whole steps lie in panels that serve the products along either of their dimensions; another head is
// read as it is.
// 8 N D V operations in all against the 6 N D V of a program that keeps the logits: the price of
// not writing and reading N V of them.
//
// G is stored as (p - [v = t]) rho_n up_of<T>() with |rho_n| <= 1 (the row's share of the largest |c_n|; 1 where
// all rows have the same); the factor common to all rows comes in at the end, in fp32.  So fp16's smallest
// number stands for p rho = 2^-38, and p below fp32's normal numbers stays a normal one (the matrix pipe may drop
// others).  Where an fp16 call's rows differ by more than kXentAlike, dH takes a G without rho_n, which comes in at its end, so
// that a row's small probabilities do not depend on the other rows; dW adds the rows up, at the scale of the largest.
// Rounding G to the inputs' type is an error of half a step of that type in each
// term of a sum whose result is rounded to that type too.  (A gradient of hidden or weight whose sum over G / c_n exceeds 2^96,
// fp16 2^114, leaves fp32's range on the way.)
#pragma once
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kans_xent.h"
#include "kans_xent_gemm.h"

namespace kans {
namespace {

constexpr long kXentPiece = 1L << 28;  // elements of G in memory at a time (2^27: 10 % slower at 3001 x 777 x 50021, 1 % at 8192 x 4096 x 65536)
constexpr long kXentHeadPiece = 1L << 28;  // elements of the head that are laid out anew at a time
constexpr int kPad = 256;              // compact rows and vocabulary of a piece are padded to this
constexpr float kNoLogit = -__builtin_inff();
template <typename TO> constexpr bool kOwnG = std::is_same_v<TO, _Float16>;  // types whose rows may need a G of their own
constexpr float kXentAlike = 64.0f;    // rows whose gradients differ by less share one G: six of fp16's 38 bits below 1

template <typename TO> struct XentTypes { typedef TO T; static constexpr int TERMS = 1; };
template <> struct XentTypes<float> { typedef __bf16 T; static constexpr int TERMS = 3; };

template <typename T> constexpr int kLogUpOf = std::is_same_v<T, _Float16> ? 14 : 32;
template <typename T> __host__ __device__ constexpr float up_of() { return std::is_same_v<T, _Float16> ? 0x1p14f : 0x1p32f; }
// A product's sum times the factor common to all rows, without the power of two of G: by itself, since a small factor times
// 1 / up_of would be no normal number any more where the result still is one.
template <typename T>
__device__ __forceinline__ float unscaled(float sum, float alpha) { return __builtin_amdgcn_ldexpf(sum * alpha, -kLogUpOf<T>); }

// (XE_GRAD_OWN: XE_GRAD of a call that may need two of G, a kernel of its own so that the others' stays as short as it is)
enum XentEpilogue { XE_STATS, XE_GRAD, XE_GRAD_OWN, XE_DW, XE_DW_SPLIT, XE_DH };

struct XentArgs {
  GemmOperand A, B;
  int m_tiles, n_tiles;
  int raw;                     // (host) narrow tiles of fp32: A is raw rows
  int steps;                   // of k; products over the rows: bounded by the compact rows as well
  int splits, most_splits;     // of k, as the grid has them; most that XE_DH makes of it
  const int* state;
  int N, V;                    // rows of the call; vocabulary (XE_STATS, XE_GRAD: entries of this piece)
  int v0;                      // first entry of the piece
  float2* part;                // XE_STATS: [m tile][Np] largest logit and sum of exp
  float* picked;               // XE_STATS: [N] the target's logit
  long Np, Vp;
  const int64_t* target;       // XE_GRAD: of the call's rows
  const float* rho;            // XE_GRAD: per compact row, or null (1)
  char* g;                     // XE_GRAD: panels [v / kStep][Np][kStep]
  char* g_own;                 // the same without rho, for dH (fp16; null: one G); made and read where alpha[1] is not 0
  const float* alpha;          // factor of all of G; whether the rows' own factors come in behind dH
  void* out;                   // XE_DW: dW of the piece [V][D]
  int D;
  float* acc;                  // XE_DH: [split][rows of its tiles][Dq] fp32; XE_DW_SPLIT: [split][Vp][Dq]
  long Dq;
  int add;                     // XE_DH: add to acc
};

// exp(x): exp2 of the rounded product, and (kExact) what the rounding left as a factor.
constexpr float kLog2eRest = 1.925963033500e-8f;  // log2(e) - kLog2e
template <bool kExact>
__device__ __forceinline__ float exp_of(float x) {
  const float h = x * kLog2e;
  const float e = __builtin_amdgcn_exp2f(h);
  if (!kExact) return e;
  const float l = __builtin_fmaf(x, kLog2eRest, __builtin_fmaf(x, kLog2e, -h));
  return h > -126.0f ? __builtin_fmaf(e, l * 0.6931471805599453f, e) : e;
}

// 2^log_up exp(x - top - rest), for x - top - rest <= 0 or so, as a function of x and a factor `by` of all of them.  The
// row's largest logit and the logarithm of its sum come apart: their sum would be rounded at the logits' size, and a
// row's probabilities with it.  The power of two goes into the exponent, so that results below 2^-126, which exp2 drops,
// are there.  16-bit G, |top| < 2^8: one fma and exp2 a logit, rounded at an exponent below 64: 2^-19 of the result, far below
// the 2^-9 and 2^-12 of G; what is constant in the exponent is rounded once a row and the rest of it is `by`.
// kExact: the differences in fp32, and what the roundings of the exponent left as a factor.
template <bool kExact>
struct ExpUp {
  float top, rest, log_up, by = 1.0f;
  __device__ __forceinline__ ExpUp(float top_, float rest_, float log_up_, bool there)
      : top(there ? top_ : __builtin_inff()), rest(rest_), log_up(log_up_) {
    if (!kExact) {
      const double all = (double)log_up_ - (double)top_ * (double)kLog2e - (double)rest_ * ((double)kLog2e + (double)kLog2eRest);
      const float at = (float)all;
      if (there) by = __builtin_amdgcn_exp2f((float)(all - (double)at));
      top = there ? at : -__builtin_inff();
    }
  }
  __device__ __forceinline__ float operator()(float x) const {
    if (!kExact) return __builtin_amdgcn_exp2f(__builtin_fmaf(x, kLog2e, top));
    x = (x - top) - rest;
    x = x < -160.0f ? -160.0f : x;  // 0 all the same (-inf would leave a NaN as its rest); a NaN stays
    const float h = __builtin_fmaf(x, kLog2e, log_up), e = __builtin_amdgcn_exp2f(h);
    const float l = __builtin_fmaf(x, kLog2eRest, __builtin_fmaf(x, kLog2e, log_up - h));
    return __builtin_fmaf(e, l * 0.6931471805599453f, e);
  }
};

// Whether some lane's `at` is too large for the short forms, which round at log2(e): below, that is 2^-16 at most in an exponent.
__device__ __forceinline__ bool far(float at) { return __builtin_amdgcn_ballot_w64(!(__builtin_fabsf(at) < 0x1p8f)) != 0; }

// 8 values as packed 16-bit pairs, or as those of their three terms.
template <typename T, int TERMS>
__device__ __forceinline__ void pack8(const float* v, uint4 (&d)[TERMS]) {
  if constexpr (TERMS == 1) {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
    __builtin_memcpy(&d[0], e, 16);
  } else {
    const Split8 s = split8_bounded(v);  // (|v| <= 2^32, or NaN)
#pragma unroll
    for (int t = 0; t < 3; ++t) d[t] = s.t[t];
  }
}

// How dH's products are shared out: a call's rows are known to the device alone, so the grid is made for all of
// them (`n_tiles` tiles of bn columns, `splits` of k), and the workgroups of tiles without a row that counts go to more splits of
// the others.
struct XentShare {
  int n_tiles, splits;
};
__device__ __forceinline__ XentShare share_of(int count, int bn, int n_tiles, int splits, int most) {
  const int there = min((count + bn - 1) / bn, n_tiles);
  return {there, min(n_tiles * splits / max(there, 1), most)};
}

// Tile of a workgroup: consecutive ones go to the 8 XCDs in turn, and each XCD gets a run of the tiles.
__device__ __forceinline__ int xcd_tile(int id, int tiles) {
  const int xcd = id & 7;
  return xcd * (tiles >> 3) + min(xcd, tiles & 7) + (id >> 3);
}

// The products.  8192 x 4096 x 65536 bf16, 256 x 256 tiles (two pieces in the backward):
//   XE_STATS 3.15 ms (1.40 PFLOP/s; a library's product of the same size 3.10), XE_GRAD 2 x 1.68, XE_DW 2 x 1.62,
//   XE_DH 2 x 1.58 ms (1.31 - 1.39).
// The matrix pipe is busy 77 - 84 % of the cycles at the 1.6 GHz that its power leaves; LDS reads meet no
// bank conflict.  4096 (3686 count) x 1024 x 32768 fp32, 256 x 128: 1.11, 1.19, 1.08 and 1.11 ms (1.25 - 1.37 PFLOP/s of bf16
// products).  Short sums leave the tiles' beginnings and ends (7 us of 27 at 13 steps of 64): 3001 (2251 count) x 777 x 50021 fp16
// 0.19, 0.22, 0.24 and 0.20 ms (0.73 - 0.92).
template <typename TO, int EPI, int BM, int BN, int WAVES_M, int WAVES_N, bool A_ONCE = false, bool A_RAW = false>
__global__ __launch_bounds__(WAVES_M* WAVES_N * 64) void k_xent_gemm(const XentArgs A) {
  typedef typename XentTypes<TO>::T T;
  constexpr int TERMS = XentTypes<TO>::TERMS;
  // a third stage of A where the tile has a CU's LDS for itself and it still fits (160 KB)
  constexpr int A_STAGES = (TERMS == 1 && BM == 256 && BN == 256) || A_RAW ? 3 : 2;
  // dW = G^T H and dH = G W run along the rows of their operands: H and G, or W
  using Tile = GemmTile<T, TERMS, BM, BN, WAVES_M, WAVES_N, A_STAGES, (EPI > XE_GRAD_OWN),
                        EPI == XE_DW || EPI == XE_DW_SPLIT, A_ONCE, A_RAW>;
  using Step = StepOf<TERMS>;
  constexpr int MB = Tile::MB, NB = Tile::NB;
  __shared__ alignas(16) char a_st0[Tile::STAGE_A], a_st1[Tile::STAGE_A], a_st2[A_STAGES == 3 ? Tile::STAGE_A : 16];
  __shared__ alignas(16) char b_st0[Tile::STAGE_B], b_st1[Tile::STAGE_B];
  const int count = A.state[0];  // compact rows
  constexpr bool kOverRows = EPI == XE_DW || EPI == XE_DW_SPLIT, kOverD = kOverRows || EPI == XE_DH;  // k; m
  int id = blockIdx.x, n_tiles = A.n_tiles, split = 0, splits = A.splits;
  if constexpr (EPI == XE_DH) {
    const XentShare share = share_of(count, BN, A.n_tiles, A.splits, A.most_splits);
    n_tiles = share.n_tiles;
    splits = share.splits;
    split = id / max(A.m_tiles * n_tiles, 1);
    id -= split * A.m_tiles * n_tiles;
    if (split >= splits) return;
  } else if constexpr (EPI == XE_DW_SPLIT) {
    split = blockIdx.y;
  } else if constexpr (!kOverRows) {
    // (G of the rows that fill up the last step of k is written too: zeros)
    n_tiles = min(n_tiles, ((EPI != XE_STATS ? (count + 63) / 64 * 64 : count) + BN - 1) / BN);
  }
  if (id >= A.m_tiles * n_tiles) return;
  int mt, nt;
  tile_of<8>(xcd_tile(id, A.m_tiles * n_tiles), A.m_tiles, n_tiles, mt, nt);
  const int m0 = mt * BM, n0 = nt * BN;
  int first = 0, steps = A.steps;
  if (kOverRows) steps = min(steps, (count + Step::kStep - 1) / Step::kStep);
  if (EPI == XE_DH || EPI == XE_DW_SPLIT) {
    const int each = (steps + splits - 1) / splits;
    first = split * each;
    steps = min(each, steps - first);
  }
  floatx16 acc[MB][NB];
  GemmOperand operand_b = A.B;
  if constexpr (EPI == XE_DH && kOwnG<TO>)
    if (A.g_own && A.alpha[1] != 0.0f) operand_b.p = A.g_own;
  Tile::run(A.A, operand_b, m0, n0, kOverD ? A.D : A.V, kOverRows ? A.V : count, first, steps, a_st0, a_st1, a_st2, b_st0, b_st1, acc);

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WAVES_N, wn = wave % WAVES_N, col = lane & 31, half = lane >> 5;
  // acc[i][j][r] is C[mrow(i, r)][ncol(j)]
  auto mrow = [&](int i, int r) { return m0 + (wm * MB + i) * 32 + 8 * (r / 4) + 4 * half + r % 4; };
  auto ncol = [&](int j) { return n0 + (wn * NB + j) * 32 + col; };

  if constexpr (EPI == XE_STATS) {
    float2* join = (float2*)a_st0;  // [WAVES_M][BN]
    const bool edge = m0 + BM > A.V;
    const int* target = A.state + kXentHead + A.N;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int n = ncol(j);
      const int t = n < count ? target[n] - A.v0 - (m0 + wm * MB * 32) : -1;  // among this wave's entries
      float top = kNoLogit, sum = 0.0f, own = 0.0f;
      if (edge) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (mrow(i, r) >= A.V) acc[i][j][r] = kNoLogit;
      }
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, acc[i][j][r]);
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float at = top == kNoLogit ? 0.0f : top;
      if (TERMS == 3 || far(at)) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) sum += exp_of<TERMS == 3>(acc[i][j][r] - at);
      } else {
        // one fma and exp2 a logit; what the rounding of at log2(e) adds to every exponent is taken out of the sum
        const float at2 = at * kLog2e;
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], kLog2e, -at2));
        sum *= __builtin_amdgcn_exp2f(-__builtin_fmaf(at, kLog2e, -at2));
      }
      sum += __shfl_xor(sum, 32, 64);
      if (t >= 0 && t < MB * 32 && ((t >> 2) & 1) == half) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (t == i * 32 + 8 * (r / 4) + 4 * half + r % 4) own = acc[i][j][r];
        A.picked[n] = own;
      }
      if (half == 0) join[wm * BN + (wn * NB + j) * 32 + col] = make_float2(top, sum);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < BN; c += Tile::THREADS) {
      float2 s = join[c];
#pragma unroll
      for (int w = 1; w < WAVES_M; ++w) {
        const float2 o = join[w * BN + c];
        const float top = fmaxf(s.x, o.x), at = top == kNoLogit ? 0.0f : top;
        s.y = s.y * exp_of<TERMS == 3>(s.x - at) + o.y * exp_of<TERMS == 3>(o.x - at);
        s.x = top;
      }
      A.part[(long)mt * A.Np + n0 + c] = s;
    }
  } else if constexpr (EPI == XE_GRAD || EPI == XE_GRAD_OWN) {
    constexpr float kUp = up_of<TO>(), kLogUp = (float)kLogUpOf<TO>;
    constexpr int K = Step::kStep;
    const int* row = A.state + kXentHead;
    const float *rest_of = (const float*)(row + A.N), *top_of = rest_of + A.N;
    if (m0 + BM > A.V) {
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (mrow(i, r) >= A.V) acc[i][j][r] = kNoLogit;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int n = ncol(j);
      const bool there = n < count;
      const float top = there ? top_of[n] : 0.0f, rest = there ? rest_of[n] : 0.0f, rho = there && A.rho ? A.rho[n] : 1.0f;
      const int64_t t64 = there ? A.target[row[n]] - A.v0 : -1;
      const int t = t64 >= 0 && t64 < A.V ? (int)t64 : -1;
      if (__builtin_amdgcn_ballot_w64(!there)) {
        // G is 0 in the rows that fill up the last step; an infinite entry's logit with their zeros would be NaN
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][j][r] = there ? acc[i][j][r] : 0.0f;
      }
      // p - 1 of the target: what a confident row has left lies far below p's rounding
      float of_target = 0.0f;
      const int at = t - (m0 + wm * MB * 32);  // among this wave's entries
      if (__builtin_amdgcn_ballot_w64((unsigned)at < (unsigned)(MB * 32))) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            of_target = at == i * 32 + 8 * (r / 4) + 4 * half + r % 4 ? acc[i][j][r] : of_target;
        of_target = expm1f((of_target - top) - rest);
      }
      auto write = [&](const auto& exp_up, auto both) {  // both: G with and without rho
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int q = 0; q < 4; q += 2) {
            const int m = mrow(i, 4 * q);  // values 0 .. 3 are its rows, 4 .. 7 those 8 further on
            float e_up[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) e_up[e] = exp_up(acc[i][j][4 * q + e]);
            const int own = t - m;
            const bool targets = __builtin_amdgcn_ballot_w64((unsigned)own < 12u && !(own & 4)) != 0;
            // the two halves of the wave hold rows 0 .. 3 and 4 .. 7 of each 8: the lower takes the first 8, the upper the others
            const int m8 = m - 4 * half + 8 * half;
            const long o = ((long)(m8 / K) * A.Np + n) * Step::row_bytes + m8 % K * 2;
            auto put = [&](char* g, float factor) {
              const float times = exp_up.by * factor;
              float v[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = e_up[e] * times;
              if (targets) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = own == e % 4 + e / 4 * 8 ? of_target * (kUp * factor) : v[e];
              }
              uint4 d[TERMS];
              pack8<T, TERMS>(v, d);
#pragma unroll
              for (int c = 0; c < TERMS; ++c) {
                const auto x = __builtin_amdgcn_permlane32_swap(d[c].x, d[c].z, false, false);
                const auto y = __builtin_amdgcn_permlane32_swap(d[c].y, d[c].w, false, false);
                *(uint4*)(g + o + c * K * 2) = make_uint4(x[0], y[0], x[1], y[1]);
              }
            };
            if constexpr (decltype(both)::value) put(A.g_own, 1.0f);
            put(A.g, rho);
          }
      };
      auto with = [&](auto both) {
        if (TERMS == 3 || far(top)) write(ExpUp<true>(top, rest, kLogUp, there), both);
        else write(ExpUp<false>(top, rest, kLogUp, there), both);
      };
      if (EPI == XE_GRAD_OWN && A.alpha[1] != 0.0f) with(std::bool_constant<EPI == XE_GRAD_OWN>{});
      else with(std::false_type{});
    }
  } else if constexpr (EPI == XE_DW) {
    const float alpha = *A.alpha;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int v = ncol(j);
      if (v >= A.V) continue;
      TO* o = (TO*)A.out + (long)v * A.D;
      if constexpr (sizeof(TO) == 2) {
        // 8 elements a lane, the halves of the wave exchanged as for G: stores of 8 bytes took twice the instructions
        // (2251 x 768 x 50021 fp16: dW 204 us, so 191)
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int q = 0; q < 4; q += 2) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = unscaled<TO>(acc[i][j][4 * q + e], alpha);
            uint4 d[1];
            pack8<TO, 1>(x, d);
            const auto lo = __builtin_amdgcn_permlane32_swap(d[0].x, d[0].z, false, false);
            const auto hi = __builtin_amdgcn_permlane32_swap(d[0].y, d[0].w, false, false);
            const uint4 u = make_uint4(lo[0], hi[0], lo[1], hi[1]);
            const int at = mrow(i, 4 * q) + 4 * half;
            if (at + 8 <= A.D) {
              __builtin_memcpy(o + at, &u, sizeof(u));
            } else {
              TO e8[8];
              __builtin_memcpy(e8, &u, sizeof(u));
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (at + e < A.D) o[at + e] = e8[e];
            }
          }
      } else {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int d = mrow(i, 4 * q);
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = unscaled<TO>(acc[i][j][4 * q + e], alpha);
            if (d + 4 <= A.D) {
              __builtin_memcpy(o + d, x, sizeof(x));
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (d + e < A.D) o[d + e] = x[e];
            }
          }
      }
    }
  } else {
    float* base = A.acc + (long)split * (EPI == XE_DH ? n_tiles * BN : A.Vp) * A.Dq;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      float* o = base + (long)ncol(j) * A.Dq;
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int d = mrow(i, 4 * q);
          if (d >= A.Dq) continue;
          float4 x = make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
          if (A.add) {
            const float4 y = *(const float4*)(o + d);
            x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
          }
          *(float4*)(o + d) = x;
        }
    }
  }
}

// ---- operands ---------------------------------------------------------------------------------------
// 8 elements of a row of D from element `at`, 0 behind its end.
template <typename TO>
__device__ __forceinline__ void row8(const TO* p, int at, int D, float* v) {
  if (at + 8 <= D) {
    TO e[8];
    __builtin_memcpy(e, p + at, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = at + i < D ? to_f32(p[at + i]) : 0.0f;
  }
}
template <typename T, int TERMS>
__device__ __forceinline__ void store8(char* p, int term, const float* v) {
  if constexpr (TERMS == 1) {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
    uint4 u;
    __builtin_memcpy(&u, e, 16);
    *(uint4*)p = u;
  } else {
    const Split8 s = split8(v);
#pragma unroll
    for (int t = 0; t < 3; ++t) *(uint4*)(p + t * term) = s.t[t];
  }
}

// A matrix [.][D] laid out for the products: panels [step of D][R][kStep] of its rows.  `padded` rows (a multiple
// of 64) are written, zeros behind the last.  With `state` the rows are the compact ones (`rows` bounds their number)
// and rows behind the last kPad that hold one stay as they are; with `numbered` too, but each workgroup numbers them for
// itself.
struct XentLayout {
  const void* src;
  const int* state;
  int numbered;
  int rows, padded, D, steps, R;
  char* dst;
  int blocks;  // of 64 rows x 64 elements
};

// What the products need before they start, in one launch: block 0 numbers the rows, the next one makes the
// common factor of G, the others lay out H and a piece of W.  H's compact rows wait for their numbers: more than
// kSelfNumbered rows of a forward are laid out by a launch of their own.
constexpr int kSelfNumbered = 1024;  // rows that a workgroup numbers in one go
struct XentBegin {
  XentLayout m[2];
  int number_rows, make_scale;
  const int64_t* target;
  int N, V;
  int64_t ignore;
  int* state;
  float *picked, *loss;        // cleared with the numbering: what the products may not write
  const float* grad;
  int reduction;
  float *alpha, *rho;
};

// Numbers the rows that count, in their order, four to a thread: per row its target and whether it counts, and its number;
// how many there are.
template <typename F>
__device__ __forceinline__ int number_rows(const XentBegin& A, int* waves, const F& each) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int base = 0;
  for (int r0 = 0; r0 < A.N; r0 += kSelfNumbered) {
    const int r = r0 + threadIdx.x * 4;
    int64_t t[4];
    bool in[4];
    int at = 0, all = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t[e] = r + e < A.N ? A.target[r + e] : A.ignore;
      in[e] = t[e] != A.ignore;
      const unsigned long long mask = __builtin_amdgcn_ballot_w64(in[e]);
      at += __builtin_popcountll(mask & ((1ull << lane) - 1));
      all += __builtin_popcountll(mask);
    }
    if (lane == 0) waves[wave] = all;
    __syncthreads();
    at += base;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      at += w < wave ? waves[w] : 0;
      base += waves[w];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (r + e < A.N) each(r + e, t[e], in[e], at);
      at += in[e];
    }
    __syncthreads();
  }
  return base;
}
__device__ __forceinline__ void keep_numbers(const XentBegin& A, int* waves) {
  const int count = number_rows(A, waves, [&](int r, int64_t t, bool in, int at) {
    if (in) {
      A.state[kXentHead + at] = r;
      A.state[kXentHead + A.N + at] = t >= 0 && t < A.V ? (int)t : -1;
    }
    A.picked[r] = __builtin_nanf("");  // of a target outside the vocabulary
    A.loss[r] = 0.0f;                  // of an ignored row
  });
  if (threadIdx.x == 0) A.state[0] = count;
}

template <typename TO>
__device__ __forceinline__ void lay_out(const XentBegin& A, const XentLayout& L, int block, int* waves, int* row_of) {
  typedef typename XentTypes<TO>::T T;
  constexpr int TERMS = XentTypes<TO>::TERMS, K = StepOf<TERMS>::kStep;
  const int across = (L.D + 63) / 64, r0 = block / across * 64, d0 = block % across * 64;
  int rows = L.rows;
  if (L.numbered) {
    rows = number_rows(A, waves, [&](int r, int64_t, bool in, int at) {
      if (in && at >= r0 && at < r0 + 64) row_of[at - r0] = r;
    });
  } else if (L.state) {
    rows = min(rows, L.state[0]);
  }
  if ((L.numbered || L.state) && r0 >= (rows + kPad - 1) / kPad * kPad) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = r0 + threadIdx.x / 8 + i * 32, c = d0 + threadIdx.x % 8 * 8, step = c / K;
    if (step >= L.steps) return;
    float v[8];
    if (r < rows) {
      const int from = L.numbered ? row_of[r - r0] : L.state ? L.state[kXentHead + r] : r;
      row8((const TO*)L.src + (long)from * L.D, c, L.D, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    }
    store8<T, TERMS>(L.dst + ((long)step * L.R + r) * StepOf<TERMS>::row_bytes + c % K * 2, K * 2, v);
  }
}

// The factor common to all rows of G and each row's share of it.
__device__ __forceinline__ void make_scale(const XentBegin& A, float* join) {
  const int count = A.state[0];
  if (A.reduction != 0) {
    if (threadIdx.x == 0) {
      A.alpha[0] = count == 0 ? 0.0f : A.reduction == 1 ? *A.grad / (float)count : *A.grad;
      A.alpha[1] = 0.0f;
    }
    return;
  }
  // (of the finite gradients: an infinite one or a NaN is its row's own, and the others' G stays in its range)
  float top = 0.0f, least = __builtin_inff();
  for (int n = threadIdx.x; n < count; n += 256) {
    const float g = __builtin_fabsf(A.grad[A.state[kXentHead + n]]);
    top = fmaxf(top, g < __builtin_inff() ? g : 0.0f);
    least = g > 0.0f ? fminf(least, g) : least;
  }
  join[threadIdx.x] = top;
  join[256 + threadIdx.x] = least;
  __syncthreads();
  for (int d = 128; d > 0; d >>= 1) {
    if ((int)threadIdx.x < d) {
      join[threadIdx.x] = fmaxf(join[threadIdx.x], join[threadIdx.x + d]);
      join[256 + threadIdx.x] = fminf(join[256 + threadIdx.x], join[256 + threadIdx.x + d]);
    }
    __syncthreads();
  }
  const float by = join[0] > 0.0f ? join[0] : 1.0f;
  if (threadIdx.x == 0) {
    A.alpha[0] = by;
    A.alpha[1] = join[256] * kXentAlike < by ? 1.0f : 0.0f;
  }
  for (int n = threadIdx.x; n < count; n += 256) A.rho[n] = A.grad[A.state[kXentHead + n]] / by;
}

template <typename TO>
__global__ __launch_bounds__(256) void k_xent_begin(const XentBegin A) {
  __shared__ float join[512];
  int block = blockIdx.x;
  if (A.number_rows && block-- == 0) return keep_numbers(A, (int*)join);
  if (A.make_scale && block-- == 0) return make_scale(A, join);
  const bool second = block >= A.m[0].blocks;
  lay_out<TO>(A, A.m[second], second ? block - A.m[0].blocks : block, (int*)join, (int*)join + 64);
}

// ---- the ends ------------------------------------------------------------------------------------------
// Joins the tiles' sums: 64 rows at a time, 16 runs of tiles.  With `out` (one workgroup): the sum of the rows'
// losses, or their mean over the rows that count.
__device__ __forceinline__ void sum_rows(const float* rows, int N, int count, int mean, float* join, float* out) {
  float s = 0.0f;
  for (int r = threadIdx.x; r < N; r += 1024) s += rows[r];
  join[threadIdx.x] = s;
  __syncthreads();
  for (int d = 512; d > 0; d >>= 1) {
    if ((int)threadIdx.x < d) join[threadIdx.x] += join[threadIdx.x + d];
    __syncthreads();
  }
  if (threadIdx.x == 0) *out = mean ? join[0] / (float)count : join[0];
}

template <bool kExact>
__global__ __launch_bounds__(1024) void k_xent_loss(const float2* __restrict__ part, int tiles, long Np, int N, int* state,
                                                    const float* __restrict__ picked, float* loss, int mean, float* out) {
  __shared__ float2 join[16][64];
  const int lane = threadIdx.x & 63, run = threadIdx.x >> 6, count = state[0];
  for (int n0 = blockIdx.x * 64; n0 < count; n0 += gridDim.x * 64) {
    const int n = n0 + lane;
    float top = kNoLogit, sum = 0.0f;
    auto add = [&](float2 o) {
      const float both = fmaxf(top, o.x), at = both == kNoLogit ? 0.0f : both;
      sum = sum * exp_of<kExact>(top - at) + o.y * exp_of<kExact>(o.x - at);
      top = both;
    };
    // eight tiles at a time, their largest logit first: the exponentials do not wait for one another
    for (int t0 = run; t0 < tiles; t0 += 128) {
      float2 o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = t0 + 16 * i < tiles ? part[(long)(t0 + 16 * i) * Np + n] : make_float2(kNoLogit, 0.0f);
      float both = top;
#pragma unroll
      for (int i = 0; i < 8; ++i) both = fmaxf(both, o[i].x);
      const float at = both == kNoLogit ? 0.0f : both;
      sum *= exp_of<kExact>(top - at);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += o[i].y * exp_of<kExact>(o[i].x - at);
      top = both;
    }
    join[run][lane] = make_float2(top, sum);
    __syncthreads();
    if (run == 0 && n < count) {
      for (int r = 1; r < 16; ++r) add(join[r][lane]);
      if (state[kXentHead + N + n] < 0) top = __builtin_nanf("");
      // (not the difference to top + log: a logit's rounding is no part of a loss)
      const float rest = __builtin_logf(sum);
      ((float*)state)[kXentHead + N + n] = rest;
      ((float*)state)[kXentHead + 2 * N + n] = top;
      loss[state[kXentHead + n]] = (top - picked[n]) + rest;
    }
    __syncthreads();
  }
  if (out) sum_rows(loss, N, count, mean, (float*)join, out);
}

__global__ __launch_bounds__(1024) void k_xent_sum(const float* __restrict__ rows, int N, const int* __restrict__ state, int mean,
                                                   float* __restrict__ out) {
  __shared__ float join[1024];
  sum_rows(rows, N, state[0], mean, join, out);
}

// The splits' sums of one row times alpha, in the inputs' type.
template <typename TO>
__device__ __forceinline__ void finish_row(const float* acc, int splits, long stride, int D, float alpha, TO* o) {
  for (int d = threadIdx.x * 4; d < D; d += 1024) {
    float4 s = *(const float4*)(acc + d);
    for (int k = 1; k < splits; ++k) {
      const float4 x = *(const float4*)(acc + k * stride + d);
      s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
    }
    const float v[4] = {unscaled<TO>(s.x, alpha), unscaled<TO>(s.y, alpha), unscaled<TO>(s.z, alpha), unscaled<TO>(s.w, alpha)};
    TO e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = from_f32<TO>(v[i]);
    if (d + 4 <= D) {
      __builtin_memcpy(o + d, e, sizeof(e));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (d + i < D) o[d + i] = e[i];
    }
  }
}

// dH: compact rows into their own places, zeros for the ignored rows.
template <typename TO>
__global__ __launch_bounds__(256) void k_xent_dh(const float* __restrict__ acc, int bn, int n_tiles, int splits, int most, long Dq, int D,
                                                 const int* __restrict__ state, const int64_t* __restrict__ target,
                                                 int64_t ignore, const float* __restrict__ alpha, const float* __restrict__ own,
                                                 TO* __restrict__ dH) {
  const int row = blockIdx.x;
  if (target[row] == ignore)
    for (int d = threadIdx.x; d < D; d += 256) dH[(long)row * D + d] = (TO)0.0f;
  const int count = state[0];
  if (row >= count) return;
  const XentShare share = share_of(count, bn, n_tiles, splits, most);
  const float factor = own && alpha[1] != 0.0f ? alpha[0] * own[row] : alpha[0];  // (own: the rows' factors, if G lacks them)
  finish_row(acc + row * Dq, share.splits, (long)share.n_tiles * bn * Dq, D, factor, dH + (long)state[kXentHead + row] * D);
}

template <typename TO>
__global__ __launch_bounds__(256) void k_xent_dw(const float* __restrict__ acc, int splits, long Vp, long Dq, int D,
                                                 const float* __restrict__ alpha, TO* __restrict__ dW) {
  finish_row(acc + (long)blockIdx.x * Dq, splits, Vp * Dq, D, *alpha, dW + (long)blockIdx.x * D);
}

// ---- plans ----------------------------------------------------------------------------------------------
inline long up_to(long v, long m) { return (v + m - 1) / m * m; }

// Tiles of a product: the large one, the small one (128 x 128) or the tiny one (64 x 64); few rows get a narrow one.
enum { TILE_LARGE, TILE_SMALL, TILE_TINY, TILE_NARROW };
template <typename TO> struct Tiles;
// per_cu, cost: small and tiny tiles that a CU holds at a time, and the time of a step of that many, in steps of a
// large tile.  Measured: 16-bit tiles of 128 x 128, two a CU, reach 3/4 of the rate of one of 256 x 256; fp32 (98 KB of
// LDS, one a CU) 2/3 of that of 256 x 128.  Tiny tiles read LDS twice as often a product, at about half the rate.
// Narrow tiles have 128 entries of the head, so that a CU holds two or three: with 256, 16 x 4096 x 32000 bf16 took 73 us
// instead of 49 (125 tiles for 256 CUs), 24 x 800 x 77870 fp32 89 instead of 69.
template <> struct Tiles<float> {
  static constexpr int large_m = 256, large_n = 128, narrow_m = 128, narrow_n = 64;
  static constexpr int per_cu[3] = {1, 1, 3};
  static constexpr double cost[3] = {1.0, 0.7, 0.6};
};
template <> struct Tiles<_Float16> {
  static constexpr int large_m = 256, large_n = 256, narrow_m = 128, narrow_n = 32;
  static constexpr int per_cu[3] = {1, 2, 5};
  static constexpr double cost[3] = {1.0, 0.65, 0.7};
};
template <> struct Tiles<__bf16> : Tiles<_Float16> {};

template <typename TO>
constexpr int tile_rows(int tile) {
  return tile == TILE_SMALL ? 128 : tile == TILE_TINY ? 64 : tile == TILE_NARROW ? Tiles<TO>::narrow_m : 256;
}
template <typename TO>
constexpr int tile_columns(int tile) {
  return tile == TILE_LARGE ? Tiles<TO>::large_n : tile == TILE_NARROW ? Tiles<TO>::narrow_n : tile_rows<TO>(tile);
}

struct SplitTile {
  int tile, splits;
};
// The tile, and the splits of the `steps` steps of k (up to max_splits, none below 4 steps), that take the
// least time by this estimate: rounds of workgroups over the 256 CUs times the steps of one, and about 6 steps' time for
// the beginning and the end of each (a split's sums are written and read again: as long once more).
template <typename TO>
SplitTile split_tile(long m, long n, long steps, int max_splits) {
  SplitTile best{TILE_LARGE, 1};
  double least = 1e300;
  for (int tile : {TILE_LARGE, TILE_SMALL, TILE_TINY}) {
    const long bm = tile_rows<TO>(tile), bn = tile_columns<TO>(tile);
    const long tiles = (m + bm - 1) / bm * ((n + bn - 1) / bn), slots = 256 * Tiles<TO>::per_cu[tile];
    for (int s = 1; s <= max_splits && (s == 1 || steps / s >= 4); ++s) {
      // (the tiles of a CU share it: a round that leaves each with one of several takes that share of the time)
      const double full = (double)(tiles * s) / (double)slots, fit = Tiles<TO>::per_cu[tile];
      const double rounds = full > 1.0 ? std::ceil(full) : std::ceil(full * fit) / fit;
      const double time = rounds * Tiles<TO>::cost[tile] * (double)((steps + s - 1) / s + (s > 1 ? 12 : 6));
      if (time < least) {
        least = time;
        best = {tile, s};
      }
    }
  }
  return best;
}
template <typename TO>
int tile_for(long m, long n, long steps) {
  return n <= Tiles<TO>::narrow_n ? (int)TILE_NARROW : split_tile<TO>(m, n, steps, 1).tile;
}

template <typename TO>
struct XentPlan {
  static constexpr int TERMS = XentTypes<TO>::TERMS, K = StepOf<TERMS>::kStep;
  static constexpr long ROW = StepOf<TERMS>::row_bytes;
  long Np, Dk, Dq;         // padded rows; D in whole steps, in fp32 quads
  int d_steps;
  bool pack_w;             // W goes through panels
  long piece, pieces;      // vocabulary of a piece (a multiple of kPad) and how many
  int stats_tile;
  SplitTile dh, dw;        // dw in splits only where the vocabulary is one piece
  int dh_most;             // splits of dh where rows are ignored (share_of)
  // offsets into the workspace
  bool own;                // a second G of the rows' own scale
  size_t h, w, part, picked, rows, g, g_own, acc, acc_w, alpha, rho, bytes;
};

template <typename TO>
XentPlan<TO> plan_xent(int N, int D, int V, const void* W, bool backward, bool own) {
  XentPlan<TO> p{};
  typedef XentPlan<TO> P;
  p.Np = up_to(N, kPad);
  p.Dk = up_to(D, P::K);
  p.d_steps = (int)(p.Dk / P::K);
  p.Dq = up_to(D, 4);
  // rows of whole steps of 16-byte chunks are read as they are; fp32 ones by the forward of few rows, which is bound by
  // reading them (24 x 800 x 77870, 249 MB: 69 us, with panels 191)
  p.pack_w = (P::TERMS == 3 && (backward || N > Tiles<TO>::narrow_n)) || D % P::K != 0 || ((uintptr_t)W & 15) != 0;
  const long all = up_to(V, kPad);
  p.own = own && kOwnG<TO> && backward;
  p.piece = std::max<long>(kPad, std::min({all, kXentPiece / p.Np / kPad * kPad, kXentHeadPiece / p.Dk / kPad * kPad}));
  // (in one piece where nothing of it is laid out; a grid holds fewer than 2^32 threads, 2^-7 of the logits)
  if (!backward && !p.pack_w) p.piece = std::max<long>(kPad, std::min(all, (1L << 37) / p.Np / kPad * kPad));
  p.pieces = (V + p.piece - 1) / p.piece;
  p.piece = up_to((V + p.pieces - 1) / p.pieces, kPad);
  p.stats_tile = tile_for<TO>(std::min<long>(V, p.piece), N, p.d_steps);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  };
  p.h = take((size_t)p.d_steps * p.Np * P::ROW);
  p.w = p.pack_w ? take((size_t)p.d_steps * p.piece * P::ROW) : 0;
  if (!backward) {
    const int bm = tile_rows<TO>(p.stats_tile);
    p.part = take((size_t)((V + bm - 1) / bm + p.pieces) * p.Np * sizeof(float2));
    p.picked = take((size_t)N * 4);
    p.rows = take((size_t)N * 4);
  } else {
    p.dh = split_tile<TO>(D, N, std::min<long>(V, p.piece) / P::K, 32);
    p.dh_most = std::max<int>(p.dh.splits, (int)(std::min<long>(V, p.piece) / P::K / 8));
    p.dw = split_tile<TO>(D, std::min<long>(V, p.piece), p.Np / P::K, p.pieces > 1 ? 1 : 32);
    p.g = take((size_t)p.piece / P::K * p.Np * P::ROW);
    p.g_own = p.own ? take((size_t)p.piece / P::K * p.Np * P::ROW) : 0;
    p.acc = take((size_t)p.dh.splits * p.Np * p.Dq * 4);
    p.acc_w = p.dw.splits > 1 ? take((size_t)p.dw.splits * p.piece * p.Dq * 4) : 0;
    p.alpha = take(8);
    p.rho = take((size_t)N * 4);
  }
  p.bytes = at;
  return p;
}

template <typename TO, int EPI>
hipError_t launch_gemm(XentArgs A, long m, long n, int tile, int splits, hipStream_t st) {
  auto go = [&](auto bm, auto bn, auto wm, auto wn, auto once, auto raw) {
    constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
    A.m_tiles = (int)((m + BM - 1) / BM);
    A.n_tiles = (int)((n + BN - 1) / BN);
    A.splits = splits;
    const long tiles = (long)A.m_tiles * A.n_tiles;
    hipLaunchKernelGGL((k_xent_gemm<TO, EPI, BM, BN, WM, WN, decltype(once)::value, decltype(raw)::value>),
                       EPI == XE_DH ? dim3((unsigned)(tiles * splits)) : dim3((unsigned)tiles, splits),
                       dim3(WM * WN * 64), 0, st, A);
    return hipGetLastError();
  };
  using std::integral_constant;
  typedef integral_constant<int, 1> c1;
  typedef integral_constant<int, 2> c2;
  typedef integral_constant<int, 4> c4;
  typedef integral_constant<int, 128> c128;
  typedef integral_constant<int, 256> c256;
  constexpr std::false_type no{};
  if constexpr (EPI <= XE_GRAD_OWN)
    if (tile == TILE_NARROW) {
      // One tile of rows reads the head's entries once.  The forward does so nontemporal where the caches (256 MB) will not hold
      // the most of the head until its next pass: 16 x 4096 x 131072 bf16 (1.1 GB) 193.8 -> 175.1 us, a step of 20 rows (820 MB)
      // 1052 -> 1013, (410 MB) 533 -> 528; 30 x 1024 x 130000 (266 MB) 333, and 344 so.  (The backward's products read it twice more:
      // nontemporal there too 1025 and 544.)
      constexpr integral_constant<int, Tiles<TO>::narrow_m> tall{};
      constexpr integral_constant<int, Tiles<TO>::narrow_n> narrow{};
      constexpr std::true_type yes{};
      if constexpr (EPI == XE_STATS) {
        const bool once = (double)m * A.steps * (A.raw ? 128 : StepOf<XentTypes<TO>::TERMS>::row_bytes) > 350e6;
        if constexpr (XentTypes<TO>::TERMS == 3)
          if (A.raw) return once ? go(tall, narrow, c4{}, c1{}, yes, yes) : go(tall, narrow, c4{}, c1{}, no, yes);
        if (once) return go(tall, narrow, c4{}, c1{}, yes, no);
      }
      return go(tall, narrow, c4{}, c1{}, no, no);
    }
  if (tile == TILE_SMALL) return go(c128{}, c128{}, c2{}, c2{}, no, no);
  if (tile == TILE_TINY) return go(integral_constant<int, 64>{}, integral_constant<int, 64>{}, c2{}, c2{}, no, no);
  if constexpr (sizeof(TO) == 4) return go(c256{}, c128{}, c4{}, c2{}, no, no);
  else return go(c256{}, c256{}, c2{}, c4{}, no, no);
}

#define XENT_TRY(expr)                  \
  do {                                  \
    const hipError_t _e = (expr);       \
    if (_e != hipSuccess) return _e;    \
  } while (0)

// Layout of H's compact rows.
template <typename TO>
XentLayout hidden_layout(const XentPlan<TO>& p, const XentCall& c) {
  return {c.H, c.state, 0, c.N, (int)p.Np, c.D, p.d_steps, (int)p.Np, c.ws + p.h, (int)(p.Np / 64 * ((c.D + 63) / 64))};
}

// Layout of the entries [v0, v0 + n) of W; none where W is read as it is.
template <typename TO>
XentLayout head_layout(const XentPlan<TO>& p, const XentCall& c, long v0, int n) {
  if (!p.pack_w) return {};
  const int padded = (int)up_to(n, kPad);  // (the products read whole tiles of panels)
  return {(const TO*)c.W + v0 * c.D, nullptr, 0, n, padded, c.D, p.d_steps, (int)p.piece, c.ws + p.w,
          padded / 64 * ((c.D + 63) / 64)};
}

// H's compact rows, G's and entries of W as operands: row after row, or column after column.
template <typename TO>
GemmOperand panel_rows(const char* p, long R, int rows) {
  constexpr long ROW = XentPlan<TO>::ROW;
  return {p, ROW, R * ROW, rows, 0, 0};
}
template <typename TO>
GemmOperand panel_columns(const char* p, long R, int blocks) {
  constexpr long ROW = XentPlan<TO>::ROW;
  return {p, ROW, XentPlan<TO>::K * ROW, blocks, R * ROW, 0};
}
template <typename TO>
GemmOperand head_rows(const XentPlan<TO>& p, const XentCall& c, long v0, int n) {
  if (p.pack_w) return panel_rows<TO>(c.ws + p.w, p.piece, (int)up_to(n, kPad));
  return {(const TO*)c.W + v0 * c.D, (long)c.D * (long)sizeof(TO), XentPlan<TO>::K * (long)sizeof(TO), n, 0, 0};
}
template <typename TO>
GemmOperand head_columns(const XentPlan<TO>& p, const XentCall& c, long v0, int n) {
  if (p.pack_w) return panel_columns<TO>(c.ws + p.w, p.piece, p.d_steps);
  const long row = (long)c.D * (long)sizeof(TO);
  return {(const TO*)c.W + v0 * c.D, row, XentPlan<TO>::K * row, p.d_steps, XentPlan<TO>::ROW, n * row};
}

template <typename TO>
hipError_t launch_begin(const XentBegin& A, hipStream_t st) {
  const unsigned blocks = (unsigned)(A.m[0].blocks + A.m[1].blocks + (A.number_rows != 0) + (A.make_scale != 0));
  if (blocks == 0) return hipSuccess;
  hipLaunchKernelGGL((k_xent_begin<TO>), dim3(blocks), dim3(256), 0, st, A);
  return hipGetLastError();
}

}  // namespace

template <typename TO>
size_t xent_workspace(int N, int D, int V, bool backward, bool rows) {
  // (W's address decides whether it is packed, the reduction whether there may be two of G: the largest plan)
  size_t most = 0;
  for (const bool own : {false, rows})
    for (const void* W : {(const void*)nullptr, (const void*)1}) most = std::max(most, plan_xent<TO>(N, D, V, W, backward, own).bytes);
  return most;
}

template <typename TO>
hipError_t xent_forward(const XentCall& c, hipStream_t st) {
  typedef XentPlan<TO> P;
  const P p = plan_xent<TO>(c.N, c.D, c.V, c.W, false, false);
  float* rows = c.reduction ? (float*)(c.ws + p.rows) : c.loss;
  float* picked = (float*)(c.ws + p.picked);
  const int bm = tile_rows<TO>(p.stats_tile);
  long tiles = 0;
  for (long v0 = 0; v0 < c.V; v0 += p.piece) {
    const int n = (int)std::min<long>(p.piece, c.V - v0);
    XentBegin F{};
    F.m[0] = head_layout<TO>(p, c, v0, n);
    const bool numbered = c.N <= kSelfNumbered;
    if (v0 == 0) {
      F.number_rows = 1;
      if (numbered) {
        F.m[1] = hidden_layout<TO>(p, c);
        F.m[1].numbered = 1;
      }
      F.target = c.target; F.N = c.N; F.V = c.V; F.ignore = c.ignore; F.state = c.state; F.picked = picked; F.loss = rows;
    }
    XENT_TRY(launch_begin<TO>(F, st));
    if (v0 == 0 && !numbered) {
      XentBegin H{};
      H.m[0] = hidden_layout<TO>(p, c);
      XENT_TRY(launch_begin<TO>(H, st));
    }
    XentArgs A{};
    A.A = head_rows<TO>(p, c, v0, n);
    A.raw = !p.pack_w;
    A.B = panel_rows<TO>(c.ws + p.h, p.Np, (int)p.Np);
    A.steps = p.d_steps;
    A.state = c.state; A.N = c.N; A.V = n; A.v0 = (int)v0;
    A.part = (float2*)(c.ws + p.part) + tiles * p.Np;
    A.picked = picked; A.Np = p.Np;
    XENT_TRY((launch_gemm<TO, XE_STATS>(A, n, c.N, p.stats_tile, 1, st)));
    tiles += (n + bm - 1) / bm;
  }
  // few rows: their losses and the sum of them in one workgroup
  const bool once = c.reduction && c.N <= 256;
  hipLaunchKernelGGL((k_xent_loss<P::TERMS == 3>), dim3(once ? 1 : (c.N + 63) / 64), dim3(1024), 0, st,
                     (const float2*)(c.ws + p.part), (int)tiles, p.Np, c.N, c.state, picked, rows, c.reduction == 1,
                     once ? c.loss : nullptr);
  XENT_TRY(hipGetLastError());
  if (c.reduction && !once) {
    hipLaunchKernelGGL(k_xent_sum, dim3(1), dim3(1024), 0, st, rows, c.N, c.state, c.reduction == 1, c.loss);
    XENT_TRY(hipGetLastError());
  }
  return hipSuccess;
}

template <typename TO>
hipError_t xent_backward(const XentCall& c, hipStream_t st) {
  typedef XentPlan<TO> P;
  const P p = plan_xent<TO>(c.N, c.D, c.V, c.W, true, c.reduction == 0 && c.dH);
  float *alpha = (float*)(c.ws + p.alpha), *rho = (float*)(c.ws + p.rho);
  for (long v0 = 0; v0 < c.V; v0 += p.piece) {
    const int n = (int)std::min<long>(p.piece, c.V - v0);
    const int n_steps = (int)(up_to(n, P::K) / P::K);
    XentBegin F{};
    F.m[0] = head_layout<TO>(p, c, v0, n);
    if (v0 == 0) {
      F.m[1] = hidden_layout<TO>(p, c);
      F.make_scale = 1;
      F.state = c.state; F.grad = c.grad; F.reduction = c.reduction; F.alpha = alpha; F.rho = rho;
    }
    XENT_TRY(launch_begin<TO>(F, st));
    XentArgs A{};
    A.A = head_rows<TO>(p, c, v0, n);
    A.B = panel_rows<TO>(c.ws + p.h, p.Np, (int)p.Np);
    A.steps = p.d_steps;
    A.state = c.state; A.N = c.N; A.V = n; A.v0 = (int)v0; A.D = c.D;
    A.Np = p.Np; A.Vp = p.piece;
    A.target = c.target;
    A.rho = c.reduction ? nullptr : rho;
    A.g = c.ws + p.g;
    A.g_own = p.own ? c.ws + p.g_own : nullptr;
    A.alpha = alpha;
    // (every entry of the padded piece is written: tiles of 256 or 128 entries and rows)
    constexpr int kMaybeOwn = kOwnG<TO> ? XE_GRAD_OWN : XE_GRAD;
    const int tile = tile_for<TO>(n, c.N, p.d_steps);
    if (p.own) XENT_TRY((launch_gemm<TO, kMaybeOwn>(A, up_to(n, kPad), up_to(c.N, 64), tile, 1, st)));
    else XENT_TRY((launch_gemm<TO, XE_GRAD>(A, up_to(n, kPad), up_to(c.N, 64), tile, 1, st)));
    if (c.dW) {
      XentArgs B = A;
      B.A = panel_columns<TO>(c.ws + p.h, p.Np, p.d_steps);
      B.B = panel_columns<TO>(c.ws + p.g, p.Np, (int)(up_to(n, kPad) / P::K));
      B.steps = (int)(p.Np / P::K);
      B.out = (TO*)c.dW + v0 * c.D;
      if (p.dw.splits == 1) {
        XENT_TRY((launch_gemm<TO, XE_DW>(B, c.D, n, p.dw.tile, 1, st)));
      } else {
        B.acc = (float*)(c.ws + p.acc_w); B.Dq = p.Dq;
        XENT_TRY((launch_gemm<TO, XE_DW_SPLIT>(B, c.D, n, p.dw.tile, p.dw.splits, st)));
        hipLaunchKernelGGL((k_xent_dw<TO>), dim3(n), dim3(256), 0, st, B.acc, p.dw.splits, p.piece, p.Dq, c.D, alpha, (TO*)c.dW);
        XENT_TRY(hipGetLastError());
      }
    }
    if (c.dH) {
      XentArgs B = A;
      B.A = head_columns<TO>(p, c, v0, n);
      B.B = panel_rows<TO>(c.ws + p.g, p.Np, (int)p.Np);
      B.steps = n_steps;
      B.most_splits = p.dh_most;
      B.acc = (float*)(c.ws + p.acc); B.Dq = p.Dq;
      B.add = v0 > 0;
      XENT_TRY((launch_gemm<TO, XE_DH>(B, c.D, c.N, p.dh.tile, p.dh.splits, st)));
    }
  }
  if (c.dH) {
    const int dh_columns = tile_columns<TO>(p.dh.tile);
    hipLaunchKernelGGL((k_xent_dh<TO>), dim3(c.N), dim3(256), 0, st, (const float*)(c.ws + p.acc), dh_columns, (c.N + dh_columns - 1) / dh_columns,
                       p.dh.splits, p.dh_most, p.Dq, c.D, c.state, c.target, c.ignore, alpha, p.own ? rho : nullptr, (TO*)c.dH);
    XENT_TRY(hipGetLastError());
  }
  return hipSuccess;
}

}  // namespace kans
