// Matrix product of the cross entropy kernels (kans_xent.hip): C[m][n] = sum_k A[m][k] B[n][k] on the 16-bit
// matrix cores, with the epilogue taking the tile from the accumulators.
//
// Operands are rows of k in steps of kStep elements: step s of row r is `row_bytes` consecutive bytes at
// base + r * row_stride + s * step_stride.  That covers a row-major matrix (step_stride = row_bytes) and panels
// [step][row][kStep], whose tile of a step is one contiguous run.  fp32 operands (TERMS = 3) are the three
// bf16 terms of kans_split.h, [row][term][32] in a step, and take six MFMAs a product.
//
// A workgroup of WAVES_M x WAVES_N waves holds a BM x BN tile.  A step's rows go from memory to LDS by DMA
// (buffer loads, 16 bytes a lane) into one of two stages; the barrier that opens stage s + 1 stands before
// the last part of step s, whose operands are in registers by then: the first operands of step s + 1 are read
// while the matrix pipe works on it.  The DMA of step s + 2 goes out in that part and the next one, one
// instruction between a few products: all of them at once fill the memory pipe's queue, and the waves stand there.  The two stages are
// separate arrays and the step loop is unrolled by two, so that the compiler sees that reads of one do not
// depend on the DMA into the other.
//
// LDS rows are 128 (or, with three terms, 192) bytes, so a column of 16-byte chunks would meet the same banks in
// every second (fourth) row: chunk c of row r lies in slot c ^ ((r >> 1) & 7) (c ^ ((r >> 2) & 3)), which
// spreads 16 rows over all 64 banks.  The DMA writes LDS in lane order, so it is the source address that is permuted,
// inside one row's step.
#pragma once
#include "kans_split.h"
#include "kans_tile.h"

namespace kans {

struct GemmOperand {
  const void* p;
  long row_stride, step_stride;  // bytes
  int rows;                      // rows that exist; those of a tile behind them repeat the last
};

template <int TERMS> struct StepOf {
  static constexpr int kStep = TERMS == 1 ? 64 : 32;              // k of a step
  static constexpr int row_bytes = kStep * 2 * TERMS;             // 128 or 192
  static constexpr int chunks = row_bytes / 16;
  static constexpr int parts = kStep / 16;                        // MFMA depths of a step
  static __device__ __forceinline__ int slot(int row, int chunk) {
    return TERMS == 1 ? chunk ^ ((row >> 1) & 7) : chunk ^ ((row >> 2) & 3);
  }
};

template <typename T, int TERMS, int BM, int BN, int WAVES_M, int WAVES_N>
struct GemmTile {
  using Step = StepOf<TERMS>;
  static constexpr int WAVES = WAVES_M * WAVES_N, THREADS = WAVES * 64;
  static constexpr int MB = BM / WAVES_M / 32, NB = BN / WAVES_N / 32;  // 32 x 32 blocks of a wave
  static constexpr int STAGE = (BM + BN) * Step::row_bytes;
  static constexpr int DMA_A = BM * Step::row_bytes / 1024 / WAVES, DMA_B = BN * Step::row_bytes / 1024 / WAVES;
  static_assert(DMA_A * 1024 * WAVES == BM * Step::row_bytes && DMA_B * 1024 * WAVES == BN * Step::row_bytes, "whole DMAs");
  typedef typename Mfma<T>::frag frag;

  // A raw buffer from p on: 32-bit offsets, not bounded (the operands' rows are: GemmOperand).
  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const char* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0, 0xffffffffu, 0x00027000);
  }

  // acc = the tile at (m0, n0) over `steps` steps from step `first`.
  static __device__ __forceinline__ void run(const GemmOperand& A, const GemmOperand& B, int m0, int n0, int first, int steps,
                                             char* st0, char* st1, floatx16 (&acc)[MB][NB]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WAVES_N, wn = wave % WAVES_N;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    if (steps <= 0) return;
    // this lane's places in the tile's rows
    unsigned off_a[DMA_A], off_b[DMA_B];
    const int a0 = min(m0, A.rows - 1), b0 = min(n0, B.rows - 1);
    auto place = [&](int q, int tile0, int row0, const GemmOperand& o) {
      const int row = q / Step::chunks, chunk = Step::slot(row, q - row * Step::chunks);
      return (unsigned)(min(tile0 + row, o.rows - 1) - row0) * (unsigned)o.row_stride + chunk * 16;
    };
#pragma unroll
    for (int i = 0; i < DMA_A; ++i) off_a[i] = place((i * WAVES + wave) * 64 + lane, m0, a0, A);
#pragma unroll
    for (int i = 0; i < DMA_B; ++i) off_b[i] = place((i * WAVES + wave) * 64 + lane, n0, b0, B);
    const char* pa = (const char*)A.p + (long)a0 * A.row_stride + (long)first * A.step_stride;
    const char* pb = (const char*)B.p + (long)b0 * B.row_stride + (long)first * B.step_stride;
    // (buffer loads, not global ones: behind a global load to LDS the compiler waits for every LDS read
    // where it could wait for the older ones)
    struct Source {
      __amdgpu_buffer_rsrc_t a, b;
    };
    auto source = [&](int s) {
      return Source{resource(pa + (long)s * A.step_stride), resource(pb + (long)s * B.step_stride)};
    };
    auto dma1 = [&](const Source& o, char* st, int i) {  // the i-th of this wave's DMAs of a step
      if (i < DMA_A)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            o.a, (__attribute__((address_space(3))) void*)(st + (i * WAVES + wave) * 1024), 16, off_a[i < DMA_A ? i : 0], 0, 0, 0);
      else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            o.b, (__attribute__((address_space(3))) void*)(st + BM * Step::row_bytes + ((i - DMA_A) * WAVES + wave) * 1024), 16,
            off_b[i < DMA_A ? 0 : i - DMA_A], 0, 0, 0);
    };
    constexpr int DMAS = DMA_A + DMA_B, EACH = (DMAS + 2 * MB - 1) / (2 * MB);  // behind each of 2 MB rows of blocks
    auto dma = [&](int s, char* st, int from, int to) {
      const Source o = source(s);
#pragma unroll
      for (int i = from; i < to; ++i) dma1(o, st, i);
    };
    const int row = lane & 31, half = lane >> 5;
    auto read = [&](const char* st, int r, int part, int term) {
      const int slot = Step::slot(r, term * (Step::kStep / 8) + part * 2 + half);
      return *(const frag*)(st + r * Step::row_bytes + slot * 16);
    };
    frag a[2][MB][TERMS], b[2][NB][TERMS];
    auto fetch = [&](const char* st, int part, frag (&fa)[MB][TERMS], frag (&fb)[NB][TERMS]) {
#pragma unroll
      for (int t = 0; t < TERMS; ++t) {
#pragma unroll
        for (int i = 0; i < MB; ++i) fa[i][t] = read(st, (wm * MB + i) * 32 + row, part, t);
#pragma unroll
        for (int j = 0; j < NB; ++j) fb[j][t] = read(st + BM * Step::row_bytes, (wn * NB + j) * 32 + row, part, t);
      }
    };
    // the products of one part; between(i) comes before those of the i-th row of blocks
    auto multiply = [&](const frag (&fa)[MB][TERMS], const frag (&fb)[NB][TERMS], auto between) {
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        between(i);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          if constexpr (TERMS == 3) acc[i][j] = mma_split(fa[i], fb[j], acc[i][j]);
          else acc[i][j] = Mfma<T>::mma(fa[i][0], fb[j][0], acc[i][j]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto dma_between = [&](bool on, int s, char* st, int from) {
      const Source o = source(s);
      return [=](int i) {
        if (!on) return;
#pragma unroll
        for (int e = 0; e < EACH; ++e)
          if (from + i * EACH + e < DMAS) dma1(o, st, from + i * EACH + e);
        __builtin_amdgcn_sched_barrier(0);
      };
    };
    auto nothing = [](int) {};
    constexpr int P = Step::parts;
    static_assert(P % 2 == 0, "the fragment buffers alternate");
    // step s from `cur`; `next`: another one follows (in `nxt`), `ahead`: and one behind it
    auto step = [&](int s, char* cur, char* nxt, bool next, bool ahead) {
#pragma unroll
      for (int p = 0; p + 1 < P; ++p) {
        fetch(cur, p + 1, a[(p + 1) & 1], b[(p + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
        if (p == 0) multiply(a[0], b[0], dma_between(next, s + 1, nxt, MB * EACH));
        else multiply(a[p & 1], b[p & 1], nothing);
      }
      if (next) {
        __syncthreads();  // every wave has read `cur`, and `nxt` has landed
        fetch(nxt, 0, a[0], b[0]);
        __builtin_amdgcn_sched_barrier(0);
      }
      multiply(a[1], b[1], dma_between(ahead, s + 2, cur, 0));
    };
    dma(0, st0, 0, DMAS);
    __syncthreads();
    if (steps > 1) dma(1, st1, 0, min(MB * EACH, DMAS));
    fetch(st0, 0, a[0], b[0]);
    int s = 0;
#pragma unroll 1
    for (; s + 3 < steps; s += 2) {
      step(s, st0, st1, true, true);
      step(s + 1, st1, st0, true, true);
    }
#pragma unroll 1
    for (; s < steps; s += 2) {  // the last one to three
      step(s, st0, st1, s + 1 < steps, s + 2 < steps);
      if (s + 1 < steps) step(s + 1, st1, st0, s + 2 < steps, false);
    }
    __syncthreads();  // the stages are free for the epilogue
  }
};

}  // namespace kans
