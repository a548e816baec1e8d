// Matrix product of the cross entropy kernels (kans_xent.hip): C[m][n] = sum_k A[m][k] B[n][k] on the 16-bit
// matrix cores, with the epilogue taking the tile from the accumulators.
//
// k goes in steps of kStep.  An operand lies in memory either way:
//   row after row: step s of row r is `row_bytes` consecutive bytes at base + r * row_stride + s * step_stride;
//   column after column (COLUMNS): row_bytes of kStep consecutive rows r = b kStep .. at one k are at
//   base + b * block_stride + k * row_stride.
// Both cover a row-major matrix (as itself or as its transpose) and panels [step][row][kStep] of one, whose rows of a
// step are one contiguous run; the second reads its operands from LDS transposed (ds_read_b64_tr_b16).  So one layout of a
// matrix serves the products along either dimension.  fp32 operands (TERMS = 3) are the three bf16 terms of
// kans_split.h, [term][32] in a step, and take six MFMAs a product; A's may lie in memory as they are (A_RAW, rows of whole
// steps of 32), and are split on their way from LDS to the products.
//
// A workgroup of WAVES_M x WAVES_N waves holds a BM x BN tile.  A step's rows go from memory to LDS by DMA
// (buffer loads, 16 bytes a lane) into one of two stages, or of three for A (A_STAGES).  The barrier that opens step
// s + 1 stands before the last part of step s, whose operands are in registers by then; a part's operands are read
// between the products of the part before it.  The DMAs into the stages that step s has left go out in that
// part and the next one, a few between the products of each row of blocks: all of them at once fill the memory pipe's queue,
// and the waves stand there.  The stages are separate arrays and the step loop is unrolled until they repeat,
// so that the compiler sees that reads of one do not depend on the DMA into another.
//
// LDS rows are 128 (or, with three terms, 192) bytes, so a column of 16-byte chunks would meet the same banks in
// every second (fourth) row: chunk c of row r lies in slot c ^ reversed 3 bits of (r >> 1) (c ^ ((r >> 2) & 3)), which
// spreads 16 rows over all 64 banks, and four rows of 32 bytes, as the transposed reads take them, too (no
// conflict counted).  The DMA writes LDS in lane order, so it is the source address that is permuted, inside one row's
// step.
#pragma once
#include "kans_split.h"
#include "kans_tile.h"

namespace kans {

struct GemmOperand {
  const void* p;
  long row_stride, step_stride;  // bytes (step_stride: from a step of k to the next)
  int rows;                      // rows that exist (COLUMNS: blocks of them); those of a tile behind them repeat the last
  long block_stride;             // COLUMNS
  long bytes;                    // COLUMNS: zeros are read from base + bytes on (0: everything that is read exists)
};

template <int TERMS> struct StepOf {
  static constexpr int kStep = TERMS == 1 ? 64 : 32;              // k of a step
  static constexpr int row_bytes = kStep * 2 * TERMS;             // 128 or 192
  static constexpr int chunks = row_bytes / 16;
  static constexpr int parts = kStep / 16;                        // MFMA depths of a step
  static __device__ __forceinline__ int slot(int row, int chunk) {
    return TERMS == 1 ? chunk ^ ((row >> 3 & 1) | (row >> 1 & 2) | (row << 1 & 4)) : chunk ^ ((row >> 2) & 3);
  }
};

template <typename T, int TERMS, int BM, int BN, int WAVES_M, int WAVES_N, int A_STAGES, bool A_COLUMNS, bool B_COLUMNS, bool A_ONCE,
          bool A_RAW>
struct GemmTile {
  static_assert(!A_RAW || (TERMS == 3 && !A_COLUMNS), "raw fp32 rows of A");
  using Step = StepOf<TERMS>;
  using LinesA = StepOf<A_RAW ? 1 : TERMS>;  // a step's rows of A in LDS: raw ones are 128 bytes, as 16-bit ones are
  static constexpr int WAVES = WAVES_M * WAVES_N, THREADS = WAVES * 64;
  static constexpr int MB = BM / WAVES_M / 32, NB = BN / WAVES_N / 32;  // 32 x 32 blocks of a wave
  static constexpr int STAGE_A = BM * LinesA::row_bytes, STAGE_B = BN * Step::row_bytes;  // bytes of a stage
  static constexpr int DMA_A = STAGE_A / 1024 / WAVES, DMA_B = STAGE_B / 1024 / WAVES;  // of a wave
  static_assert(DMA_A * 1024 * WAVES == STAGE_A && DMA_B * 1024 * WAVES == STAGE_B, "whole DMAs");
  static_assert(A_STAGES == 2 || (A_STAGES == 3 && DMA_A < 16), "stages of A");
  typedef typename Mfma<T>::frag frag;

  // A raw buffer from p on, 32-bit offsets, zeros behind `records` bytes.  Buffer loads, not global ones: behind a
  // global load to LDS the compiler waits for every LDS read where it could wait for the older ones.
  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const char* p, unsigned records) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0, (int)records, 0x00027000);
  }
  template <bool COLUMNS>
  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t source(const GemmOperand& o, const char* p, int s, int first) {
    const unsigned records =
        COLUMNS && o.bytes ? (unsigned)(o.bytes - (long)(first + s) * o.step_stride - (p - (const char*)o.p)) : 0xffffffffu;
    return resource(p + (long)(first + s) * o.step_stride, records);
  }

  // acc = the tile at (m0, n0) over `steps` steps from step `first`; zeros in the waves whose rows of A or B are all
  // behind the first `rows_m` or `rows_n`.
  static __device__ __forceinline__ void run(const GemmOperand& A, const GemmOperand& B, int m0, int n0, int rows_m, int rows_n,
                                             int first, int steps,
                                             char* a_st0, char* a_st1, char* a_st2, char* b_st0, char* b_st1,
                                             floatx16 (&acc)[MB][NB]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WAVES_N, wn = wave % WAVES_N;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    if (steps <= 0) return;
    // the tile's first row, and this lane's places in its rows
    unsigned off_a[DMA_A], off_b[DMA_B];
    constexpr int KS = Step::kStep;
    auto start = [&](const GemmOperand& o, int tile0, auto columns) {
      if constexpr (decltype(columns)::value) return (const char*)o.p + (long)min(tile0 / KS, o.rows - 1) * o.block_stride;
      else return (const char*)o.p + (long)min(tile0, o.rows - 1) * o.row_stride;
    };
    auto place = [&](int q, int tile0, const GemmOperand& o, auto columns, auto lines) {
      using L = decltype(lines);
      const int row = q / L::chunks, chunk = L::slot(row, q - row * L::chunks);
      if constexpr (decltype(columns)::value) {
        const int b0 = min(tile0 / KS, o.rows - 1), block = min(tile0 / KS + row / KS, o.rows - 1) - b0;
        return (unsigned)block * (unsigned)o.block_stride + (unsigned)(row % KS) * (unsigned)o.row_stride + chunk * 16;
      } else {
        return (unsigned)(min(tile0 + row, o.rows - 1) - min(tile0, o.rows - 1)) * (unsigned)o.row_stride + chunk * 16;
      }
    };
    constexpr std::integral_constant<bool, A_COLUMNS> a_columns{};
    constexpr std::integral_constant<bool, B_COLUMNS> b_columns{};
#pragma unroll
    for (int i = 0; i < DMA_A; ++i) off_a[i] = place((i * WAVES + wave) * 64 + lane, m0, A, a_columns, LinesA{});
#pragma unroll
    for (int i = 0; i < DMA_B; ++i) off_b[i] = place((i * WAVES + wave) * 64 + lane, n0, B, b_columns, Step{});
    const char *pa = start(A, m0, a_columns), *pb = start(B, n0, b_columns);
    auto source_a = [&](int s) { return source<A_COLUMNS>(A, pa, s, first); };
    auto source_b = [&](int s) { return source<B_COLUMNS>(B, pb, s, first); };
    // (A_ONCE: no other tile reads A's rows, so they need not stay in a cache: nontemporal)
    auto dma_a = [&](const __amdgpu_buffer_rsrc_t& o, char* st, int i) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(o, (__attribute__((address_space(3))) void*)(st + (i * WAVES + wave) * 1024), 16,
                                               off_a[i], 0, 0, A_ONCE ? 2 : 0);
    };
    auto dma_b = [&](const __amdgpu_buffer_rsrc_t& o, char* st, int i) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(o, (__attribute__((address_space(3))) void*)(st + (i * WAVES + wave) * 1024), 16,
                                               off_b[i], 0, 0, 0);
    };
    const int row = lane & 31, half = lane >> 5;
    // operand of the 32 rows from 32 * block of a stage, at one part of the step
    auto read_rows = [&](const char* st, int block, int part, int term) {
      const int r = block * 32 + row, slot = Step::slot(r, term * (KS / 8) + part * 2 + half);
      return *(const frag*)(st + r * Step::row_bytes + slot * 16);
    };
    // Groups of 16 lanes take four k of 16 rows: a lane reads four rows' values at one k and gets four k of one row.  Its
    // places in this wave's blocks, by the block's half of a 128-byte row (16-bit: two blocks share one) and the four k of
    // eight; everything else is a constant distance from them.
    constexpr int HALVES = TERMS == 1 ? 2 : 1;
    static_assert(TERMS == 3 || ((MB % 2 == 0 || MB == 1) && (NB % 2 == 0 || NB == 1)), "a wave's blocks are whole pairs, or one");
    int at_a[HALVES][2], at_b[HALVES][2];
    if constexpr (A_COLUMNS || B_COLUMNS) {
      const int in16 = lane & 15, rows16 = lane >> 4 & 1;
      auto place_columns = [&](int w, int blocks, int q, int h) {  // of wave row or column w with so many blocks
        const int k = half * 8 + h * 4 + in16 / 4, pair = TERMS == 3 ? 0 : blocks == 1 ? w & 1 : q;
        const int first = TERMS == 3 ? w * blocks * 32 : w * blocks / 2 * 64;
        return (first + k) * Step::row_bytes + Step::slot(k, pair * 4 + rows16 * 2 + in16 % 4 / 2) * 16 + in16 % 2 * 8;
      };
#pragma unroll
      for (int q = 0; q < HALVES; ++q)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          at_a[q][h] = place_columns(wm, MB, q, h);
          at_b[q][h] = place_columns(wn, NB, q, h);
        }
    }
    auto read_columns = [&](const char* st, const int (&at)[HALVES][2], int block, int part, int term) {
      typedef short short4_t __attribute__((ext_vector_type(4)));
      struct { short4_t v[2]; } f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        f.v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(
            st + (block * 32 / KS * KS + part * 16) * Step::row_bytes + term * 64 + at[block % HALVES][h]));
      return __builtin_bit_cast(frag, f);
    };
    // raw rows: eight fp32 values, made into their terms before the products
    struct Raw8 { float4 v[2]; };
    auto read_raw = [&](const char* st, int block, int part) {
      const int r = block * 32 + row, chunk = part * 4 + half * 2;
      Raw8 f;
#pragma unroll
      for (int h = 0; h < 2; ++h) f.v[h] = *(const float4*)(st + r * LinesA::row_bytes + LinesA::slot(r, chunk + h) * 16);
      return f;
    };
    Raw8 raw[2][A_RAW ? MB : 1];
    frag a[2][MB][TERMS], b[2][NB][TERMS];
    // The operands of one part in MB pieces: A's i-th block and its share of B's.
    auto fetch = [&](const char* sa, const char* sb, int part, int to, int i) {
      auto& fa = a[to];
      auto& fb = b[to];
      if constexpr (A_RAW) raw[to][i] = read_raw(sa, wm * MB + i, part);
#pragma unroll
      for (int t = 0; t < TERMS; ++t) {
        if constexpr (A_RAW) {
        } else if constexpr (A_COLUMNS) fa[i][t] = read_columns(sa, at_a, i, part, t);
        else fa[i][t] = read_rows(sa, wm * MB + i, part, t);
#pragma unroll
        for (int j = 0; j < NB; ++j)
          if (j % MB == i) {
            if constexpr (B_COLUMNS) fb[j][t] = read_columns(sb, at_b, j, part, t);
            else fb[j][t] = read_rows(sb, wn * NB + j, part, t);
          }
      }
    };
    // The products of one part.  between(i) goes out behind the first of the i-th row of blocks: what it issues is
    // hidden by the matrix pipe (all of the next part's reads before the first product cost a tenth of dW's time).
    auto multiply = [&](int from, auto between) {
      auto& fa = a[from];
      const auto& fb = b[from];
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        if constexpr (A_RAW) {
          float v[8];
          __builtin_memcpy(v, &raw[from][i], sizeof(v));
          const Split8 s = split8(v);
#pragma unroll
          for (int t = 0; t < TERMS; ++t) fa[i][t] = __builtin_bit_cast(frag, s.t[t]);
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          if constexpr (TERMS == 3) acc[i][j] = mma_split(fa[i], fb[j], acc[i][j]);
          else acc[i][j] = Mfma<T>::mma(fa[i][0], fb[j][0], acc[i][j]);
          if (j == 0) {
            __builtin_amdgcn_sched_barrier(0);
            between(i);
          }
          if (j == 0 || j == NB - 1) __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    // The DMAs that go out behind the barrier of step s: B of step s + 2, then A of step s + A_STAGES (so that those
    // which the next barrier need not wait for are the last); EACH of them before each of 2 MB rows of blocks.
    // `all`: both steps exist.
    constexpr int DMAS = DMA_A + DMA_B, EACH = (DMAS + 2 * MB - 1) / (2 * MB);
    auto dma_between = [&](int s, char* sa, char* sb, int from, bool all) {
      const auto ra = source_a(s + A_STAGES), rb = source_b(s + 2);
      const bool on_a = all || s + A_STAGES < steps, on_b = all || s + 2 < steps;
      return [=](int i) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          const int k = from + i * EACH + e;
          if (k < DMA_B) {
            if (on_b) dma_b(rb, sb, k < DMA_B ? k : 0);
          } else if (k < DMAS) {
            if (on_a) dma_a(ra, sa, k < DMAS ? k - DMA_B : 0);
          }
        }
      };
    };
    // What this wave has read and asked for is there, but for the newest DMAs of A (of the step after the next) where
    // they have gone out; then all waves meet.
    auto meet = [&](bool newest_a_out) {
      asm volatile("" ::: "memory");
      if (A_STAGES == 3 && newest_a_out) __builtin_amdgcn_s_waitcnt(0x70 | DMA_A);  // vmcnt(DMA_A) lgkmcnt(0)
      else __builtin_amdgcn_s_waitcnt(0x70);                                        // vmcnt(0) lgkmcnt(0)
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    constexpr int P = Step::parts;
    static_assert(P % 2 == 0, "the fragment buffers alternate");
    // step s from (a_cur, b_cur); the next one is in (a_nxt, b_nxt), the one before was in (a_old, b_nxt)
    auto step = [&](int s, char* a_old, char* a_cur, char* a_nxt, char* b_cur, char* b_nxt, bool all) {
#pragma unroll
      for (int p = 0; p + 1 < P; ++p) {
        if (p == 0) {
          const auto dma = dma_between(s - 1, a_old, b_nxt, MB * EACH, all);
          multiply(0, [&](int i) {
            fetch(a_cur, b_cur, p + 1, 1, i);
            dma(i);
          });
        } else {
          multiply(p & 1, [&](int i) { fetch(a_cur, b_cur, p + 1, (p + 1) & 1, i); });
        }
      }
      const bool next = all || s + 1 < steps;
      if (next) meet(all || s + 2 < steps);  // every wave has read step s, and step s + 1 has landed
      const auto dma = dma_between(s, a_cur, b_cur, 0, all);
      multiply(1, [&](int i) {
        if (next) fetch(a_nxt, b_nxt, 0, 0, i);
        dma(i);
      });
    };
    // step 0, and what would have gone out behind the steps before it
    {
      const auto ra = source_a(0), rb = source_b(0), ra1 = source_a(1);
#pragma unroll
      for (int i = 0; i < DMA_A; ++i) dma_a(ra, a_st0, i);
#pragma unroll
      for (int i = 0; i < DMA_B; ++i) dma_b(rb, b_st0, i);
      if (A_STAGES == 3 && steps > 1) {
#pragma unroll
        for (int i = 0; i < DMA_A; ++i) dma_a(ra1, a_st1, i);
      }
      meet(steps > 1);
      const auto first_half = dma_between(-1, A_STAGES == 3 ? a_st2 : a_st1, b_st1, 0, false);
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        fetch(a_st0, b_st0, 0, 0, i);
        first_half(i);
      }
    }
    constexpr int ROUND = A_STAGES == 3 ? 6 : 2;  // steps until the stages repeat
    char* const as[3] = {a_st0, a_st1, a_st2};
    char* const bs[2] = {b_st0, b_st1};
    if (m0 + wm * MB * 32 >= rows_m || n0 + wn * NB * 32 >= rows_n) {
      // nothing to multiply: this wave's DMAs and barriers, in the same order
      char *old = a_st2, *cur = a_st0, *nxt = a_st1, *b_cur = b_st0, *b_nxt = b_st1;
      if (A_STAGES == 2) old = a_st1;
#pragma unroll 1
      for (int s = 0; s < steps; ++s) {
        const auto second_half = dma_between(s - 1, old, b_nxt, MB * EACH, false);
#pragma unroll
        for (int i = 0; i < MB; ++i) second_half(i);
        if (s + 1 < steps) meet(s + 2 < steps);
        const auto first_half = dma_between(s, cur, b_cur, 0, false);
#pragma unroll
        for (int i = 0; i < MB; ++i) first_half(i);
        char *const a_third = old, *const b_first = b_cur;
        old = cur;
        cur = nxt;
        nxt = A_STAGES == 3 ? a_third : old;
        b_cur = b_nxt;
        b_nxt = b_first;
      }
      __syncthreads();
      return;
    }
    auto round = [&](int s, bool all) {
      static_for<0, ROUND>([&](auto k) {
        constexpr int i = decltype(k)::value;
        if (all || s + i < steps)
          step(s + i, as[(i + A_STAGES - 1) % A_STAGES], as[i % A_STAGES], as[(i + 1) % A_STAGES], bs[i % 2], bs[(i + 1) % 2], all);
      });
    };
    int s = 0;
#pragma unroll 1
    for (; s + ROUND + A_STAGES - 1 < steps; s += ROUND) round(s, true);
#pragma unroll 1
    for (; s < steps; s += ROUND) round(s, false);
    __syncthreads();  // the stages are free for the epilogue
  }
};

}  // namespace kans
