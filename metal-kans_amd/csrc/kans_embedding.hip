// Rows of a table for the tokens of a batch, scaled, and the table's gradient (gfx950).
//
//   out[n] = s W[token[n]],   dW[v] = s sum of dout[n] over the n with token[n] = v
//
// Both directions move memory and do nothing else.  The gradient reads every row of dout once and writes every row of dW
// once, rows of tokens that the batch has not as zeros.  A sum in the order of arrival (atomics) would change with every
// run and read dW as well; here the tokens are sorted first, equal ones in the order of their positions, and runs of
// equal tokens are added up in fp32:
//   1. k_embed_sort: a workgroup for each range of the vocabulary looks through all tokens (a few of them are its own)
//      and puts the positions of its own where they belong in the sorted order.  It counts the smaller tokens on the
//      way, so that no workgroup waits for another.
//   2. k_embed_sum: the sorted positions in pieces of equal length, whatever tokens they hold, so that a token that
//      fills a tenth of the batch holds nothing up.  Runs inside a piece are finished there; those that cross its ends
//      leave a partial row in fp32.  Further workgroups write the rows without tokens.
//   3. k_embed_join adds the partial rows of a run in their order.
// bf16, 16384 tokens of 65536 x 4096: rows 33 us (268 MB, 8 TB/s: frequent rows come from the caches); the gradient's sort 15, sums
// and zeros 104 (671 MB, 6.4 TB/s), join 7.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "kans_api_internal.h"

namespace kans {
namespace {

template <typename T> constexpr int vec() { return 16 / (int)sizeof(T); }  // elements of a 16-byte access

template <typename T> struct Vec { T v[vec<T>()]; };
// (rows start at any element: the device takes wide accesses at any address)
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {
  Vec<T> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <typename T> using Wide = unsigned __attribute__((ext_vector_type(4), aligned(sizeof(T))));
// Results leave nontemporal: lines that are written whole need not be read or kept.
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& v) {
  __builtin_nontemporal_store(__builtin_bit_cast(Wide<T>, v), (Wide<T>*)p);
}

// Where thread i of a row's accesses reads: the last access ends with the row and overlaps the one before, whose elements
// both compute alike.  Rows shorter than an access go by elements (step 1).
__device__ __forceinline__ int column(int i, int step, int D) { return min(i * step, D - step); }

// ---- forward ------------------------------------------------------------------------------------------
struct LookupArgs {
  const int64_t* tokens;
  const void* w;
  void* out;
  long n;
  int64_t ignore;
  int D, V, per_row;  // per_row: threads of a row
  float scale;
};

template <typename T, bool kWide>
__global__ __launch_bounds__(256) void k_embed_lookup(const LookupArgs A) {
  constexpr int S = kWide ? vec<T>() : 1;
  const int rows = 256 / A.per_row, lane = threadIdx.x % A.per_row, accesses = (A.D + S - 1) / S;
  const long row = (long)blockIdx.x * rows + threadIdx.x / A.per_row;
  if (row >= A.n) return;
  const int64_t token = A.tokens[row];
  const bool there = token >= 0 && token < A.V, ignored = token == A.ignore;
  const T* w = (const T*)A.w + (there && !ignored ? token : 0) * A.D;
  T* out = (T*)A.out + row * A.D;
  for (int i = lane; i < accesses; i += A.per_row) {
    const int c = column(i, S, A.D);
    auto value = [&](T v) { return from_f32<T>(ignored ? 0.0f : there ? to_f32(v) * A.scale : __builtin_nanf("")); };
    if constexpr (kWide) {
      Vec<T> v = load_vec(w + c);
#pragma unroll
      for (int e = 0; e < S; ++e) v.v[e] = value(v.v[e]);
      store_vec(out + c, v);
    } else {
      out[c] = value(w[c]);
    }
  }
}

// ---- gradient -----------------------------------------------------------------------------------------
// Workspace: position[N] and token[N] in sorted order, count[V], total[1] (ints), then partial rows in fp32, two for each piece.
struct GradArgs {
  const int64_t* tokens;
  const void* dout;
  void* dw;
  int *position, *token, *count, *total;
  float* part;
  int n;
  int64_t ignore;
  int D, V, range;              // range: tokens of a sorting workgroup
  int piece, pieces;            // positions of a piece
  int col_blocks, fill_rows;    // workgroups beside each other along a row; rows of a workgroup that writes zeros
  float scale;
};

constexpr int kSortThreads = 1024, kWaves = kSortThreads / 64, kPer = 8, kRound = kSortThreads * kPer;  // tokens of a thread, of a round
constexpr int kHeld = 4 * kRound;  // tokens that stay in registers between counting and placing
// Lists of more entries than kAlone are placed by all waves, where their counters (of up to kShared tokens each) fit:
// 16384 tokens by their frequency in a language, 65536 in all: 22 -> 15 us.  A range has V / 256 tokens, so that beyond 131072
// rows one wave places every list: 16 us at 131072, 22 at 131073, 20 at 262144.
constexpr int kAlone = 256, kShared = 512;
constexpr int kMaxRange = 8192;
constexpr int kMaxPiece = 64;  // positions of a piece at most
constexpr int kMaxFill = 256;  // rows of a workgroup that writes zeros, a wave's counts one a lane

__global__ __launch_bounds__(kSortThreads) void k_embed_sort(const GradArgs A) {
  __shared__ int place[kMaxRange];                     // counts of the range's tokens, then where the next one goes
  __shared__ unsigned list_at[kRound];    // this workgroup's positions of a round, in order
  __shared__ unsigned short list_token[kRound];
  __shared__ int sums[kPer * kSortThreads / 64];  // of each 64 tokens of a round, in order
  __shared__ int of_wave[kWaves][kShared];
  __shared__ int below_all, carry, listed;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int lo = blockIdx.x * A.range, hi = min(lo + A.range, A.V), mine = hi - lo;
  for (int i = t; i < mine; i += kSortThreads) place[i] = 0;
  if (t == 0) below_all = carry = 0;
  __syncthreads();
  // counts
  int below = 0, held[kHeld / kSortThreads];
  auto hold = [&](int first) {
    constexpr int kAll = kHeld / kSortThreads;
    int64_t v[kAll];
#pragma unroll
    for (int j = 0; j < kAll; ++j)
      if (first + j * kSortThreads < A.n) v[j] = A.tokens[min(first + j * kSortThreads + t, A.n - 1)];
#pragma unroll
    for (int j = 0; j < kAll; ++j)
      held[j] = first + j * kSortThreads >= A.n || first + j * kSortThreads + t >= A.n || v[j] == A.ignore || v[j] < 0 || v[j] >= A.V ? A.V : (int)v[j];
  };
  for (int first = 0; first < A.n; first += kHeld) {
    hold(first);
#pragma unroll
    for (int j = 0; j < kHeld / kSortThreads; ++j) {
      if (first + j * kSortThreads >= A.n) break;
      below += held[j] < lo;
      if (held[j] >= lo && held[j] < hi) atomicAdd(&place[held[j] - lo], 1);
    }
  }
  for (int d = 32; d > 0; d >>= 1) below += __shfl_xor(below, d, 64);
  if (lane == 0) atomicAdd(&below_all, below);
  __syncthreads();
  // places: an exclusive sum of the counts, behind the smaller tokens
  for (int first = 0; first < mine; first += kSortThreads) {
    const int i = first + t, c = i < mine ? place[i] : 0;
    if (i < mine) A.count[lo + i] = c;
    int s = c;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(s, d, 64);
      if (lane >= d) s += o;
    }
    if (lane == 63) sums[wave] = s;
    __syncthreads();
    int before = below_all + carry;
    for (int w = 0; w < wave; ++w) before += sums[w];
    if (i < mine) place[i] = before + s - c;
    __syncthreads();
    if (t == kSortThreads - 1) carry += before - below_all - carry + s;
    __syncthreads();
  }
  if (hi == A.V && t == 0) *A.total = below_all + carry;
  // positions: those of this range listed in order, then placed by one wave, 64 at a time
  int bits = 0;
  while (mine > 1 << bits) ++bits;
  for (int first = 0; first < A.n; first += kHeld) {
    if (A.n > kHeld) hold(first);
#pragma unroll
    for (int round = 0; round < kHeld / kRound; ++round) {
      const int from = first + round * kRound;
      if (from >= A.n) break;
      const int* v = held + round * kPer;
      unsigned long long own[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        own[j] = __ballot(v[j] >= lo && v[j] < hi);
        if (lane == 0) sums[j * (kSortThreads / 64) + wave] = __popcll(own[j]);
      }
      __syncthreads();
      if (wave == 0) {  // what comes before each 64
        static_assert(kPer * kSortThreads / 64 == 128, "two sums a lane");
        const int a = sums[2 * lane], b = sums[2 * lane + 1];
        int s = a + b;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const int o = __shfl_up(s, d, 64);
          if (lane >= d) s += o;
        }
        sums[2 * lane] = s - a - b;
        sums[2 * lane + 1] = s - b;
        if (lane == 63) listed = s;
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (v[j] >= lo && v[j] < hi) {
          const int at = sums[j * (kSortThreads / 64) + wave] + __popcll(own[j] & ((1ull << lane) - 1));
          list_at[at] = (unsigned)(from + j * kSortThreads + t);
          list_token[at] = (unsigned short)(v[j] - lo);
        }
      __syncthreads();
      // Entries [i, end) of the list by one wave, 64 at a time: the rank among equal tokens from the votes on each bit.
      auto put = [&](int* to, int i, int end) {
        int next = list_token[min(i + lane, kRound - 1)];
        unsigned next_at = list_at[min(i + lane, kRound - 1)];
        for (; i < end; i += 64) {
          const bool on = i + lane < end;
          const int k = on ? next : 0;
          const unsigned position = next_at;
          next = list_token[min(i + 64 + lane, kRound - 1)];
          next_at = list_at[min(i + 64 + lane, kRound - 1)];
          unsigned long long same = __ballot(on);
          for (int b = 0; b < bits; ++b) {
            const unsigned long long set = __ballot(k >> b & 1);
            same &= k >> b & 1 ? set : ~set;
          }
          const int rank = __popcll(same & ((1ull << lane) - 1));
          const int at = on ? to[k] + rank : 0;
          // (the loads of `to` by the whole wave are done before the first of each token's lanes moves it on)
          if (on) {
            A.position[at] = (int)position;
            A.token[at] = lo + k;
            if (rank == 0) to[k] += __popcll(same);
          }
        }
      };
      if (listed <= kAlone || mine > kShared) {
        if (wave == 0) put(place, 0, listed);
      } else {
        const int each = (listed + kSortThreads - 1) / kSortThreads * 64, first_of = min(wave * each, listed), end_of = min(first_of + each, listed);
        for (int i = t; i < kWaves * kShared; i += kSortThreads) of_wave[0][i] = 0;
        __syncthreads();
        for (int i = first_of + lane; i < end_of; i += 64) atomicAdd(&of_wave[wave][list_token[i]], 1);
        __syncthreads();
        if (t < mine) {
          int at = place[t];
#pragma unroll
          for (int w = 0; w < kWaves; ++w) {
            const int c = of_wave[w][t];
            of_wave[w][t] = at;
            at += c;
          }
          place[t] = at;
        }
        __syncthreads();
        put(of_wave[wave], first_of, end_of);
      }
      __syncthreads();
    }
  }
}

// Zeros in those of A.fill_rows rows from `first` on that have no tokens, 64 rows' counts read at once.
template <typename T, bool kWide>
__device__ __forceinline__ void fill_rows(const GradArgs& A, int first) {
  constexpr int S = kWide ? vec<T>() : 1;
  const int lane = threadIdx.x & 63, rows = A.fill_rows / 4, accesses = (A.D + S - 1) / S;
  first += (threadIdx.x >> 6) * rows;
  unsigned long long empty = __ballot(lane < rows && first + lane < A.V && A.count[min(first + lane, A.V - 1)] == 0);
  Vec<T> zero;
#pragma unroll
  for (int e = 0; e < vec<T>(); ++e) zero.v[e] = from_f32<T>(0.0f);
  for (; empty; empty &= empty - 1) {
    T* row = (T*)A.dw + (long)(first + __builtin_ctzll(empty)) * A.D;
    for (int i = lane; i < accesses; i += 64) {
      if constexpr (kWide) store_vec(row + column(i, S, A.D), zero);
      else row[i] = zero.v[0];
    }
  }
}

// One access of a row for each thread; the sum of a run of equal tokens stays in registers.
template <typename T, bool kWide>
__global__ __launch_bounds__(256) void k_embed_sum(const GradArgs A) {
  constexpr int S = kWide ? vec<T>() : 1, kAhead = 8;
  const int accesses = (A.D + S - 1) / S;
  T* dw = (T*)A.dw;
  if ((int)blockIdx.x >= A.pieces * A.col_blocks) {
    fill_rows<T, kWide>(A, (blockIdx.x - A.pieces * A.col_blocks) * A.fill_rows);
    return;
  }
  const int p = blockIdx.x / A.col_blocks, i = (blockIdx.x - p * A.col_blocks) * 256 + threadIdx.x;
  const int total = *A.total, first = p * A.piece, end = min(first + A.piece, total);
  if (first >= total || i >= accesses) return;
  const int c = column(i, S, A.D);
  const T* dout = (const T*)A.dout + c;
  float s[S] = {};
  int key = A.token[first];
  bool open = first > 0 && A.token[first - 1] == key;  // the run began before this piece
  auto finish = [&](bool goes_on) {
    if (open || goes_on) {
      float* part = A.part + (2L * p + (open ? 0 : 1)) * A.D + c;
#pragma unroll
      for (int e = 0; e < S; ++e) part[e] = s[e];
      return;
    }
    T* row = dw + (long)key * A.D + c;
    if constexpr (kWide) {
      Vec<T> o;
#pragma unroll
      for (int e = 0; e < S; ++e) o.v[e] = from_f32<T>(s[e] * A.scale);
      store_vec(row, o);
    } else {
      row[0] = from_f32<T>(s[0] * A.scale);
    }
  };
  for (int at = first; at < end; at += kAhead) {
    Vec<T> v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const T* row = dout + (long)A.position[min(at + j, end - 1)] * A.D;
      if constexpr (kWide) v[j] = load_vec(row);
      else v[j].v[0] = row[0];
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (at + j >= end) break;
      const int k = A.token[at + j];
      if (k != key) {
        finish(false);
        key = k;
        open = false;
#pragma unroll
        for (int e = 0; e < S; ++e) s[e] = 0.0f;
      }
#pragma unroll
      for (int e = 0; e < S; ++e) s[e] += to_f32(v[j].v[e]);
    }
  }
  finish(end < total && A.token[end] == key);
}

// The runs that begin in a piece and end in a later one.
template <typename T, bool kWide>
__global__ __launch_bounds__(256) void k_embed_join(const GradArgs A) {
  constexpr int S = kWide ? vec<T>() : 1;
  const int p = blockIdx.x / A.col_blocks, i = (blockIdx.x - p * A.col_blocks) * 256 + threadIdx.x;
  const int total = *A.total, first = p * A.piece, end = first + A.piece;
  if (end >= total || i >= (A.D + S - 1) / S) return;
  const int key = A.token[end];
  if (A.token[end - 1] != key || (A.token[first] == key && first > 0 && A.token[first - 1] == key)) return;
  const int c = column(i, S, A.D);
  // the run's first position in the piece and its length give the piece in which it ends
  int begin = end - 1;
  for (int half = kMaxPiece; half > 0; half >>= 1)  // (powers of two, whatever the piece: they add up to any distance)
    if (begin - half >= first && A.token[begin - half] == key) begin -= half;
  const int last = (begin + A.count[key] - 1) / A.piece;
  float s[S];
#pragma unroll
  for (int e = 0; e < S; ++e) s[e] = A.part[(2L * p + 1) * A.D + c + e];
#pragma unroll 8
  for (int q = p + 1; q <= last; ++q) {
    const float* part = A.part + 2L * q * A.D + c;
#pragma unroll
    for (int e = 0; e < S; ++e) s[e] += part[e];
  }
  T* row = (T*)A.dw + (long)key * A.D + c;
#pragma unroll
  for (int e = 0; e < S; ++e) row[e] = from_f32<T>(s[e] * A.scale);
}

// ---- launches -----------------------------------------------------------------------------------------
struct EmbedPlan {
  int range, groups;   // tokens of a sorting workgroup, and how many such
  int piece, pieces;
  int accesses, col_blocks;
  bool wide;
  long ints, bytes;    // ints of the workspace before the partial rows
};
EmbedPlan plan_embed(int esize, long n, int D, int V) {
  EmbedPlan p{};
  // every sorting workgroup reads all tokens
  p.range = (V + 255) / 256;
  p.range = std::min(p.range, kMaxRange);
  p.groups = (V + p.range - 1) / p.range;
  p.piece = (int)std::min((long)kMaxPiece, std::max(8L, (n + 511) / 512 + 7 & ~7L));
  p.pieces = (int)((n + p.piece - 1) / p.piece);
  const int step = 16 / esize;
  p.wide = D >= step;
  p.accesses = p.wide ? (D + step - 1) / step : D;
  p.col_blocks = (p.accesses + 255) / 256;
  p.ints = (2 * n + V + 1 + 3) & ~3L;
  p.bytes = p.ints * 4 + 2L * p.pieces * D * 4;
  return p;
}

int check_embed(int dtype, long n, int D, int V, double scale) {
  if (dtype != DT_F32 && dtype != DT_F16 && dtype != DT_BF16) return kans_fail(KANS_ERR_ARG, "dtype %d", dtype);
  if (n < 0 || D <= 0 || V <= 0) return kans_fail(KANS_ERR_ARG, "bad dims N=%ld D=%d V=%d", n, D, V);
  // (the kernels multiply in fp32: zeros would meet an infinite scale, and a scale below its normal numbers has lost digits)
  if (!(scale == 0.0 || (std::fabs(scale) >= FLT_MIN && std::fabs(scale) <= FLT_MAX)))
    return kans_fail(KANS_ERR_ARG, "scale must be zero or a normal number of fp32");
  // (a grid holds fewer than 2^32 threads along x)
  if (n > (1L << 23) || D > (1 << 16) || V > (1 << 24))
    return kans_fail(KANS_ERR_UNSUPPORTED, "N=%ld D=%d V=%d, up to 2^23 tokens, 2^16 columns and 2^24 rows", n, D, V);
  return 0;
}

template <typename F>
hipError_t by_type(int dtype, bool wide, F f) {
  auto go = [&](auto t) { return wide ? f(t, std::true_type{}) : f(t, std::false_type{}); };
  if (dtype == DT_F32) return go(0.0f);
  return dtype == DT_F16 ? go((_Float16)0.0f) : go((__bf16)0.0f);
}

}  // namespace
}  // namespace kans

using namespace kans;

extern "C" {

int kans_embedding_forward(int dtype, const int64_t* tokens, const void* W, long N, int D, int V, int64_t ignore_index, double scale,
                           void* out, void* stream) {
  int rc = check_embed(dtype, N, D, V, scale);
  if (rc || N == 0) return rc;
  if (!tokens || !W || !out) return kans_fail(KANS_ERR_ARG, "null argument");
  std::lock_guard<std::mutex> lk(kans_mutex());
  if ((rc = kans_ensure_init())) return rc;
  const EmbedPlan p = plan_embed(dtype == DT_F32 ? 4 : 2, N, D, V);
  LookupArgs A{tokens, W, out, N, ignore_index, D, V, 256, (float)scale};
  while (A.per_row > 16 && A.per_row / 2 >= p.accesses) A.per_row /= 2;
  const int rows = 256 / A.per_row;
  HIP_TRY(by_type(dtype, p.wide, [&](auto t, auto wide) {
    hipLaunchKernelGGL((k_embed_lookup<decltype(t), decltype(wide)::value>), dim3((unsigned)((N + rows - 1) / rows)), dim3(256), 0,
                       kans_caller_stream(stream), A);
    return hipGetLastError();
  }));
  return 0;
}

long kans_embedding_workspace(int dtype, long N, int D, int V) {
  const int rc = check_embed(dtype, N, D, V, 1.0);
  return rc ? rc : plan_embed(dtype == DT_F32 ? 4 : 2, N, D, V).bytes;
}

int kans_embedding_backward(int dtype, const int64_t* tokens, const void* dout, long N, int D, int V, int64_t ignore_index,
                            double scale, void* dW, void* workspace, long workspace_bytes, void* stream) {
  int rc = check_embed(dtype, N, D, V, scale);
  if (rc) return rc;
  if (!dW || (N && (!tokens || !dout))) return kans_fail(KANS_ERR_ARG, "null argument");
  const int esize = dtype == DT_F32 ? 4 : 2;
  const EmbedPlan p = plan_embed(esize, N, D, V);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < p.bytes)
    return kans_fail(KANS_ERR_ARG, "workspace of %ld bytes, %ld at a multiple of 16 needed", workspace ? workspace_bytes : 0, p.bytes);
  std::lock_guard<std::mutex> lk(kans_mutex());
  if ((rc = kans_ensure_init())) return rc;
  hipStream_t st = kans_caller_stream(stream);
  GradArgs A{};
  A.tokens = tokens; A.dout = dout; A.dw = dW;
  A.position = (int*)workspace;
  A.token = A.position + N;
  A.count = A.token + N;
  A.total = A.count + V;
  A.part = (float*)workspace + p.ints;
  A.n = (int)N; A.ignore = ignore_index; A.D = D; A.V = V; A.range = p.range;
  A.piece = p.piece; A.pieces = p.pieces; A.col_blocks = p.col_blocks; A.scale = (float)scale;
  A.fill_rows = 4 * (int)std::max(1L, std::min(kMaxFill / 4L, 16384L / ((long)D * esize)));
  hipLaunchKernelGGL(k_embed_sort, dim3(p.groups), dim3(kSortThreads), 0, st, A);
  HIP_TRY(hipGetLastError());
  const long blocks = (long)p.pieces * p.col_blocks;
  HIP_TRY(by_type(dtype, p.wide, [&](auto t, auto wide) {
    hipLaunchKernelGGL((k_embed_sum<decltype(t), decltype(wide)::value>), dim3((unsigned)(blocks + (V + A.fill_rows - 1) / A.fill_rows)),
                       dim3(256), 0, st, A);
    return hipGetLastError();
  }));
  if (p.pieces < 2) return 0;
  HIP_TRY(by_type(dtype, p.wide, [&](auto t, auto wide) {
    hipLaunchKernelGGL((k_embed_join<decltype(t), decltype(wide)::value>), dim3((unsigned)blocks), dim3(256), 0, st, A);
    return hipGetLastError();
  }));
  return 0;
}

}  // extern "C"
