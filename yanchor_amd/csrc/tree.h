// Drafted trees: the packed nodes of a request, their ancestors, and division
// by a run-time constant, shared by the kernels that work on them.
#pragma once
#include "common.h"

namespace yh {
namespace tree {

constexpr int kNodes = 64;   // most nodes of a request: one wave, one 64-bit set

// The packed rows [first, first + count) of request r: offsets are clamped to
// the rows that exist, so no offset leads outside them.
struct Span {
  int64_t first;
  int64_t count;
};
__device__ __forceinline__ Span span_of(const int32_t* cu, int64_t r, int64_t total) {
  int64_t s = cu[r], e = cu[r + 1];
  s = s < 0 ? 0 : s > total ? total : s;
  e = e < s ? s : e > total ? total : e;
  return {s, e - s};
}

// Lane i's node i (one wave, all lanes active), `up` its parent: the set of its
// ancestors, itself included, by doubling -- after step k, `set` holds the nodes
// less than 2^k steps up and `up` the node 2^k steps up (-1: the context).  A
// parent that is not an earlier node counts as the context.  The sum of `x` along
// the path is formed with it.
__device__ __forceinline__ uint64_t ancestors_of(int up, double* x = nullptr) {
  const int lane = threadIdx.x & (kWave - 1);
  if (up >= lane || up < 0) up = -1;
  uint64_t set = 1ull << lane;
  double v = x ? *x : 0.;
#pragma unroll
  for (int step = 0; step < 6; ++step) {
    const int from = up < 0 ? lane : up;
    const uint64_t other = __shfl(set, from, kWave);
    const double ov = x ? __shfl(v, from, kWave) : 0.;
    const int next = __shfl(up, from, kWave);
    if (up >= 0) {
      set |= other;
      v += ov;
      up = next;
    }
  }
  if (x) *x = v;
  return set;
}
// The same for the n nodes whose parents are at `parents` (null: a chain).
__device__ __forceinline__ uint64_t ancestors(const int32_t* parents, int n, double* x = nullptr) {
  const int lane = threadIdx.x & (kWave - 1);
  return ancestors_of(lane >= n ? -1 : parents ? parents[lane] : lane - 1, x);
}

// n / d for 0 <= n < 2^31 by a multiplication: m = ceil(2^(31 + l) / d) with
// l = ceil(log2 d) is below 2^32, and its error e = m d - 2^(31 + l) < d <= 2^l
// keeps n e below 2^(31 + l).
struct Div {
  uint32_t m, d;
  int s;
  __device__ __forceinline__ uint32_t quot(uint32_t n) const {
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * m) >> s);
  }
};
inline Div make_div(uint32_t d) {
  int l = 0;
  while ((1ull << l) < d) ++l;
  const unsigned __int128 p = static_cast<unsigned __int128>(1) << (31 + l);
  return {static_cast<uint32_t>((p + d - 1) / d), d, 31 + l};
}

// Request of packed row t among r in [lo, hi]: the last with cu[r] <= t.
__device__ __forceinline__ int request_of(const int32_t* cu, int lo, int hi, int64_t t) {
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__host__ __device__ inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Packed rows behind the last request become zeros.  How many there are only the
// device knows, and a step captured for its largest batch has mostly those: one
// workgroup for every 64 KB that there could be, up to one a CU, at the end of the
// grid.  (128 requests of 6 nodes in 8192 rows of 32 x 128: attention 6013 us with
// one workgroup, 102 now, the delta rule 3028 and 78; without such rows
// 92 and 72.)
inline int64_t clearing(int64_t total, int64_t row) {
  const int64_t n = total * row >> 16;
  return n < 1 ? 1 : n < 256 ? n : 256;
}
// Workgroup `share` of `shares`, THREADS each: its part of rows [cu[R], total) of
// `row` bytes, a multiple of 16.
template <int THREADS>
__device__ __forceinline__ void clear_rows(void* out, const int32_t* cu, int R, int64_t total, int64_t row,
                                           int64_t share, int64_t shares) {
  const int64_t end = R ? cu[R] : 0, first = end < 0 ? 0 : end;
  const int64_t at = share * THREADS + threadIdx.x, step = shares * THREADS;
  if (aligned16(out)) {
    uint4* x = static_cast<uint4*>(out);
    for (int64_t i = first * (row / 16) + at; i < total * (row / 16); i += step) x[i] = make_uint4(0, 0, 0, 0);
  } else {
    uint16_t* x = static_cast<uint16_t*>(out);
    for (int64_t i = first * (row / 2) + at; i < total * (row / 2); i += step) x[i] = 0;
  }
}

}  // namespace tree
}  // namespace yh
