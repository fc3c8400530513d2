// Attention of one new token a request over a block cache of 16, 8 or 4 bits.
//
// Request r has L positions in its cache, the new token's among them (the last).
// Query head h of KV head g = h / (H / G) sees p from max(starts, L - window, 0,
// L - columns * block) to L - 1:
//   x_p = q . k_p scale;  x_p = cap tanh(x_p / cap);  x_p -= slope_h (L - 1 - p)
//   out = sum_p softmax(x)_p v_p (* sigmoid(gate)),  zeros where nothing is seen
//
// A wave takes 16 NT positions of a KV head (NT 4, 2 or 1, as a row is short or
// long) and up to 16 of its query heads on 16x16x32 MFMA:
//   S^T = K Q^T      row i of product t is position 16 t + i, so that the lane
//                    (column lane % 16, quarter lane / 16) ends with the scores of
//                    positions 16 t + 4 quarter + j
//   O^T += V^T P^T   and that is where the B operand of step t wants their weights
// The order of a product's terms is free, so a lane loads K and V rows straight
// into the places of the A operands, whole pieces of a row (a quarter's D / 4 dims
// of K, D / 16 dims of V), and nothing goes through LDS.  Codes become bf16 by
// v_cvt_scalef32, exactly, two dims of a position to a dword.  K wants them so; for
// V a dword's two slots of the reduction are one position's two dims, so B holds
// the position's weight in the even slot and zero in the odd one for a column of
// the even dim, the other way round for the odd dim: with HP <= 8 heads the columns
// head and head + HP are those two, with 16 heads there are two products.
// With HP = 4 the other eight columns take half of the positions, each lane half of
// the exponentials; their sums join at the end.  (Pairs transposed by v_perm, as many
// as there are conversions, and all exponentials in every column: 156 us for 135 with
// 64 requests over 4 bits.)  In 16 bits, where there are no conversions beside it, the
// pairs are transposed.
// A weight of zero does not take out a value that is not finite (NaN codes, 16-bit
// infinities, codes of 2^128 and more, which bf16 holds as infinities), so a part's
// sums that are not finite are formed again by dims.
// Weights enter as two values of the product's type each (hi + lo, 16 bits at
// least), since the denominator sums them as they are: rounded once, equal weights
// would all be off the same way.  With fp16 queries over codes, whose 11 bits bf16
// does not hold, the queries do too.
//
// Requests are few or of very different lengths, so tiles of 16 NT positions are
// cut into parts of about one size, which every workgroup finds from the lengths
// by itself; its four waves take the part's tiles in turn and join their sums in
// LDS.  Parts of a request that was cut leave theirs, with their maximum, in the
// workspace, and a second launch joins them in order.
//
// Bound by HBM: 133 ragged requests over 8 bits 216 us (1.18 GB, 5.5 TB/s), 8 long
// contexts 194 (6.1), 64 requests over 4 bits 120 (5.3), heads of 256 in 16 bits 151
// (5.6), where a large copy reaches 6.2 and a read alone 7.0.  Nontemporal loads,
// since up to 16 query heads of a KV head share one read of its rows: the long
// contexts 201 us for 217.  (Every 16 heads more are a workgroup of their own that
// reads them once more.)  Blocks that runs of 16 positions straddle (block % 16) have
// their table entries and rows a lane: 220 us for the long contexts with blocks of 24,
// 367 with blocks of 1.
#include <type_traits>

#include "attn_tile.h"
#include "qcache.h"
#include "tree.h"

namespace yh {
namespace {

using namespace qcache;
using tree::Div;
using attn::bf16x8_t;
using attn::f16x8_t;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kCols = 16;        // query heads that a wave takes
// Products of 16 positions in a tile: as many as keep its keys in 32 registers, and leave room for queries of two parts.
constexpr int products(int row_bytes, bool pair) {
  return row_bytes < 128 || (row_bytes == 128 && !pair) ? 4 : row_bytes <= 256 ? 2 : 1;
}
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kFloor = -3.0e38f;   // below every score: the maximum of nothing
// fp16 weights are e^(x - max) 2^14, up to a quarter of the type's range: weights below 2^-14 of the largest, of which
// a long cache may have very many, then keep 22 bits down to 2^-17 and 11 down to 2^-28.  The denominator carries the
// same factor.
constexpr float kLift = 14.f;

struct DecodeArgs {
  const uint16_t* q;       // [R, H, D], tokens q_ts apart
  int64_t q_ts;
  const char* keys;        // [blocks, G, block, row bytes]
  const char* values;
  const uint8_t* key_scales;     // [blocks, G, D / 32, block]
  const uint8_t* value_scales;
  const int32_t* tables;   // [R, columns]
  const int64_t* lengths;  // [R]
  const int64_t* starts;   // [R] or null
  const float* slopes;     // [H] or null
  const uint16_t* gate;    // [R, H, D] with strides, or null
  int64_t g_ts, g_hs;
  uint16_t* out;           // [R, H, D]
  int64_t window;          // 0: none
  float scale, cap;        // cap 0: none
  Div block, columns;
  int R, H, G, rep, mtiles, blocks, target;
  int32_t* first;          // [R + 1] first part of each request
  float* part;             // [parts][H][D]
  float2* stat;            // [parts][H] maximum and denominator
};

// Tables through the scalar cache: a run of 16 positions lies in one block.
typedef __attribute__((address_space(4))) int32_t ConstInt;

// The table's entry for position p of request r.
__device__ __forceinline__ int table_entry(const DecodeArgs& a, int r, int p) {
  const uint32_t b = a.block.quot(p);
  return ((const ConstInt*)(a.tables + static_cast<int64_t>(r) * a.columns.d))[b - a.columns.quot(b) * a.columns.d];
}
__device__ __forceinline__ bool block_there(const DecodeArgs& a, int id) {
  return static_cast<uint32_t>(id) < static_cast<uint32_t>(a.blocks);
}
// The row of all rows of all heads, and where its scale of run 0 lies.  An entry that is no block of the cache leads
// to block 0, whose contents are masked.
struct Row {
  int64_t row, scale;
};
template <int D>
__device__ __forceinline__ Row row_at(const DecodeArgs& a, int g, int id, int p) {
  const uint32_t in = p - a.block.quot(p) * a.block.d;
  const int64_t first = (static_cast<int64_t>(block_there(a, id) ? id : 0) * a.G + g) * a.block.d;
  return {first + in, first * (D / kRun) + in};
}

// The kernel's arguments, loaded where this stands: kept over a loop before it they would take the loop's scalar registers.
__device__ __forceinline__ const DecodeArgs& arguments_again() {
  typedef __attribute__((address_space(4))) DecodeArgs Const;
  Const* p = (Const*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const DecodeArgs*)p;
}

// First and last + 1 of the positions that request r sees.
struct Seen {
  int lo, hi;
};
__device__ __forceinline__ Seen seen_of(const DecodeArgs& a, int r) {
  const int64_t len = a.lengths[r];
  if (len <= 0) return {0, 0};
  int64_t lo = len - static_cast<int64_t>(a.columns.d) * a.block.d;
  if (a.window && len - a.window > lo) lo = len - a.window;
  if (a.starts && a.starts[r] > lo) lo = a.starts[r];
  if (lo < 0) lo = 0;
  if (lo >= len || len > 0x7ffff000ll || a.blocks == 0) return {0, 0};
  return {static_cast<int>(lo), static_cast<int>(len)};
}
template <int TILE>
__device__ __forceinline__ int tiles_of(Seen s) {
  return s.hi > s.lo ? (s.hi + TILE - 1) / TILE - s.lo / TILE : 0;
}

// Wave-inclusive sum over lanes.
__device__ __forceinline__ int scan_wave(int x) {
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int y = __shfl_up(x, off, kWave);
    if (lane >= off) x += y;
  }
  return x;
}

struct Part {
  int r, index, count, slot;   // request, which of its parts, how many, number of the part among all
  int tile, tiles;             // its tiles, from the request's first
  Seen seen;
};

// Tiles of a part, of `total` of each KV head: as many as leave `target` parts, and a turn of the waves at least; up to
// four turns (eight of 16 positions) where there are more than two parts a CU, since each begins with a chain of loads.
// (us of captured calls, 8 KV heads of 128 in 8 bits, with a turn at least: 64 requests of 900 positions 27 for 37, 200
// of 1800 157 for 169; heads of 256 in 16 bits, eight turns and four: 93 and 98 with 64 requests of 900.)
template <int TILE>
__device__ __forceinline__ int chunk_of(const DecodeArgs& a, int total) {
  if (a.target == 0) return 0x7fffffff;
  constexpr int kMost = (TILE == 16 ? 8 : 4) * kWaves;
  const int fine = (total + a.target - 1) / a.target;
  const int64_t room = static_cast<int64_t>(total) * (a.G * a.mtiles) / 512;
  const int turns = room < kWaves ? kWaves : room > kMost ? kMost : static_cast<int>(room);
  return fine > turns ? fine : turns;
}
__device__ __forceinline__ int parts_of(int tiles, int chunk) { return tiles > chunk ? (tiles + chunk - 1) / chunk : 1; }
// Part `index` of `count` of a request of n tiles; they differ by a tile.
__device__ __forceinline__ Part part_of(int r, int index, int count, int slot, int n, Seen seen) {
  const int each = n / count, rest = n % count;
  return {r, index, count, slot, index * each + (index < rest ? index : rest), each + (index < rest ? 1 : 0), seen};
}

// Part `which` of all, found from the lengths; count 0: there is none.  Every wave finds it by itself where it has a
// lane for each request (one request: 7.6 us for 9.8 with the workgroup's scan; four requests a lane: 8.3, and nothing
// gained for 133).
template <int TILE>
__device__ Part find_part(const DecodeArgs& a, int which) {
  if (a.R <= kWave) {
    const int lane = threadIdx.x & (kWave - 1);
    const Seen seen = lane < a.R ? seen_of(a, lane) : Seen{0, 0};
    const int n = tiles_of<TILE>(seen);
    const int chunk = chunk_of<TILE>(a, __shfl(scan_wave(n), kWave - 1, kWave));
    const int c = lane < a.R ? parts_of(n, chunk) : 0, end = scan_wave(c);
    const uint64_t behind = __ballot(end > which);
    if (behind == 0) return {0, 0, 0, 0, 0, 0, {0, 0}};
    const int r = __ffsll(static_cast<unsigned long long>(behind)) - 1;
    const auto of = [&](int x) { return __builtin_amdgcn_readlane(x, r); };
    return part_of(r, which - (of(end) - of(c)), of(c), which, of(n), {of(seen.lo), of(seen.hi)});
  }
  __shared__ int sums[kWaves], found[4];
  const int t = threadIdx.x, w = t / kWave;
  // a thread takes `each` requests in a row
  const int each = (a.R + kThreads - 1) / kThreads, r0 = t * each, r1 = r0 + each < a.R ? r0 + each : a.R;
  int mine = 0;
  for (int r = r0; r < r1; ++r) mine += tiles_of<TILE>(seen_of(a, r));
  int s = scan_wave(mine);
  if ((t & (kWave - 1)) == kWave - 1) sums[w] = s;
  if (t == 0) found[0] = -1;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) total += sums[i];
  __syncthreads();
  const int chunk = chunk_of<TILE>(a, total);
  mine = 0;
  for (int r = r0; r < r1; ++r) mine += parts_of(tiles_of<TILE>(seen_of(a, r)), chunk);
  s = scan_wave(mine);
  if ((t & (kWave - 1)) == kWave - 1) sums[w] = s;
  __syncthreads();
  int at = s - mine;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) at += i < w ? sums[i] : 0;
  if (which >= at && which < at + mine) {
    for (int r = r0; r < r1; ++r) {
      const int n = tiles_of<TILE>(seen_of(a, r)), c = parts_of(n, chunk);
      if (which < at + c) {
        found[0] = r;
        found[1] = which - at;
        found[2] = c;
        found[3] = n;
        break;
      }
      at += c;
    }
  }
  __syncthreads();
  if (found[0] < 0) return {0, 0, 0, 0, 0, 0, {0, 0}};
  return part_of(found[0], found[1], found[2], which, found[3], seen_of(a, found[0]));
}

// Two dims of one position's codes to bf16 under the scale 2^(s - 127), given as a float whose exponent s is: the
// conversion takes no more of it, and makes NaN of any code under s = 255.
__device__ __forceinline__ float exponent(uint32_t s) { return __uint_as_float(s << 23); }
template <int FMT>
struct Codes;
template <>
struct Codes<kFp8> {
  static constexpr int kBits = 8;
  template <int PAIR>
  static __device__ __forceinline__ uint32_t two(const uint32_t* w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[PAIR / 2], s, PAIR % 2 == 1));
  }
};
template <>
struct Codes<kFp4> {
  static constexpr int kBits = 4;
  template <int PAIR>
  static __device__ __forceinline__ uint32_t two(const uint32_t* w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[PAIR / 4], s, PAIR % 4));
  }
};
template <>
struct Codes<k16> {
  static constexpr int kBits = 16;
  template <int PAIR>
  static __device__ __forceinline__ uint32_t two(const uint32_t* w, float) {
    return w[PAIR];
  }
};

// BYTES bytes (2 to 32) into dwords.
template <int BYTES>
__device__ __forceinline__ void load_bytes(uint32_t* w, const char* p) {
  if constexpr (BYTES == 2) {
    w[0] = *reinterpret_cast<const uint16_t*>(p);
  } else if constexpr (BYTES == 4) {
    w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  } else if constexpr (BYTES == 8) {
    const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
    w[0] = x[0];
    w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + 16 * i));
#pragma unroll
      for (int j = 0; j < 4; ++j) w[4 * i + j] = x[j];
    }
  }
}

// Value `dim` of the row at `row` of all rows, its scale of run 0 at `scale`, runs `run` apart.
template <int DT, int FMT, int D>
__device__ __forceinline__ float value_of(const char* data, const uint8_t* scales, int64_t row, int64_t scale, uint32_t run,
                                          int dim) {
  if constexpr (FMT == k16) {
    return attn::Mfma<DT>::widen(reinterpret_cast<const uint16_t*>(data)[row * D + dim]);
  } else {
    const float s = scale_value(scales[scale + static_cast<int64_t>(dim / kRun) * run]);
    if constexpr (FMT == kFp8) {
      return __builtin_amdgcn_cvt_f32_fp8(static_cast<uint8_t>(data[row * D + dim]), 0) * s;
    } else {
      const auto two = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(static_cast<uint8_t>(data[(row * D + dim) / 2]), 1.f, 0);
      return (dim & 1 ? two[1] : two[0]) * s;
    }
  }
}

template <int I, int N, class F>
__device__ __forceinline__ void each(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each<I + 1, N>(f);
  }
}

// 1 - 2 / (e^2x + 1), which is off by some 2^-24: below 0.3 the series to x^9 (2^-24 of its value there), since a cap
// far above the scores makes all of them small.
__device__ __forceinline__ float tanh_of(float x) {
  const float y = x * x;
  const float p = fmaf(y, fmaf(y, fmaf(y, fmaf(y, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
  const float e = 1.f - 2.f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(2.f * kLog2e * x) + 1.f);
  return y < 0.09f ? x * p : e;
}

// The product's type: the queries' for a 16-bit cache, bf16 for codes.
template <int MT>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (MT == YH_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
// With four positions of each quarter.
template <int MT>
__device__ __forceinline__ f32x4 mfma(u32x2 a, u32x2 b, f32x4 c) {
  if constexpr (MT == YH_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
}
// Two weights as hi + lo, each rounded to the product's type.
template <int MT>
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  using P = attn::Mfma<MT>;
  hi = P::round2(x, y);
  lo = P::round2(x - P::widen(hi & 0xffff), y - P::widen(hi >> 16));
}
// The compiler puts no wait where a matrix result is first read behind branches that meet.
template <int N>
__device__ __forceinline__ void settle(f32x4 (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
  asm volatile("s_nop 7\n\ts_nop 7" : "+v"(x[0]));
#pragma unroll
  for (int i = 1; i < N; ++i) asm volatile("" : "+v"(x[i]));
}

// Four dims of a head's output: o / den, gated.  Where nothing was seen they are zeros, whatever the gate of an idle row
// holds.
template <int DT>
__device__ __forceinline__ void put4(const DecodeArgs& a, int r, int head, int dim, int D, const float* o, float den) {
  using M = attn::Mfma<DT>;
  const float inv = 1.f / den;
  uint16_t y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float z = o[e] * inv;
    if (a.gate) z *= 1.f / (1.f + __expf(-M::widen(a.gate[r * a.g_ts + head * a.g_hs + dim + e])));
    y[e] = den == 0.f ? 0 : M::round(z);
  }
  const int64_t to = (static_cast<int64_t>(r) * a.H + head) * D + dim;
  *reinterpret_cast<u32x2*>(a.out + to) = u32x2{attn::pack2(y[0], y[1]), attn::pack2(y[2], y[3])};
}

// Whether four dims' sums can be taken as they are.  Where the denominator is no number, no dim is one; elsewhere a sum
// that is not finite says nothing of its own dim.
__device__ __forceinline__ bool all_finite(float den, const float* o) {
  return den != den || fabsf(o[0]) + fabsf(o[1]) + fabsf(o[2]) + fabsf(o[3]) < INFINITY;
}

// Waves a SIMD that the registers are held to: as many as fit without spilling, but
// for fp16 queries over 8 bits with sixteen columns of heads of 256, which spill up to 9 registers (us of the long contexts
// with 128 heads, blocks of 64 and 24: 462 and 549, with one wave a SIMD 524 and 582).
constexpr int waves_for(int DT, int FMT, int D, int HP, bool RUNS) {
  if (D == 64) return 3;
  if (D == 128 && FMT == kFp4 && DT == YH_BF16 && HP == 4 && RUNS) return 4;
  return D == 256 || (FMT != k16 && (HP == 16 || !RUNS || (FMT == kFp8 && DT == YH_F16))) ? 2 : 3;
}

template <int DT, int FMT, int D, int HP, bool RUNS>
__global__ void __launch_bounds__(kThreads, waves_for(DT, FMT, D, HP, RUNS)) decode_attention_kernel(DecodeArgs a) {
  using C = Codes<FMT>;
  constexpr int MT = FMT == k16 ? DT : YH_BF16;
  using P = attn::Mfma<MT>;
  constexpr bool kPair = FMT != k16 && DT == YH_F16;    // queries as hi + lo
  constexpr int kRow = D * C::kBits / 8;                // bytes of a row
  constexpr int kKd = D / 4, kVd = D / 16;              // dims of a lane: K, V
  constexpr int kKb = kRow / 4, kVb = kRow / 16;        // and their bytes
  constexpr int kKw = (kKb + 3) / 4, kVw = (kVb + 3) / 4;
  // A lane's K dims come in pieces of 16 bytes, piece c of quarter q at byte 64 c + 16 q, so that a load takes whole
  // 64 bytes of each row (D / 4 dims in a row a lane: 513 us for 400 with 8 bits, D = 256 and 2.4 GB).
  constexpr int kPb = kKb < 16 ? kKb : 16, kPd = kPb * 8 / C::kBits, kPieces = kKb / kPb;
  constexpr int kSteps = D / 32;                        // products over the dims
  constexpr int NT = products(kRow, kPair && D == 256), kTile = 16 * NT, kU = 4 * NT;   // kU: positions of a quarter
  constexpr int kSel = HP == 16 || FMT == k16 ? 1 : 2;               // columns of a head: two dims, halves of the positions
  constexpr int kHalves = HP == 16 ? 1 : 2 * 8 / (HP * kSel);
  constexpr int kAcc = kVd / kSel, kMine = kU / kHalves;             // positions whose weights a lane forms
  __shared__ float2 wave_stat[kWaves][kHalves][HP];
  __shared__ float wave_acc[kWaves][kHalves][HP][D + 4];
  // columns whose sums are not finite, and what forms them again
  __shared__ uint32_t spoiled;
  __shared__ float redo_weight[kThreads], redo_sum[kThreads / (D / 4)][D];
  __shared__ int redo_id[kThreads];

  const int g = blockIdx.x % a.G, mt = blockIdx.x / a.G % a.mtiles;
  const Part part = find_part<kTile>(a, blockIdx.x / a.G / a.mtiles);
  if (part.count == 0) return;
  // the whole workgroup's
  const int r = __builtin_amdgcn_readfirstlane(part.r), tiles = __builtin_amdgcn_readfirstlane(part.tiles);
  const int lo = __builtin_amdgcn_readfirstlane(part.seen.lo), hi = __builtin_amdgcn_readfirstlane(part.seen.hi);
  if (a.first && part.index == 0 && g == 0 && mt == 0 && threadIdx.x == 0) {
    a.first[r] = part.slot;
    if (r == a.R - 1) a.first[a.R] = part.slot + part.count;
  }

  const int lane = threadIdx.x & (kWave - 1), w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int quarter = lane >> 4, piece = lane & 15;     // piece: the lane's part of a V row, its position of K rows
  const int col = piece % HP, sel = piece / HP % kSel, half = piece / (HP * kSel);
  const int cols = a.rep - mt * kCols < HP ? a.rep - mt * kCols : HP;
  const int head = g * a.rep + mt * kCols + (col < cols ? col : 0);

  // the queries as the B operand: column `col`, dims as the K rows have them
  u32x4 qh[kSteps], ql[kPair ? kSteps : 1];
#pragma unroll
  for (int c = 0; c < kSteps; ++c) {
    const int dim = 8 * c / kPd * (4 * kPd) + kPd * quarter + 8 * c % kPd;
    u32x4 x = *reinterpret_cast<const u32x4*>(a.q + r * a.q_ts + static_cast<int64_t>(head) * D + dim);
    if (col >= cols) x = u32x4{0, 0, 0, 0};
    if constexpr (kPair) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x0 = f16_to_f32(x[i] & 0xffff), x1 = f16_to_f32(x[i] >> 16);
        const uint16_t h0 = f32_to_bf16(x0), h1 = f32_to_bf16(x1);
        qh[c][i] = attn::pack2(h0, h1);
        ql[c][i] = attn::pack2(f32_to_bf16(x0 - bf16_to_f32(h0)), f32_to_bf16(x1 - bf16_to_f32(h1)));
      }
    } else {
      qh[c] = x;
    }
  }
  // scores in powers of two, of a cap in caps
  const bool plain = a.cap == 0.f && !a.slopes;
  const float mul = a.cap > 0.f ? a.scale / a.cap : kLog2e * a.scale;
  const float cap2 = a.cap * kLog2e, slope = a.slopes ? a.slopes[head] * kLog2e : 0.f;
  // Biases count from the end that has the least: the sum of a large one and a score would lose the score.
  const int origin = slope < 0.f ? lo : hi - 1;
  // which of a dword's two slots holds a weight in this lane's column
  const uint32_t slot_mask = kSel == 1 ? 0u : sel ? 0xffff0000u : 0xffffu;

  float top = kFloor, den = 0.f;
  f32x4 acc[kAcc];
#pragma unroll
  for (int n = 0; n < kAcc; ++n) acc[n] = f32x4{0, 0, 0, 0};

  auto id_of = [&](int p) { return table_entry(a, r, p); };
  auto is_block = [&](int id) { return block_there(a, id); };
  auto row_of = [&](int id, int p) { return row_at<D>(a, g, id, p); };
  const int first_tile = lo / kTile + __builtin_amdgcn_readfirstlane(part.tile);

  // The lane's positions of product t, of 16 t on: `piece` of K, 4 quarter + j of V.
  uint32_t kw[NT][kKw], vw[kU][kVw];
  uint32_t ksc[NT][kPieces], vsc[NT];      // scale bytes of a K position, of four V positions
  // Table entries of the next tile's products, the whole wave's where blocks hold whole runs of 16 positions, of the
  // lane's K positions elsewhere, and their rows, or the entries of the tile whose V is loaded.
  int ids[NT], own_ids[NT];
  Row rows[NT];
  auto load_ids = [&](int i) {
#pragma unroll
    for (int t = 0; t < NT; ++t) ids[t] = id_of((first_tile + i) * kTile + 16 * t + (RUNS ? 0 : piece));
  };
  uint32_t holes = 0, vhole = 0;       // V's positions without a block: of the next tile, of this one
  const uint32_t k_off = (RUNS ? piece * kRow : 0) + quarter * kPb;
  const uint32_t v_off = RUNS ? 4 * quarter * kRow + piece * kVb : 0;
  const uint32_t ks_off = (quarter * kPd / kRun) * a.block.d + (RUNS ? piece : 0);
  const uint32_t vs_off = RUNS ? (piece * kVd / kRun) * a.block.d + 4 * quarter : 0;
  auto k_row = [&](int t, const char* p) {
#pragma unroll
    for (int c = 0; c < kPieces; ++c) load_bytes<kPb>(kw[t] + kPb / 4 * c, p + 64 * c);
  };
  auto k_scale = [&](int t, int64_t at) {
    if constexpr (FMT != k16) {
#pragma unroll
      for (int c = 0; c < kPieces; ++c)
        ksc[t][c] = *(a.key_scales + at + static_cast<int64_t>(c * (4 * kPd / kRun)) * a.block.d + ks_off);
    }
  };
  auto load_k = [&](int i) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int p = (first_tile + i) * kTile + 16 * t;
      if constexpr (RUNS) {      // the run's block is the whole wave's
        const Row at = rows[t];
        k_row(t, a.keys + at.row * kRow + k_off);
        k_scale(t, at.scale);
      } else {
        const Row at = row_of(ids[t], p + piece);
        k_row(t, a.keys + at.row * kRow + k_off);
        k_scale(t, at.scale);
      }
    }
  };
  auto load_v = [&](int i) {
    vhole = RUNS ? holes : 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int p = (first_tile + i) * kTile + 16 * t;
      if constexpr (RUNS) {
        const Row at = rows[t];
#pragma unroll
        for (int j = 0; j < 4; ++j) load_bytes<kVb>(vw[4 * t + j], a.values + at.row * kRow + v_off + j * kRow);
        if constexpr (FMT != k16) vsc[t] = *reinterpret_cast<const uint32_t*>(a.value_scales + at.scale + vs_off);
      } else {
        vsc[t] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // that of the lane which has the position for K
          const int at_p = p + 4 * quarter + j, id = __shfl(own_ids[t], 4 * quarter + j, kWave);
          const Row at = row_of(id, at_p);
          vhole |= is_block(id) ? 0u : 1u << (4 * t + j);
          load_bytes<kVb>(vw[4 * t + j], a.values + at.row * kRow + piece * kVb);
          if constexpr (FMT != k16)
            vsc[t] |= static_cast<uint32_t>(a.value_scales[at.scale + static_cast<int64_t>(piece * kVd / kRun) * a.block.d])
                      << (8 * j);
        }
      }
    }
  };
  auto find_rows = [&](int i) {
    if constexpr (RUNS) {
      holes = 0;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        rows[t] = row_of(ids[t], (first_tile + i) * kTile + 16 * t);
        holes |= is_block(ids[t]) ? 0u : 15u << (4 * t);
      }
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t) own_ids[t] = ids[t];
    }
  };

  // Loads run ahead of their use: a tile's keys while the tile before is turned into weights and sums, its values
  // while its own scores form, table entries a tile ahead.
  if (w < tiles) {
    load_ids(w);
    find_rows(w);
    load_k(w);
    load_v(w);
    if (w + kWaves < tiles) load_ids(w + kWaves);
  }
  for (int i = w; i < tiles; i += kWaves) {
    const int base = (first_tile + i) * kTile;
    const bool more = i + kWaves < tiles;

    // S^T, product t: positions 16 t on
    f32x4 s[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      s[t] = f32x4{0, 0, 0, 0};
      each<0, kSteps>([&](auto step) {
        constexpr int ST = decltype(step)::value;
        u32x4 x;
        const float sc = FMT == k16 ? 1.f : exponent(ksc[t][ST * 8 / kPd]);
        each<0, 4>([&](auto pair) {
          constexpr int I = decltype(pair)::value;
          x[I] = C::template two<4 * ST + I>(kw[t], sc);
        });
        s[t] = mfma<MT>(x, qh[ST], s[t]);
        if constexpr (kPair) s[t] = mfma<MT>(x, ql[ST], s[t]);
      });
    }
    settle(s);
    if (more) {
      find_rows(i + kWaves);
      load_k(i + kWaves);
    }

    // u = 4 t + j is position 16 t + 4 quarter + j, its score s[t][j]; with halves a lane has j = 2 half + {0, 1}
    const int own = 4 * quarter + (kHalves == 2 ? 2 * half : 0);
    auto step_of = [](int u) { return kHalves == 2 ? 16 * (u / 2) + u % 2 : 16 * (u / 4) + u % 4; };
    float x[kMine];
#pragma unroll
    for (int u = 0; u < kMine; ++u)
      x[u] = kHalves == 2 ? (half ? s[u / 2][2 + u % 2] : s[u / 2][u % 2]) : s[u / 4][u % 4];
    if (a.cap > 0.f) {
#pragma unroll
      for (int u = 0; u < kMine; ++u) x[u] = cap2 * tanh_of(x[u] * mul);
    }
    if (a.slopes) {
      const float back = static_cast<float>(origin - base - own), f = a.cap > 0.f ? 1.f : mul;
#pragma unroll
      for (int u = 0; u < kMine; ++u) x[u] = x[u] * f - slope * (back - static_cast<float>(step_of(u)));
    }
    uint32_t dead = vhole;     // what of the quarter is not seen
    if (base < lo || base + kTile > hi) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int p = base + 16 * (u / 4) + 4 * quarter + u % 4;
        dead |= p < lo || p >= hi ? 1u << u : 0u;
      }
    }
    if (__ballot(dead != 0)) {
      // it may be anything: its values are cleared too
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (dead >> u & 1) {
#pragma unroll
          for (int e = 0; e < kVw; ++e) vw[u][e] = 0;
          vsc[u / 4] = (vsc[u / 4] & ~(0xffu << (8 * (u % 4)))) | 0x7fu << (8 * (u % 4));
        }
      const uint32_t gone = kHalves == 2 ? dead >> (2 * half) : dead;
#pragma unroll
      for (int u = 0; u < kMine; ++u)
        x[u] = gone >> (kHalves == 2 ? 4 * (u / 2) + u % 2 : u) & 1 ? -INFINITY : x[u];
    }
    float m = x[0];
#pragma unroll
    for (int u = 1; u < kMine; ++u) m = fmaxf(m, x[u]);
    m = fmaxf(m, __shfl_xor(m, 16, kWave));
    m = fmaxf(m, __shfl_xor(m, 32, kWave));
    const float unit = plain ? mul : 1.f;      // x is in scores, or in powers of two already
    m *= unit;
    if (__ballot(m > top)) {
      const float next = fmaxf(top, m), f = __builtin_amdgcn_exp2f(top - next);
      top = next;
      den *= f;
#pragma unroll
      for (int n = 0; n < kAcc; ++n) acc[n] *= f;
    }
    const float low = MT == YH_F16 ? kLift - top : -top;
#pragma unroll
    for (int u = 0; u < kMine; ++u) {
      x[u] = __builtin_amdgcn_exp2f(fmaf(x[u], unit, low));
      den += x[u];
    }
    // O^T: step st takes positions 16 st + 4 quarter + e, product n dims 2 n and 2 n + 1 of each lane's kVd
#pragma unroll
    for (int st = 0; st < NT; ++st) {
      if constexpr (FMT == k16) {
        u32x2 ph, pl;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int at = kHalves == 2 ? 2 * st : 4 * st + 2 * e;
          uint32_t hi, lo;
          split2<MT>(x[at], x[at + 1], hi, lo);
          ph[e] = kHalves == 2 && half != e ? 0u : hi;
          pl[e] = kHalves == 2 && half != e ? 0u : lo;
        }
        each<0, kVd / 2>([&](auto pair) {
          constexpr int I = decltype(pair)::value;
          u32x2 lo, hi;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            lo[e] = __builtin_amdgcn_perm(vw[4 * st + 2 * e + 1][I], vw[4 * st + 2 * e][I], 0x05040100u);
            hi[e] = __builtin_amdgcn_perm(vw[4 * st + 2 * e + 1][I], vw[4 * st + 2 * e][I], 0x07060302u);
          }
          acc[2 * I] = mfma<MT>(lo, ph, acc[2 * I]);
          acc[2 * I + 1] = mfma<MT>(hi, ph, acc[2 * I + 1]);
          acc[2 * I] = mfma<MT>(lo, pl, acc[2 * I]);
          acc[2 * I + 1] = mfma<MT>(hi, pl, acc[2 * I + 1]);
        });
        continue;
      }
      // a step's weights are split in the step: all steps' at once spill with eight heads over 8 bits (248 us for 206
      // with 64 heads and the long contexts)
      __builtin_amdgcn_sched_barrier(0);
      u32x4 ph[2], pl[2];      // [1]: the odd dim's with one column a head
      float sc[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = x[kHalves == 2 ? 2 * st + e % 2 : 4 * st + e];
        const uint32_t hi = P::round2(y, y);
        const float rest = y - __uint_as_float(hi & 0xffff0000u);
        const uint32_t lo = P::round2(rest, rest);
        if constexpr (kSel == 2) {
          const uint32_t mask = kHalves == 2 ? (half == e / 2 ? slot_mask : 0u) : slot_mask;
          ph[0][e] = hi & mask;
          pl[0][e] = lo & mask;
        } else {
          ph[0][e] = hi & 0xffffu;
          ph[1][e] = hi & 0xffff0000u;
          pl[0][e] = lo & 0xffffu;
          pl[1][e] = lo & 0xffff0000u;
        }
        sc[e] = exponent((vsc[st] >> (8 * e)) & 0xff);
      }
      each<0, kVd / 2>([&](auto pair) {
        constexpr int I = decltype(pair)::value;
        u32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = C::template two<I>(vw[4 * st + e], sc[e]);
#pragma unroll
        for (int n = 0; n < 2 / kSel; ++n) {
          acc[2 / kSel * I + n] = mfma<MT>(v, ph[n], acc[2 / kSel * I + n]);
          acc[2 / kSel * I + n] = mfma<MT>(v, pl[n], acc[2 / kSel * I + n]);
        }
      });
    }
    if (more) {
      load_v(i + kWaves);
      if (i + 2 * kWaves < tiles) load_ids(i + 2 * kWaves);
    }
  }
  settle(acc);

  const DecodeArgs& b = arguments_again();

  // the waves' sums: lane (column, quarter) has dims (4 quarter + j) kVd + 2 n + sel, or + n, of its head in acc[n][j]
  den += __shfl_xor(den, 16, kWave);
  den += __shfl_xor(den, 32, kWave);
  if (quarter == 0 && sel == 0) wave_stat[w][half][col] = make_float2(top, den);
  if (col < cols) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int n = 0; n < kAcc; ++n) wave_acc[w][half][col][(4 * quarter + j) * kVd + kSel * n + sel] = acc[n][j];
  }
  if (threadIdx.x == 0) spoiled = 0;
  __syncthreads();
  // Four dims of a column: the largest score, the denominator and the sums of all waves.
  auto join = [&](int c, int dim, float& m, float& dn, float* o) {
    m = kFloor;
#pragma unroll
    for (int i = 0; i < kWaves * kHalves; ++i) m = fmaxf(m, wave_stat[i / kHalves][i % kHalves][c].x);
    dn = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves * kHalves; ++i) {
      const float2 st = wave_stat[i / kHalves][i % kHalves][c];
      const float f = __builtin_amdgcn_exp2f(st.x - m);
      dn = fmaf(st.y, f, dn);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(wave_acc[i / kHalves][i % kHalves][c][dim + e], f, o[e]);
    }
  };
  auto put = [&](int c, int dim, float m, float dn, const float* o) {
    const int hd = g * b.rep + mt * kCols + c;
    if (part.count > 1) {
      const int64_t slot = static_cast<int64_t>(part.slot) * b.H + hd;
      *reinterpret_cast<float4*>(b.part + slot * D + dim) = make_float4(o[0], o[1], o[2], o[3]);
      if (dim == 0) b.stat[slot] = make_float2(m, dn);
    } else {
      put4<DT>(b, r, hd, dim, D, o, dn);
    }
  };
  for (int at = threadIdx.x; at < cols * (D / 4); at += kThreads) {
    const int c = at / (D / 4), dim = at % (D / 4) * 4;
    float m, dn, o[4];
    join(c, dim, m, dn, o);
    if (all_finite(dn, o)) put(c, dim, m, dn, o);
    else atomicOr(&spoiled, 1u << c);
  }
  __syncthreads();
  // Values that are not finite reach, through weights of 0, the other dim of their dword and the other half of the
  // positions.  Sums that are not finite are formed again without such products, for the columns that have any: a lane
  // a position for the weights, four dims a lane for the sums.
#pragma unroll 1
  for (uint32_t left = spoiled; left; left &= left - 1) {
    constexpr int kLanes = D / 4, kShares = kThreads / kLanes;
    const int c = __builtin_ctz(left), share = threadIdx.x / kLanes, dim = threadIdx.x % kLanes * 4;
    const int hd = g * b.rep + mt * kCols + c;
    const uint16_t* qr = b.q + r * b.q_ts + static_cast<int64_t>(hd) * D;
    const float steep = b.slopes ? b.slopes[hd] * kLog2e : 0.f;
    const int end = (first_tile + tiles) * kTile < hi ? (first_tile + tiles) * kTile : hi;
    float m, dn, o[4], sum[4] = {0.f, 0.f, 0.f, 0.f};
    join(c, dim, m, dn, o);
#pragma unroll 1
    for (int p0 = first_tile * kTile < lo ? lo : first_tile * kTile; p0 < end; p0 += kThreads) {
      const int p = p0 + static_cast<int>(threadIdx.x);
      const int id = p < end ? table_entry(b, r, p) : -1;
      float wt = -1.f;
      if (block_there(b, id)) {
        const Row at = row_at<D>(b, g, id, p);
        float x = 0.f;
#pragma unroll 8
        for (int d = 0; d < D; ++d)
          x = fmaf(attn::Mfma<DT>::widen(qr[d]), value_of<DT, FMT, D>(b.keys, b.key_scales, at.row, at.scale, b.block.d, d), x);
        x = b.cap > 0.f ? b.cap * kLog2e * tanh_of(x * (b.scale / b.cap)) : x * (kLog2e * b.scale);
        if (b.slopes) x -= steep * static_cast<float>((steep < 0.f ? lo : hi - 1) - p);
        wt = __builtin_amdgcn_exp2f(x + (MT == YH_F16 ? kLift - m : -m));
      }
      __syncthreads();      // the positions before are summed
      redo_weight[threadIdx.x] = wt;
      redo_id[threadIdx.x] = id;
      __syncthreads();
      for (int j = share; j < kThreads && p0 + j < end; j += kShares) {
        const float wj = redo_weight[j];
        if (wj < 0.f) continue;
        const Row at = row_at<D>(b, g, redo_id[j], p0 + j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = value_of<DT, FMT, D>(b.values, b.value_scales, at.row, at.scale, b.block.d, dim + e);
          sum[e] = fabsf(v) < INFINITY ? fmaf(wj, v, sum[e]) : sum[e] + v;      // however small the weight
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) redo_sum[share][dim + e] = sum[e];
    __syncthreads();
    if (share == 0 && !all_finite(dn, o)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (fabsf(o[e]) < INFINITY) continue;
        o[e] = 0.f;
        for (int i = 0; i < kShares; ++i) o[e] += redo_sum[i][dim + e];
      }
      put(c, dim, m, dn, o);
    }
  }
}

// The parts of a cut request joined: a workgroup a head, D / 4 lanes a part, the others take every kShares-th part;
// their sums meet in LDS, in order.
template <int DT, int D>
__global__ void __launch_bounds__(kThreads) decode_join_kernel(DecodeArgs a) {
  constexpr int kLanes = D / 4, kShares = kThreads / kLanes;
  __shared__ float sums[kShares][D + 4], dens[kShares], tops[kShares];
  const int r = blockIdx.x / a.H, hd = blockIdx.x % a.H;
  const int share = threadIdx.x / kLanes, dim = threadIdx.x % kLanes * 4;
  const int first = a.first[r], count = a.first[r + 1] - first;
  if (count <= 1) return;
  const int64_t slot = static_cast<int64_t>(first) * a.H + hd;
  float m = kFloor, dn = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int j = share; j < count; j += kShares) {
    const int64_t s = slot + static_cast<int64_t>(j) * a.H;
    const float2 st = a.stat[s];
    const float4 x = *reinterpret_cast<const float4*>(a.part + s * D + dim);
    const float next = fmaxf(m, st.x), f = __builtin_amdgcn_exp2f(m - next), h = __builtin_amdgcn_exp2f(st.x - next);
    m = next;
    dn = fmaf(dn, f, st.y * h);
    o[0] = fmaf(o[0], f, x.x * h);
    o[1] = fmaf(o[1], f, x.y * h);
    o[2] = fmaf(o[2], f, x.z * h);
    o[3] = fmaf(o[3], f, x.w * h);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) sums[share][dim + e] = o[e];
  if (dim == 0) {
    dens[share] = dn;
    tops[share] = m;
  }
  __syncthreads();
  if (share) return;
#pragma unroll
  for (int i = 0; i < kShares; ++i) m = fmaxf(m, tops[i]);
  dn = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = 0.f;
#pragma unroll
  for (int i = 0; i < kShares; ++i) {
    const float f = __builtin_amdgcn_exp2f(tops[i] - m);
    dn = fmaf(dens[i], f, dn);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(sums[i][dim + e], f, o[e]);
  }
  if (!all_finite(dn, o)) {
    // a part's infinity stays one, where float32 holds its factor as 0
    auto scaled = [](float x, float f) { return fabsf(x) == INFINITY ? x : x * f; };
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = 0.f;
#pragma unroll 1
    for (int j = 0; j < count; ++j) {
      const int64_t s = slot + static_cast<int64_t>(j) * a.H;
      const float4 x = *reinterpret_cast<const float4*>(a.part + s * D + dim);
      const float f = __builtin_amdgcn_exp2f(a.stat[s].x - m);
      o[0] += scaled(x.x, f);
      o[1] += scaled(x.y, f);
      o[2] += scaled(x.z, f);
      o[3] += scaled(x.w, f);
    }
  }
  put4<DT>(a, r, hd, dim, D, o, dn);
}

// Parts aimed at, over all heads, so that the last of those that fit the chip (two or three workgroups a CU) end at
// about one time.  us of 133 requests over 8 bits, 64 over 4 bits and 8 long contexts: 1024 parts 236, 160, 236; 2048 229,
// 156, 219; 4096 239, 145, 230.
constexpr int kWorkgroups = 2048;

// Positions of a tile.
int64_t tile_of(int bits, int64_t D, int dtype) {
  return 16 * products(static_cast<int>(D * bits / 8), bits != 16 && dtype == YH_F16 && D == 256);
}
// Parts aimed at for each KV head, 0 where no request is cut and the second launch is not made: up to two turns of the
// waves, or eight where there are heads enough.  (400 positions, before the weights' second product: one request 7.7 us captured and 13 called for 8.9 and
// 18, 64 requests 15 for 22, 200 47 for 61.)
int64_t target_for(int64_t R, int64_t H, int64_t G, int64_t D, int64_t block, int64_t columns, int64_t window,
                   int64_t max_length, int bits, int dtype) {
  int64_t most = columns * block;
  if (window && window < most) most = window;
  if (max_length >= 0 && max_length < most) most = max_length;
  const int64_t each = G * ((H / G + kCols - 1) / kCols), tile = tile_of(bits, D, dtype), tiles = (most + tile - 1) / tile;
  if (tiles <= 2 * kWaves || (R * each >= 512 && tiles <= 8 * kWaves)) return 0;
  const int64_t n = (kWorkgroups + each - 1) / each;
  return n < 1 ? 1 : n;
}
int64_t plan_bytes(int64_t R) { return ((R + 1) * 4 + 255) / 256 * 256; }

template <int DT, int FMT, int D, int HP>
void launch_heads(const DecodeArgs& a, bool runs, unsigned grid, hipStream_t st) {
  // for blocks that runs of 16 positions straddle, a form off the main path, four heads or sixteen are kernels enough
  constexpr int kOdd = HP == 4 ? 4 : 16;
  if (runs) hipLaunchKernelGGL((decode_attention_kernel<DT, FMT, D, HP, true>), dim3(grid), dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((decode_attention_kernel<DT, FMT, D, kOdd, false>), dim3(grid), dim3(kThreads), 0, st, a);
}
template <int DT, int FMT, int D>
void launch(const DecodeArgs& a, unsigned grid, hipStream_t st) {
  const bool runs = a.block.d % 16 == 0;
  if (a.rep <= 4 && FMT != k16) launch_heads<DT, FMT, D, FMT == k16 ? 8 : 4>(a, runs, grid, st);
  else if (a.rep <= 8) launch_heads<DT, FMT, D, 8>(a, runs, grid, st);
  else launch_heads<DT, FMT, D, 16>(a, runs, grid, st);
  if (a.target) hipLaunchKernelGGL((decode_join_kernel<DT, D>), dim3(a.R * a.H), dim3(kThreads), 0, st, a);
}
template <int DT, int FMT>
void launch_dim(const DecodeArgs& a, int64_t D, unsigned grid, hipStream_t st) {
  if (D == 64) launch<DT, FMT, 64>(a, grid, st);
  else if (D == 128) launch<DT, FMT, 128>(a, grid, st);
  else launch<DT, FMT, 256>(a, grid, st);
}
template <int DT>
void launch_bits(const DecodeArgs& a, int bits, int64_t D, unsigned grid, hipStream_t st) {
  if (bits == 16) launch_dim<DT, k16>(a, D, grid, st);
  else if (bits == 8) launch_dim<DT, kFp8>(a, D, grid, st);
  else launch_dim<DT, kFp4>(a, D, grid, st);
}

}  // namespace
}  // namespace yh

extern "C" int64_t yh_decode_attention_workspace_bytes(int64_t n_seqs, int64_t H, int64_t G, int64_t D, int64_t block,
                                                       int64_t columns, int64_t window, int64_t max_length, int bits,
                                                       int dtype) {
  using namespace yh;
  if (n_seqs <= 0 || G <= 0 || H < G || D <= 0 || block <= 0 || columns <= 0 || columns >= (1ll << 31) ||
      block >= (1ll << 31) || (bits != 4 && bits != 8 && bits != 16))
    return 0;
  const int64_t target = target_for(n_seqs, H, G, D, block, columns, window, max_length, bits, dtype);
  return target ? plan_bytes(n_seqs) + (n_seqs + target) * H * (D * 4 + 8) : 0;
}

extern "C" int yh_decode_attention(const void* q, int64_t q_stride, const void* keys, const void* values,
                                   const uint8_t* key_scales, const uint8_t* value_scales, const int32_t* tables,
                                   const int64_t* lengths, const int64_t* starts, const float* slopes,
                                   const void* gate, int64_t gate_token_stride, int64_t gate_head_stride, void* out,
                                   int64_t n_seqs, int64_t blocks, int64_t columns, int64_t H, int64_t G, int64_t D,
                                   int64_t block, int64_t window, int64_t max_length, float scale, float softcap,
                                   int bits, int dtype, void* workspace, int64_t workspace_bytes, yh_stream_t stream) {
  using namespace yh;
  YH_CHECK_ARG(n_seqs >= 0 && blocks >= 0 && columns > 0 && H > 0 && G > 0 && H % G == 0 && block > 0 && window >= 0,
               "decode_attention: bad sizes");
  YH_CHECK_ARG(D == 64 || D == 128 || D == 256, "decode_attention: head dim must be 64, 128 or 256");
  YH_CHECK_ARG(bits == 4 || bits == 8 || bits == 16, "decode_attention: a cache holds 4, 8 or 16 bits a value");
  YH_CHECK_ARG(scale > 0.f && scale < INFINITY, "decode_attention: scale must be positive");
  YH_CHECK_ARG(softcap == 0.f || (softcap >= 1e-30f && softcap <= 1e30f),
               "decode_attention: softcap must be 1e-30 to 1e30, or 0 for none");
  if (dtype != YH_BF16 && dtype != YH_F16) {
    set_error("decode_attention: dtype must be bf16 or fp16");
    return YH_ERR_UNSUPPORTED;
  }
  if (n_seqs == 0) return YH_OK;
  YH_CHECK_ARG(q && out && lengths && tables && ((keys && values) || blocks == 0), "decode_attention: null pointer");
  YH_CHECK_ARG(bits == 16 || blocks == 0 || (key_scales && value_scales), "decode_attention: a quantised cache needs its scales");
  YH_CHECK_ARG(tree::aligned16(q) && tree::aligned16(out) && tree::aligned16(keys) && tree::aligned16(values) &&
                   (block % 16 || (tree::aligned16(key_scales) && tree::aligned16(value_scales))),
               "decode_attention: tensors must be 16-byte aligned");
  YH_CHECK_ARG(q_stride % 8 == 0 && q_stride >= H * D, "decode_attention: the token stride must hold whole heads and keep 16-byte rows");
  YH_CHECK_ARG(!gate || (gate_head_stride >= D && gate_token_stride >= H * gate_head_stride),
               "decode_attention: bad gate strides");
  const int64_t each = G * ((H / G + kCols - 1) / kCols);
  YH_CHECK_ARG(n_seqs < (1ll << 20) && columns < (1ll << 31) && block < (1ll << 31) && H < (1ll << 16) &&
                   blocks < (1ll << 31) && blocks * block < (1ll << 40) && (bits == 16 || D / kRun * block < (1ll << 32)),
               "decode_attention: sizes too large");
  const int64_t target = target_for(n_seqs, H, G, D, block, columns, window, max_length, bits, dtype);
  int64_t most = columns * block;
  if (window && window < most) most = window;
  if (most > (1ll << 31)) most = 1ll << 31;      // positions are below
  YH_CHECK_ARG(n_seqs * (most / 16 + 2) < (1ll << 31), "decode_attention: sizes too large");
  const int64_t grid = (n_seqs + target) * each;
  YH_CHECK_ARG(grid < (1ll << 24) && n_seqs * H < (1ll << 24), "decode_attention: sizes too large");
  const int64_t need = yh_decode_attention_workspace_bytes(n_seqs, H, G, D, block, columns, window, max_length,
                                                            bits, dtype);
  YH_CHECK_ARG(need == 0 || (workspace && tree::aligned16(workspace) && workspace_bytes >= need),
               "decode_attention: workspace too small");
  DecodeArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_ts = q_stride;
  a.keys = static_cast<const char*>(keys);
  a.values = static_cast<const char*>(values);
  a.key_scales = key_scales;
  a.value_scales = value_scales;
  a.tables = tables;
  a.lengths = lengths;
  a.starts = starts;
  a.slopes = slopes;
  a.gate = static_cast<const uint16_t*>(gate);
  a.g_ts = gate_token_stride;
  a.g_hs = gate_head_stride;
  a.out = static_cast<uint16_t*>(out);
  a.window = window;
  a.scale = scale;
  a.cap = softcap;
  a.block = tree::make_div(static_cast<uint32_t>(block));
  a.columns = tree::make_div(static_cast<uint32_t>(columns));
  a.R = static_cast<int>(n_seqs);
  a.H = static_cast<int>(H);
  a.G = static_cast<int>(G);
  a.rep = static_cast<int>(H / G);
  a.mtiles = (a.rep + kCols - 1) / kCols;
  a.blocks = static_cast<int>(blocks);
  a.target = static_cast<int>(target);
  if (need) {
    a.first = static_cast<int32_t*>(workspace);
    char* sums = static_cast<char*>(workspace) + plan_bytes(n_seqs);
    a.part = reinterpret_cast<float*>(sums);
    a.stat = reinterpret_cast<float2*>(sums + (n_seqs + target) * H * D * 4);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == YH_BF16) launch_bits<YH_BF16>(a, bits, D, static_cast<unsigned>(grid), st);
  else launch_bits<YH_F16>(a, bits, D, static_cast<unsigned>(grid), st);
  YH_CHECK_LAUNCH("decode_attention");
  return YH_OK;
}
