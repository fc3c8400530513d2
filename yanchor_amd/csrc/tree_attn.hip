// Attention of drafted trees over a block cache.
//
// A request's nodes i (at most 64) sit at position L + depth(i), L the tokens in
// its cache.  Node i sees the cached positions p < L that its window reaches and
// its own ancestors, itself included, among the nodes:
//   s_ij = q_i . k_j / sqrt(D);  out_i = sum_j softmax_j(s_i)_j v_j (* sigmoid(gate_i))
// Position p of request r is row p % block of cache block
// tables[r][p / block % columns], so the last columns * block positions are
// there; a ring is a table of one column whose block is the ring.
//
// A workgroup of NW waves (2, 4 or 8, as the rows need) takes a request, a KV
// head and 32 NW of the rows (node, query head of the group): the waves, 32 rows
// each, share 64-key tiles (attn_tile.h) that begin at multiples of 64
// positions; the nodes themselves are the last tile, its mask the ancestor sets.
//
// Requests are few or of very different lengths, so the tiles of an item
// (request, rows, head) are cut into parts of about one size (`chunk`, about
// kParts parts a workgroup that fits the chip): every workgroup finds its part
// from the lengths by itself, parts of a cut item leave their unnormalised sums
// with their maximum, and a second launch joins them in order.
//
// Few rows are bound by HBM, which the copies of four workgroups a CU keep at
// 5.1 to 5.6 TB/s (128 rings of 1024 slots, a third of them not full: 478 MB in
// 91 us; 64 block tables: 732 MB in 131 us).  256 rows and more a KV head are bound
// by the tiles' products and softmax: 516 GFLOP in 724 to 771 us from run to run,
// 0.7 PFLOP/s; the copies alone take 376 of 745, the products alone 549.
#include <type_traits>

#include "attn_tile.h"
#include "tree.h"

namespace yh {
namespace {

using tree::Div;

struct TreeArgs {
  const uint16_t* q;       // [N, H, D], tokens q_ts apart
  const uint16_t* k;       // [N, G, D]
  const uint16_t* v;
  int64_t q_ts, k_ts, v_ts;
  const int32_t* parents;  // [N] or null: chains
  const int32_t* cu;       // [R + 1]
  const int64_t* lengths;  // [R]
  const uint16_t* keys;    // [NB, G, block, D]
  const uint16_t* values;
  const int32_t* tables;   // [R, columns]
  const uint16_t* gate;    // [N, H, D] or null
  int64_t g_ts, g_hs;
  uint16_t* out;           // [N, H, D]
  int64_t total, window;   // window 0: none
  Div block, columns, rep;
  int R, H, G, NB, max_nodes, mtiles;
  int gate8;               // gate rows keep 8-byte alignment
  float scale;
  unsigned clear;          // workgroups at the end of the grid that clear the rows of no request
  // the cut: parts aimed at, and for requests [0, R] the first part, the first partial sum
  int target, slot_rows;   // target 0: no item is cut
  int32_t* first;          // [R + 1]
  int32_t* slot;           // [R + 1]
  float* part;             // [slots, slot_rows, D]
  float2* stat;            // [slots, slot_rows]: maximum (log2), denominator
};

constexpr int kMinChunk = 2;   // tiles a part at least (but for short items)

// What a request asks for: rows, and the positions [lo, L) of its cache that
// some node sees, in tiles from `base`.
struct Geometry {
  tree::Span span;
  int64_t length;
  int n, lo, L, base, ctx;
};
__device__ __forceinline__ Geometry geometry(const TreeArgs& a, const tree::Span& span, int64_t length) {
  Geometry q;
  q.span = span;
  q.n = static_cast<int>(span.count < a.max_nodes ? span.count : a.max_nodes);
  q.length = length < 0 ? 0 : length;
  const int64_t room = static_cast<int64_t>(a.columns.d) * a.block.d;
  int64_t oldest = q.length - room;
  if (a.window && q.length - a.window + 1 > oldest) oldest = q.length - a.window + 1;
  oldest = oldest < 0 ? 0 : oldest > q.length ? q.length : oldest;
  constexpr int64_t kEnd = (1ll << 31) - 4096;   // a window of tiles past it still fits an int
  q.lo = static_cast<int>(oldest < kEnd ? oldest : kEnd);
  q.L = static_cast<int>(q.length < kEnd ? q.length : kEnd);
  q.base = q.lo & ~(attn::kTile - 1);
  q.ctx = q.L > q.lo ? (q.L - q.base + attn::kTile - 1) / attn::kTile : 0;
  return q;
}

// Four rows of zeros for those that do not exist.
__device__ const uint4 zero_rows[4 * attn::kD / 8] = {};

// attn::copy16 from a scalar address plus a lane's offset, past the caches: a
// cache row is read once.
__device__ __forceinline__ void copy_run(const uint16_t* src, int voff, const void* lds) {
  const unsigned m0v = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(reinterpret_cast<uintptr_t>(lds)));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(m0v), "v"(voff), "s"(src)
               : "memory", "m0");
}

// A part: tiles [t0, t1) of an item, its partial sum's place (-1: the item is whole).
struct Part {
  int64_t first, count, length;
  int r, mt, g, t0, t1, slot;
};

template <int TH>
__device__ __forceinline__ int64_t block_sum(int64_t x, int64_t* before) {   // total, and the sum of earlier threads
  __shared__ int64_t sums[TH / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int64_t incl = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t y = __shfl_up(incl, off, 64);
    if (lane >= off) incl += y;
  }
  if (lane == 63) sums[w] = incl;
  __syncthreads();
  int64_t all = 0, early = 0;
#pragma unroll
  for (int i = 0; i < TH / 64; ++i) {
    early += i < w ? sums[i] : 0;
    all += sums[i];
  }
  __syncthreads();
  *before = early + incl - x;
  return all;
}

// Part `id` of the call, false if there are not so many.  An item of T tiles is
// cut into ceil(T / chunk) parts; chunk is at least the mean (all tiles / target),
// so there are at most target + items parts, and, two and more being at most
// 2 T / chunk, at most 2 target that leave partial sums.
template <int NW>
__device__ __forceinline__ bool find_part(const TreeArgs& a, int64_t id, Part* out) {
  constexpr int TH = NW * 64, kM = NW * attn::kRows;
  __shared__ Part found;
  const int tid = threadIdx.x;
  Geometry geo{};
  if (a.target == 0) {   // every item whole, one a workgroup
    const int g = static_cast<int>(id % a.G), mt = static_cast<int>(id / a.G % a.mtiles), r = static_cast<int>(id / a.G / a.mtiles);
    if (r >= a.R) return false;
    geo = geometry(a, tree::span_of(a.cu, r, a.total), a.lengths[r]);
    *out = Part{geo.span.first, geo.span.count, geo.length, r, mt, g, 0, geo.ctx + 1, -1};
    return mt * kM < geo.n * static_cast<int>(a.rep.d);
  }
  auto shape = [&](int64_t r, int64_t* items, int* tiles) {
    *items = 0;
    *tiles = 1;
    if (r >= a.R) return;
    geo = geometry(a, tree::span_of(a.cu, r, a.total), a.lengths[r]);
    *items = static_cast<int64_t>((geo.n * static_cast<int>(a.rep.d) + kM - 1) / kM) * a.G;
    *tiles = geo.ctx + 1;
  };
  int64_t units = 0, before, items = 0;
  int tiles = 1;
  for (int64_t r = tid; r - tid < a.R; r += TH) {
    shape(r, &items, &tiles);
    units += block_sum<TH>(items * tiles, &before);
  }
  // The longest part decides: of sizes from the mean on, the first that gives at
  // most `target` parts (more items than that: 1.5 times the mean).
  constexpr int kSizes = 8;
  constexpr float kSize[kSizes] = {1.f, 1.06f, 1.12f, 1.2f, 1.28f, 1.36f, 1.45f, 1.5f};
  const float mean = fmaxf(static_cast<float>(units) / a.target, kMinChunk);
  float guess[kSizes] = {};
  for (int64_t r = tid; r - tid < a.R; r += TH) {
    if (a.R > TH) shape(r, &items, &tiles);   // otherwise the first loop's
#pragma unroll
    for (int i = 0; i < kSizes; ++i) guess[i] += items * ceilf(tiles / ceilf(mean * kSize[i]));
  }
  int pick = kSizes - 1;
#pragma unroll
  for (int i = 0; i < kSizes; ++i) guess[i] = wave_sum(guess[i]);
  __shared__ float guesses[NW][kSizes];
  if ((tid & 63) == 0)
#pragma unroll
    for (int i = 0; i < kSizes; ++i) guesses[tid >> 6][i] = guess[i];
  __syncthreads();
#pragma unroll
  for (int i = kSizes - 1; i >= 0; --i) {
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) all += guesses[w][i];
    if (all <= a.target) pick = i;
  }
  const int64_t chunk = static_cast<int64_t>(ceilf(mean * kSize[pick]));
  int64_t parts = 0, cut = 0;
  if (tid == 0) found.r = -1;
  for (int64_t r = tid; r - tid < a.R; r += TH) {
    if (a.R > TH) shape(r, &items, &tiles);
    const int64_t p = (tiles + chunk - 1) / chunk, mine = items * p;
    int64_t first, slot;
    const int64_t all = block_sum<TH>(mine, &first), all_cut = block_sum<TH>(p > 1 ? mine : 0, &slot);
    first += parts;
    slot += cut;
    if (r < a.R) {
      if (id == 0) {
        a.first[r] = static_cast<int32_t>(first);
        a.slot[r] = static_cast<int32_t>(slot);
        if (r == a.R - 1) a.first[a.R] = static_cast<int32_t>(first + mine);
      }
      if (id >= first && id < first + mine) {
        const int64_t in = id - first, item = in / p, j = in - item * p;
        found = Part{geo.span.first, geo.span.count, geo.length, static_cast<int>(r), static_cast<int>(item / a.G),
                     static_cast<int>(item % a.G), static_cast<int>(j * tiles / p), static_cast<int>((j + 1) * tiles / p),
                     p > 1 ? static_cast<int>(slot + in) : -1};
      }
    }
    parts += all;
    cut += all_cut;
  }
  __syncthreads();
  *out = found;
  return found.r >= 0;
}

// read * sigmoid(gate) and the rounding to 16 bits of 4 outputs of dims dim .. dim + 3
template <int DT>
__device__ __forceinline__ void put4(const TreeArgs& a, int64_t row, int head, int dim, int D, float4 o) {
  using M = attn::Mfma<DT>;
  if (a.gate) {
    const uint16_t* gate = a.gate + row * a.g_ts + head * a.g_hs + dim;
    uint16_t x[4];
    if (a.gate8) {
      const uint2 y = *reinterpret_cast<const uint2*>(gate);
      x[0] = y.x & 0xffff;
      x[1] = y.x >> 16;
      x[2] = y.y & 0xffff;
      x[3] = y.y >> 16;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = gate[e];
    }
    o.x *= 1.f / (1.f + __expf(-M::widen(x[0])));
    o.y *= 1.f / (1.f + __expf(-M::widen(x[1])));
    o.z *= 1.f / (1.f + __expf(-M::widen(x[2])));
    o.w *= 1.f / (1.f + __expf(-M::widen(x[3])));
  }
  *reinterpret_cast<uint2*>(a.out + (row * a.H + head) * D + dim) = make_uint2(M::round2(o.x, o.y), M::round2(o.z, o.w));
}

// The pipeline: keys and values of tile after tile pass through S slots of LDS,
// one barrier a slot: at step q (the keys, then the values of a tile) slot q has
// arrived, q - 1 is consumed, and its place is filled again, so that S - 2 to
// S - 1 slots are in flight.  S fills the LDS that the workgroups of a CU leave:
// 2 waves 2 slots (four workgroups), 4 waves 4 (two), 8 waves 8 (one).  (2 waves
// with 3 slots, three workgroups a CU: 134 us for 122 in the 128 rings.)
//
// With blocks of whole fours of rows (RUNS) the addresses are scalars: lane l
// holds where the rows 4 l .. 4 l + 3 of a window of four tiles lie, from block
// ids that come through LDS as the copies do, a window ahead (a load into
// registers would have its wait drain the copies).  Resolved row by row in every
// tile instead: 767 us for 746 at 8 long contexts.
//
// Other blocks (not RUNS) load their ids into registers in every tile, whose wait
// drains the copies in flight, and with D = 128 spill 11 to 26 vector registers:
// 64 block tables of blocks of 15 take 430 us, of 16 142; 8 long contexts in blocks
// of one token 1909, of 64 768.
template <int NW>
struct Pipe {
  static constexpr int S = NW == 8 ? 8 : NW == 4 ? 4 : 2;
  static constexpr int kCopies = 16 / NW;                // a wave's copies of a slot
  static constexpr int kWait = (S - 2) * kCopies;        // younger than slot q's at step q, at least
  static constexpr bool kEarly = S <= 4;                 // refill before the products: few slots
};
template <int N>
__device__ __forceinline__ void copies_left() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void copy4(const int32_t* src, const void* lds) {   // 4 bytes a lane
  const unsigned m0v = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(reinterpret_cast<uintptr_t>(lds)));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(m0v), "v"(src) : "memory", "m0");
}

template <int DT, int D, int NW, bool RUNS>
__global__ void __launch_bounds__(NW * 64, 2) tree_attention_kernel(TreeArgs a) {
  constexpr int kM = NW * attn::kRows;   // rows of the workgroup
  using P = Pipe<NW>;
  constexpr int S = P::S;
  __shared__ attn::Rows stage[S];
  __shared__ int32_t ids[2][NW][64];
  __shared__ uint64_t s_set[tree::kNodes];
  __shared__ int s_deep;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  if (blockIdx.x >= gridDim.x - a.clear) {   // rows of no request
    tree::clear_rows<NW * 64>(a.out, a.cu, a.R, a.total, static_cast<int64_t>(a.H) * D * 2,
                              blockIdx.x - (gridDim.x - a.clear), a.clear);
    return;
  }
  Part part;
  if (!find_part<NW>(a, blockIdx.x, &part)) return;
  const int g = __builtin_amdgcn_readfirstlane(part.g), mt = __builtin_amdgcn_readfirstlane(part.mt),
            r = __builtin_amdgcn_readfirstlane(part.r);
  const Geometry geo = geometry(a, tree::Span{part.first, part.count}, part.length);
  const tree::Span span = geo.span;
  const int n = geo.n, rep = a.rep.d;
  const int lo = geo.lo, L = geo.L, base = geo.base, ctx = geo.ctx, tiles = part.t1;
  if (mt == 0 && part.t0 == 0) {   // nodes past the most that the call takes: not a number
    const int64_t first = span.first + n, row = static_cast<int64_t>(a.H) * D;
    for (int64_t i = threadIdx.x; i < (span.count - n) * rep * D; i += NW * 64) {
      const int64_t t = i / (rep * D);
      a.out[(first + t) * row + static_cast<int64_t>(g) * rep * D + (i - t * rep * D)] = DT == YH_BF16 ? 0x7fc0 : 0x7e00;
    }
  }

  // this lane's query: row m of the request's (node, head of the group) rows
  const int m = mt * kM + w * attn::kRows + (lane & 31);
  const bool active = mt * kM + w * attn::kRows < n * rep;   // of the wave
  const bool mine = m < n * rep;
  const int node = mine ? a.rep.quot(m) : 0, head = g * rep + (mine ? m - node * rep : 0);
  const int64_t W = a.window ? a.window : (1ll << 40);
  const float k2 = a.scale * 1.4426950408889634f;
  const int32_t* table = a.tables + static_cast<int64_t>(r) * a.columns.d;
  // where position p is in the cache, -1: nowhere (the id may be a row's of a window that is not all there)
  auto entry = [&](int p) {
    const uint32_t qd = a.block.quot(p >= lo && p < L ? p : lo);
    return table + (qd - a.columns.quot(qd) * a.columns.d);
  };
  auto row_at = [&](int p, int id) {
    const int in = p - static_cast<int>(a.block.quot(p) * a.block.d);
    return id >= 0 && id < a.NB ? (id * a.G + g) * static_cast<int>(a.block.d) + in : -1;
  };
  // RUNS: window j holds tiles 4 j .. 4 j + 3 from `base`; a four is there if its
  // block is (rows of it outside [lo, L) are copied too, and masked)
  auto four = [&](int j) { return base + 256 * j + 4 * lane; };
  auto fetch = [&](int j) {
    if constexpr (RUNS) {   // any of the four's positions in [lo, L) names the block
      const int p = four(j);
      copy4(entry(p < lo ? p + 3 : p), ids[j & 1][w]);
    }
  };
  int fours = -1;                       // the lane's four of the window being copied
  uint64_t there_now = 0, there_next = 0;   // the fours that are there, of the window at hand and of the next
  auto open_window = [&](int j) {       // its ids have arrived
    const int p = four(j);
    fours = p + 3 >= lo && p < L ? row_at(p, ids[j & 1][w][lane]) : -1;
    there_next = __ballot(fours >= 0);
  };
  auto copy_slot = [&](int t, int slot, bool values) {
    attn::Rows& to = stage[slot];
    if (t >= ctx) {   // the nodes; rows past them repeat the last and are masked
      const int64_t ts = values ? a.v_ts : a.k_ts;
      const uint16_t* src = (values ? a.v : a.k) + span.first * ts + static_cast<int64_t>(g) * D;
      attn::load_rows<NW>(to, [&](int rr, int e, const void* l) {
        if (D == attn::kD || e < D) attn::copy16(src + min(rr, n - 1) * ts + e, l);
      });
      return;
    }
    const uint16_t* src = values ? a.values : a.keys;
    if constexpr (RUNS) {
#pragma unroll
      for (int it = 0; it < 16 / NW; ++it) {
        const int row = __builtin_amdgcn_readlane(fours, 16 * (t & 3) + it * NW + w);
        const uint16_t* from = row < 0 ? reinterpret_cast<const uint16_t*>(zero_rows) : src + static_cast<int64_t>(row) * D;
        // the lane's piece of the four rows (load_rows' order)
        const int piece = (lane & 15) ^ (((lane >> 4) << 2) | ((it * NW + w) & 3));
        if (D == attn::kD || piece < D / 8) copy_run(from, ((lane >> 4) * D + piece * 8) * 2, &to[64 * (it * NW + w)]);
      }
    } else {
      const int p0 = base + t * attn::kTile;
      attn::load_rows<NW>(to, [&](int rr, int e, const void* l) {
        const int p = p0 + rr, row = p >= lo && p < L ? row_at(p, *entry(p)) : -1;
        const uint16_t* from = row < 0 ? reinterpret_cast<const uint16_t*>(zero_rows) : src + static_cast<int64_t>(row) * D;
        if (D == attn::kD || e < D) attn::copy16(from + e, l);
      });
    }
  };

  // slot q: the keys (even q) or the values of tile part.t0 + q / 2
  const int t0 = part.t0, slots = 2 * (tiles - t0);
  auto issue = [&](int q) {
    if (q >= slots) return;
    const int t = t0 + (q >> 1);
    if constexpr (RUNS)
      if ((q & 1) == 0 && t < ctx && ((t & 3) == 0 || q == 0)) {
        open_window(t >> 2);
        if (q) fetch((t >> 2) + 1);   // arrives with the keys of tile t, 8 slots before it is opened
      }
    copy_slot(t, q % S, (q & 1) != 0);
  };
  // the keys of tile t that are there, a bit a row
  auto rows_there = [&](int t) -> uint64_t {
    const int p0 = base + t * attn::kTile;
    if constexpr (RUNS) {
      uint64_t m = (there_now >> (16 * (t & 3))) & 0xffffull;   // every bit to four
      m = (m | m << 24) & 0x000000ff000000ffull;
      m = (m | m << 12) & 0x000f000f000f000full;
      m = (m | m << 6) & 0x0303030303030303ull;
      m = (m | m << 3) & 0x1111111111111111ull;
      m *= 15;
      const int head = min(max(lo - p0, 0), 63), tail = min(max(p0 + 63 - (L - 1), 0), 63);
      return m & (~0ull << head) & (~0ull >> tail);
    } else {
      const int p = p0 + lane;
      return __ballot(p >= lo && p < L && row_at(p, *entry(p)) >= 0);
    }
  };
  // The block ids, the queries and the parents together, then the first slots;
  // the masks are formed while they arrive.
  fetch(t0 >> 2);
  fetch((t0 >> 2) + 1);   // the first window may be short
  attn::State<DT, false, D> st;
  st.init(false);
  st.load_q(a.q + (span.first + node) * a.q_ts + static_cast<int64_t>(head) * D, mine);
  int up = -1;
  if (w == 0 && lane < n) up = a.parents ? a.parents[span.first + lane] : lane - 1;
  // as a builtin, so that the compiler counts the queries as loaded too and waits for none in the loop
  __builtin_amdgcn_s_waitcnt(0x0F70);
  asm volatile("" ::: "memory");
  issue(0);
  there_now = there_next;
#pragma unroll
  for (int q = 1; q < S - 1; ++q) issue(q);
  if (w == 0) {
    const uint64_t set = tree::ancestors_of(up);
    s_set[lane] = set;
    int d = lane < n ? __popcll(set) - 1 : 0;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) d = max(d, __shfl_xor(d, off, 64));
    if (lane == 0) s_deep = d;
  }
  attn::tile_barrier();
  const int deep = s_deep;
  uint64_t see = mine ? s_set[node] : 0;
  const int depth = mine ? __popcll(see) - 1 : 0;
  for (int far = depth + 1; far > W; --far) see &= see - 1;   // ancestors past the window: the earliest nodes of the path
  // the first position that this lane's query sees, and the wave's rows' earliest
  const int from = static_cast<int>(min(max(geo.length + depth - W + 1, static_cast<int64_t>(0)), (1ll << 31) - 1));
  int wfrom = mine ? from : 0x7fffffff, wto = mine ? from : 0;   // (and the latest such)
  uint64_t wsee = see;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    wfrom = min(wfrom, __shfl_xor(wfrom, off, 64));
    wto = max(wto, __shfl_xor(wto, off, 64));
    wsee |= __shfl_xor(wsee, off, 64);
  }
  const int64_t allfrom = geo.length + deep - W + 1;   // from here on every node sees
  int t = t0, q = 0;
  auto arrive = [&]() {   // slot q is there for all waves, and q - 1 consumed by them
    if (q + S - 2 < slots) copies_left<P::kWait>();
    else copies_left<0>();
    attn::tile_barrier();
    if constexpr (P::kEarly) issue(q + S - 1);
  };
  auto inner = [&]() {
    const int p0 = base + t * attn::kTile;
    if constexpr (RUNS)
      return t < ctx && p0 >= lo && p0 + attn::kTile <= L && p0 >= allfrom && ((there_now >> (16 * (t & 3))) & 0xffff) == 0xffff;
    else
      return false;
  };
  auto tile = [&](auto edge) {
    attn::f32x16 c[2];
    uint64_t there = 0;
    arrive();
    if (active) st.scores(stage[q % S], c);
    if constexpr (!P::kEarly) issue(q + S - 1);
    const int p0 = base + t * attn::kTile;
    if constexpr (edge.value) {
      there = t < ctx ? rows_there(t) : 0;
      if (active) {
        const int skip = min(max(from - p0, 0), 64);
        const uint64_t live = t < ctx ? (skip > 63 ? 0 : there & (~0ull << skip)) : see;   // keys that the lane's query sees
        const uint64_t sh = live >> (4 * (lane >> 5));
        st.mask(c, [&](int key, int) { return ((key < 32 ? static_cast<uint32_t>(sh) >> key : static_cast<uint32_t>(sh >> 32) >> (key - 32)) & 1) != 0; });
      }
    }
    ++q;
    arrive();
    if (active) {
      uint64_t keep = ~0ull;
      if constexpr (edge.value) {
        const int wskip = min(max(wfrom - p0, 0), 64);
        keep = t < ctx ? (wskip > 63 ? 0 : there & (~0ull << wskip)) : wsee;
      }
      // The weights enter the product rounded to the type's 16 bits, as in the window prefill: eps / 2 of each
      // (sum p |v| eps / 2, as much as the output's own rounding where values have one sign).  As hi + lo pairs
      // they take a second matrix instruction: 8 long contexts 950 us for 768, 128 rings 105 for 97.
      st.template step<false, edge.value, true>(c, stage[q % S], k2, keep);
    }
    if constexpr (!P::kEarly) issue(q + S - 1);
    ++q;
    ++t;
    if ((t & 3) == 0) there_now = there_next;
  };
  // Tiles whose keys all rows see and the others take a loop each: as branches
  // of one loop the RUNS kernels spill vector registers too (the waves' conditions may differ: both loops pass
  // two barriers a tile).
  while (t < tiles) {
#pragma unroll 1
    while (t < tiles && inner()) tile(std::false_type{});
#pragma unroll 1
    while (t < tiles && !inner()) tile(std::true_type{});
  }
  // A value that is not finite reaches, through its weights of 0, the queries of
  // the wave that do not see it, where the part holds keys that only some of them
  // see.  Then its rows are computed again one by one without such products, a
  // lane a key for the scores: some 30 times slower.  (Taking such rows out of the
  // tiles they are in would cost every call 4 %.)
  float mark = st.den;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) mark = fmaf(st.acc[d][i], 0.f, mark);
  const bool mixed = (tiles > ctx && n > 1) ||
                     (wto > wfrom && base + t0 * attn::kTile < wto && base + min(tiles, ctx) * attn::kTile > wfrom);
  if (mixed && __any(mine && !(fabsf(mark) < INFINITY))) {
    constexpr int kOwn = D / 64;   // dims of a lane
    using M = attn::Mfma<DT>;
    typedef uint16_t own_t __attribute__((ext_vector_type(kOwn)));
#pragma unroll 1
    for (int i = 0; i < attn::kRows; ++i) {
      const int mi = mt * kM + w * attn::kRows + i;
      if (mi >= n * rep) break;
      const int nd = a.rep.quot(mi), hd = g * rep + (mi - nd * rep), first = __shfl(from, i, 64);
      const uint64_t sees = __shfl(see, i, 64);
      const uint4* qr = reinterpret_cast<const uint4*>(a.q + (span.first + nd) * a.q_ts + static_cast<int64_t>(hd) * D);
      float top = -3.0e38f, den = 0.f, o[kOwn] = {};
#pragma unroll 1
      for (int u = t0; u < tiles; ++u) {
        int64_t krow = -1, vrow = 0;   // the lane's key: elements from the start of its tensor
        if (u < ctx) {
          const int p = base + u * attn::kTile + lane;
          if (p >= lo && p < L && p >= first) {
            const int row = row_at(p, *entry(p));
            krow = vrow = row < 0 ? -1 : static_cast<int64_t>(row) * D;
          }
        } else if ((sees >> lane) & 1) {
          krow = (span.first + lane) * a.k_ts + static_cast<int64_t>(g) * D;
          vrow = (span.first + lane) * a.v_ts + static_cast<int64_t>(g) * D;
        }
        uint64_t live = __ballot(krow >= 0);
        if (live == 0) continue;
        float x = -INFINITY;
        if (krow >= 0) {
          const uint4* kr = reinterpret_cast<const uint4*>((u < ctx ? a.keys : a.k) + krow);
          x = 0.f;
#pragma unroll 4
          for (int e = 0; e < D / 8; ++e) {
            const uint4 y = kr[e], z = qr[e];
            const uint32_t ky[4] = {y.x, y.y, y.z, y.w}, qz[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              x = fmaf(M::widen(ky[j] & 0xffff), M::widen(qz[j] & 0xffff), fmaf(M::widen(ky[j] >> 16), M::widen(qz[j] >> 16), x));
          }
          x *= k2;
        }
        const float now = fmaxf(top, wave_max(x)), f = __builtin_amdgcn_exp2f(top - now);
        const float pr = krow >= 0 ? __builtin_amdgcn_exp2f(x - now) : 0.f;
        den = fmaf(den, f, wave_sum(pr));
        top = now;
#pragma unroll
        for (int e = 0; e < kOwn; ++e) o[e] *= f;
        const uint16_t* values = u < ctx ? a.values : a.v;
        for (; live; live &= live - 1) {
          const int key = __builtin_ctzll(live);
          const own_t y = *reinterpret_cast<const own_t*>(values + __shfl(vrow, key, 64) + lane * kOwn);
          const float pk = __shfl(pr, key, 64);
#pragma unroll
          for (int e = 0; e < kOwn; ++e) o[e] = fmaf(pk, M::widen(y[e]), o[e]);
        }
      }
      const int64_t token = span.first + nd, slot = static_cast<int64_t>(part.slot) * a.slot_rows + w * attn::kRows + i;
      if (part.slot >= 0 && lane == 0) a.stat[slot] = make_float2(top, den);
#pragma unroll
      for (int e = 0; e < kOwn; ++e) {
        const int dim = lane * kOwn + e;
        if (part.slot >= 0) {
          a.part[slot * D + dim] = o[e];
        } else {
          float x = o[e] / den;
          if (a.gate) x *= 1.f / (1.f + __expf(-M::widen(a.gate[token * a.g_ts + hd * a.g_hs + dim])));
          a.out[(token * a.H + hd) * D + dim] = M::round(x);
        }
      }
    }
    return;
  }
  if (!mine) return;

  const float den = st.den + __shfl_xor(st.den, 32, 64), inv = 1.f / den;
  const int64_t token = span.first + node;
  const int at = w * attn::kRows + (lane & 31), half4 = 4 * (lane >> 5);
  const int64_t slot = static_cast<int64_t>(part.slot) * a.slot_rows + at;
  if (part.slot >= 0 && lane < 32) a.stat[slot] = make_float2(st.base, den);
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int rr = 0; rr < 4; ++rr) {
      const int dim = 32 * d + 8 * rr + half4;
      const float4 o = make_float4(st.acc[d][4 * rr], st.acc[d][4 * rr + 1], st.acc[d][4 * rr + 2], st.acc[d][4 * rr + 3]);
      if (part.slot >= 0) *reinterpret_cast<float4*>(a.part + slot * D + dim) = o;
      else put4<DT>(a, token, head, dim, D, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    }
}

// The parts of the cut items joined in order, D / 4 lanes a row: the largest of
// their maxima, then the sums at its scale.
template <int DT, int D>
__global__ void __launch_bounds__(256) tree_join_kernel(TreeArgs a, int rows) {
  constexpr int kLanes = D / 4;
  const int g = blockIdx.x % a.G, mt = blockIdx.x / a.G % a.mtiles, r = blockIdx.x / a.G / a.mtiles;
  const tree::Span span = tree::span_of(a.cu, r, a.total);
  const int n = static_cast<int>(span.count < a.max_nodes ? span.count : a.max_nodes), rep = a.rep.d;
  const int items = (n * rep + rows - 1) / rows * a.G, all = a.first[r + 1] - a.first[r];
  if (all == items) return;   // not cut
  const int p = all / items, dim = 4 * (threadIdx.x % kLanes);
  const int64_t first = (static_cast<int64_t>(a.slot[r]) + static_cast<int64_t>(mt * a.G + g) * p) * a.slot_rows;
  for (int at = blockIdx.y * (256 / kLanes) + threadIdx.x / kLanes; at < rows; at += gridDim.y * (256 / kLanes)) {
    const int m = mt * rows + at;
    if (m >= n * rep) return;
    const int64_t slot = first + at;
    float top = -3.0e38f;
#pragma unroll 4
    for (int j = 0; j < p; ++j) top = fmaxf(top, a.stat[slot + static_cast<int64_t>(j) * a.slot_rows].x);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float den = 0.f;
#pragma unroll 4
    for (int j = 0; j < p; ++j) {
      const int64_t s = slot + static_cast<int64_t>(j) * a.slot_rows;
      const float2 st = a.stat[s];
      const float4 x = *reinterpret_cast<const float4*>(a.part + s * D + dim);
      const float f = __builtin_amdgcn_exp2f(st.x - top);
      den = fmaf(st.y, f, den);
      o.x = fmaf(x.x, f, o.x);
      o.y = fmaf(x.y, f, o.y);
      o.z = fmaf(x.z, f, o.z);
      o.w = fmaf(x.w, f, o.w);
    }
    const float inv = 1.f / den;
    const int node = a.rep.quot(m);
    put4<DT>(a, span.first + node, g * rep + (m - node * rep), dim, D,
             make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
  }
}

// Rows of a workgroup: 64 (two waves), 128 or 256.
int rows_of(int64_t max_nodes, int64_t rep) { return max_nodes * rep > 128 ? 256 : max_nodes * rep > 64 ? 128 : 64; }
// Parts aimed at: kParts for every workgroup that fits the chip (4, 2 or 1 a CU).
constexpr int kParts = 1;
int target_of(int rows) { return (rows == 64 ? 1024 : rows == 128 ? 512 : 256) * kParts; }
int64_t plan_bytes(int64_t n_seqs) { return (2 * (n_seqs + 1) * 4 + 255) / 256 * 256; }

template <int DT, int D, bool RUNS>
void launch_rows(const TreeArgs& a, int rows, unsigned grid, hipStream_t st) {
  if (rows == 256) hipLaunchKernelGGL((tree_attention_kernel<DT, D, 8, RUNS>), dim3(grid), dim3(512), 0, st, a);
  else if (rows == 128) hipLaunchKernelGGL((tree_attention_kernel<DT, D, 4, RUNS>), dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((tree_attention_kernel<DT, D, 2, RUNS>), dim3(grid), dim3(128), 0, st, a);
}

template <int DT, int D>
void launch(const TreeArgs& a, int rows, unsigned grid, hipStream_t st) {
  if (a.block.d % 4 == 0) launch_rows<DT, D, true>(a, rows, grid, st);
  else launch_rows<DT, D, false>(a, rows, grid, st);
  const int most = static_cast<int>(a.max_nodes * a.rep.d < static_cast<uint32_t>(rows) ? a.max_nodes * a.rep.d : rows);
  if (a.R == 0 || a.target == 0) return;
  // rows of an item: as many workgroups as 1024 of them need
  const int items = a.R * a.G * a.mtiles, per = 256 / (D / 4), all = (most + per - 1) / per, some = 1024 / items;
  hipLaunchKernelGGL((tree_join_kernel<DT, D>), dim3(items, all < some ? all : some < 1 ? 1 : some), dim3(256), 0, st, a,
                     rows);
}

// Parts aimed at, 0 where every item stays whole: as many of them as workgroups fit the chip, none longer than
// 32 tiles.  (128 rings of 1024 slots, 8 groups: the second launch is 5 us of 97.)
int64_t target_for(int64_t n_seqs, int64_t H, int64_t G, int64_t block, int64_t columns, int64_t window,
                   int64_t max_nodes, int64_t max_length) {
  const int rows = rows_of(max_nodes, H / G);
  const int64_t items = n_seqs * G * ((max_nodes * (H / G) + rows - 1) / rows), target = target_of(rows);
  int64_t most = columns * block;
  if (window && window - 1 < most) most = window - 1;
  if (max_length >= 0 && max_length < most) most = max_length;
  return items >= target && most <= 30 * attn::kTile ? 0 : target;
}

}  // namespace
}  // namespace yh

extern "C" int64_t yh_tree_attention_workspace_bytes(int64_t n_seqs, int64_t H, int64_t G, int64_t D, int64_t block,
                                                     int64_t columns, int64_t window, int64_t max_nodes,
                                                     int64_t max_length) {
  using namespace yh;
  if (n_seqs <= 0 || G <= 0 || H < G || D <= 0 || block <= 0 || columns <= 0 || columns >= (1ll << 31) ||
      block >= (1ll << 31) || max_nodes <= 0 || max_nodes > tree::kNodes)
    return 0;
  const int64_t rep = H / G, rows = rows_of(max_nodes, rep), used = max_nodes * rep < rows ? max_nodes * rep : rows;
  const int64_t slots = target_for(n_seqs, H, G, block, columns, window, max_nodes, max_length) * 2;
  return slots ? plan_bytes(n_seqs) + slots * used * (D * 4 + 8) : 0;
}

extern "C" int yh_tree_attention(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                                 int64_t v_stride, const int32_t* parents, const int32_t* cu_seqlens,
                                 const int64_t* lengths, const void* keys, const void* values, const int32_t* tables,
                                 const void* gate, int64_t gate_token_stride, int64_t gate_head_stride, void* out,
                                 int64_t n_seqs, int64_t total, int64_t blocks, int64_t columns, int64_t H, int64_t G,
                                 int64_t D, int64_t block, int64_t window, int64_t max_nodes, int64_t max_length,
                                 float scale, int dtype, void* workspace, int64_t workspace_bytes, yh_stream_t stream) {
  using namespace yh;
  YH_CHECK_ARG(n_seqs >= 0 && total >= 0 && blocks >= 0 && columns > 0 && H > 0 && G > 0 && H % G == 0 && block > 0 &&
                   window >= 0,
               "tree_attention: bad sizes");
  YH_CHECK_ARG(max_nodes > 0 && max_nodes <= tree::kNodes, "tree_attention: max_nodes must be 1 to %d", tree::kNodes);
  YH_CHECK_ARG(D == 64 || D == 128, "tree_attention: head dim must be 64 or 128");
  YH_CHECK_ARG(scale > 0.f && scale < INFINITY, "tree_attention: scale must be positive");
  if (dtype != YH_BF16 && dtype != YH_F16) {
    set_error("tree_attention: dtype must be bf16 or fp16");
    return YH_ERR_UNSUPPORTED;
  }
  if (total == 0) return YH_OK;
  YH_CHECK_ARG(q && k && v && out && ((cu_seqlens && lengths && tables) || n_seqs == 0) &&
                   ((keys && values) || blocks == 0),
               "tree_attention: null pointer");
  YH_CHECK_ARG(tree::aligned16(q) && tree::aligned16(k) && tree::aligned16(v) && tree::aligned16(out) &&
                   tree::aligned16(keys) && tree::aligned16(values),
               "tree_attention: tensors must be 16-byte aligned");
  YH_CHECK_ARG(q_stride % 8 == 0 && k_stride % 8 == 0 && v_stride % 8 == 0 && q_stride >= H * D &&
                   k_stride >= G * D && v_stride >= G * D,
               "tree_attention: token strides must hold whole heads and keep 16-byte rows");
  YH_CHECK_ARG(!gate || (gate_head_stride >= D && gate_token_stride >= H * gate_head_stride),
               "tree_attention: bad gate strides");
  YH_CHECK_ARG(total < (1ll << 31) && columns < (1ll << 31) && block < (1ll << 31) &&
                   H < (1ll << 20) && blocks < (1ll << 31) && block * G < (1ll << 31) && blocks * (G * block) < (1ll << 31),
               "tree_attention: sizes too large");
  const int64_t rep = H / G, rows = rows_of(max_nodes, rep), mtiles = (max_nodes * rep + rows - 1) / rows;
  const int64_t items = n_seqs * G * mtiles;
  const int64_t target = target_for(n_seqs, H, G, block, columns, window, max_nodes, max_length);
  const int64_t need = yh_tree_attention_workspace_bytes(n_seqs, H, G, D, block, columns, window, max_nodes, max_length);
  YH_CHECK_ARG(items < (1ll << 22), "tree_attention: sizes too large");
  YH_CHECK_ARG(need == 0 || (workspace && tree::aligned16(workspace) && workspace_bytes >= need),
               "tree_attention: workspace too small");
  const bool gate8 = gate && (reinterpret_cast<uintptr_t>(gate) & 7) == 0 && gate_token_stride % 4 == 0 &&
                     gate_head_stride % 4 == 0;
  TreeArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
             q_stride, k_stride, v_stride, parents, cu_seqlens, lengths, static_cast<const uint16_t*>(keys),
             static_cast<const uint16_t*>(values), tables, static_cast<const uint16_t*>(gate), gate_token_stride,
             gate_head_stride, static_cast<uint16_t*>(out), total, window,
             tree::make_div(static_cast<uint32_t>(block)), tree::make_div(static_cast<uint32_t>(columns)),
             tree::make_div(static_cast<uint32_t>(rep)), (int)n_seqs, (int)H, (int)G, (int)blocks, (int)max_nodes,
             (int)mtiles, gate8 ? 1 : 0, scale, static_cast<unsigned>(tree::clearing(total, H * D * 2)), (int)target, (int)(max_nodes * rep < rows ? max_nodes * rep : rows),
             nullptr, nullptr, nullptr, nullptr};
  if (need) {
    char* sums = static_cast<char*>(workspace) + plan_bytes(n_seqs);
    a.first = static_cast<int32_t*>(workspace);
    a.slot = a.first + n_seqs + 1;
    a.part = reinterpret_cast<float*>(sums);
    a.stat = reinterpret_cast<float2*>(sums + target * 2 * a.slot_rows * D * 4);
  }
  const unsigned grid = static_cast<unsigned>(target + items) + a.clear;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == YH_BF16) {
    if (D == 128) launch<YH_BF16, 128>(a, (int)rows, grid, st);
    else launch<YH_BF16, 64>(a, (int)rows, grid, st);
  } else {
    if (D == 128) launch<YH_F16, 128>(a, (int)rows, grid, st);
    else launch<YH_F16, 64>(a, (int)rows, grid, st);
  }
  YH_CHECK_LAUNCH("tree_attention");
  return YH_OK;
}
