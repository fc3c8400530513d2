// Block tables, slot maps and the cache write of a block cache: keys / values
// [blocks, G, block, D], request r's position p in row p % block of block
// tables[r][p / block % columns].  A ring is one block a request.
//
//   extend   blocks for the new tokens of every request off the top of a stack
//            of free block ids, and the cache slot of every new token
//   trim     the blocks past a shorter length back onto the stack
//   slots    the slots of the nodes of drafted trees: all, or the path to the
//            last accepted node
//   write    key / value rows into their slots
//
// The i-th block that a call hands out, in the order of requests and columns,
// is free[count - 1 - i], and trim puts its i-th block where the next extend
// takes it as the i-th again: the results do not depend on the order in which
// workgroups run, and trimming takes an extension back.
//
// The tables move a few bytes a request and are bound by latency (128 requests:
// extend 7.1 us, slots 3.7, trim 3.1 and 3.8), so launches are few: extend writes
// the slots in its one launch when the tokens are few, trim takes one launch for
// few requests with short tables.
#include "tree.h"

namespace yh {
namespace {

using tree::Div;
using tree::Span;

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;

// Block-wide exclusive scan of one int64 a thread; the total in *total.
__device__ __forceinline__ int64_t scan(int64_t x, int64_t* total) {
  __shared__ int64_t wsum[kWaves];
  const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
  int64_t incl = x;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int64_t y = __shfl_up(incl, off, kWave);
    if (lane >= off) incl += y;
  }
  if (lane == kWave - 1) wsum[w] = incl;
  __syncthreads();
  int64_t before = 0, all = 0;
  for (int i = 0; i < kWaves; ++i) {
    before += i < w ? wsum[i] : 0;
    all += wsum[i];
  }
  __syncthreads();
  *total = all;
  return before + incl - x;
}

constexpr int64_t kMaxLength = (1ll << 31) - 1;   // positions fit 31 bits

__device__ __forceinline__ int64_t clamp_length(int64_t x) { return x < 0 ? 0 : x > kMaxLength ? kMaxLength : x; }
__device__ __forceinline__ int32_t clamp_count(const int32_t* count, int64_t n) {
  const int32_t c = *count;
  return c < 0 ? 0 : c > n ? static_cast<int32_t>(n) : c;
}

// Columns in use at length x.
__device__ __forceinline__ int64_t used(int64_t x, int block, int columns, int wrap) {
  const int64_t n = (x + block - 1) / block;
  return wrap && n > columns ? columns : n;
}

// ---------------------------------------------------------------------------
struct ExtendArgs {
  const int64_t* lengths;   // [R] tokens already there
  const int32_t* cu;        // [R + 1] new tokens
  int32_t* tables;          // [R, columns]
  const int32_t* free;      // [n_free]
  int32_t* count;           // [1]
  int64_t* slots;           // [total]
  uint8_t* served;          // [R]
  int32_t* plan;            // [R + 1]: first block of each request in the call's order (-1: not served), free blocks before
  int64_t n_free, total;
  Div block, columns;
  int R, wrap;
};

// Position pos of a request that ends at `end`: a later one takes its row of a ring.
__device__ __forceinline__ bool passed(int64_t pos, int64_t end, const Div& block, const Div& columns) {
  return pos + static_cast<int64_t>(block.d) * columns.d < end;
}

// The slot of token i of n, given its request's share of the call (off < 0: none).
__device__ __forceinline__ int64_t token_slot(const ExtendArgs& a, int r, int64_t length, int64_t i, int64_t n,
                                              int32_t off, int32_t top) {
  const int64_t pos = length + i;
  if (off < 0 || pos > kMaxLength) return -1;
  const uint32_t q = a.block.quot(static_cast<uint32_t>(pos)), in = static_cast<uint32_t>(pos) - q * a.block.d;
  const uint32_t c = q - a.columns.quot(q) * a.columns.d;
  const int64_t held = used(length, a.block.d, a.columns.d, a.wrap);
  int32_t* row = a.tables + static_cast<int64_t>(r) * a.columns.d;
  int32_t id;
  if (c >= held) {   // a block of this call; its first token is always one of the call's
    const int64_t at = top - 1 - (off + (c - held));
    id = at >= 0 ? a.free[at] : -1;   // only offsets that fall lead below the stack
    if (in == 0 && q < a.columns.d) row[c] = id;
  } else {
    id = row[c];
  }
  return id < 0 || passed(pos, length + n, a.block, a.columns) ? -1 : static_cast<int64_t>(id) * a.block.d + in;
}

// One workgroup: the requests in order, and with TOKENS (few of them) the
// slots in the same launch.  All of a request's blocks or none, in the order of
// requests: after one that the stack cannot serve no later one takes blocks.
template <bool TOKENS>
__global__ void __launch_bounds__(kThreads) extend_plan_kernel(ExtendArgs a) {
  __shared__ int32_t s_off[TOKENS ? kThreads : 1], s_cu[TOKENS ? kThreads + 1 : 1], s_len[TOKENS ? kThreads : 1];
  const int32_t top = clamp_count(a.count, a.n_free);
  int64_t carry = 0, given = 0;
  for (int64_t base = 0; base < a.R; base += kThreads) {
    const int64_t r = base + threadIdx.x;
    int64_t need = 0, length = 0;
    bool fits = false;
    Span s{0, 0};
    if (r < a.R) {
      s = tree::span_of(a.cu, r, a.total);
      length = clamp_length(a.lengths[r]);
      const int64_t held = used(length, a.block.d, a.columns.d, a.wrap);
      const int64_t want = used(length + s.count, a.block.d, a.columns.d, a.wrap);
      fits = want <= a.columns.d;
      need = fits ? want - held : 0;
    }
    int64_t all = 0, taken = 0;
    const int64_t off = carry + scan(need, &all);
    const bool ok = fits && (need == 0 || off + need <= top);
    (void)scan(ok ? need : 0, &taken);
    carry += all;
    given += taken;
    if (r < a.R) {
      a.served[r] = ok;
      // a request that takes no block has no share of the stack: its offset is not used
      const int32_t mine = ok ? (need ? static_cast<int32_t>(off) : 0) : -1;
      if constexpr (TOKENS) {
        s_off[threadIdx.x] = mine;
        s_len[threadIdx.x] = static_cast<int32_t>(length);
        s_cu[threadIdx.x] = static_cast<int32_t>(s.first);
        if (r == a.R - 1) s_cu[threadIdx.x + 1] = static_cast<int32_t>(s.first + s.count);
      } else {
        a.plan[r] = mine;
      }
    }
  }
  if (threadIdx.x == 0) {
    *a.count = static_cast<int32_t>(top - given);
    if constexpr (!TOKENS) a.plan[a.R] = top;
  }
  if constexpr (TOKENS) {
    __syncthreads();
    for (int64_t t = threadIdx.x; t < a.total; t += kThreads) {
      int64_t slot = -1;
      if (a.R > 0 && t >= s_cu[0] && t < s_cu[a.R]) {
        const int r = tree::request_of(s_cu, 0, a.R - 1, t);
        slot = token_slot(a, r, s_len[r], t - s_cu[r], s_cu[r + 1] - s_cu[r], s_off[r], top);
      }
      a.slots[t] = slot;
    }
  }
}

// The requests that packed rows [t0, t1) of a workgroup touch.
__device__ __forceinline__ void row_range(const int32_t* cu, int R, int64_t t0, int64_t t1, int* lo, int* hi) {
  *lo = tree::request_of(cu, 0, R - 1, t0);
  *hi = tree::request_of(cu, *lo, R - 1, t1 - 1);
}

constexpr int kTokens = 512;   // of a workgroup

__global__ void __launch_bounds__(256) extend_slots_kernel(ExtendArgs a) {
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kTokens, t1 = t0 + kTokens < a.total ? t0 + kTokens : a.total;
  int lo, hi;
  row_range(a.cu, a.R, t0, t1, &lo, &hi);
  const int32_t top = a.plan[a.R];
  for (int64_t t = t0 + threadIdx.x; t < t1; t += 256) {
    const int r = tree::request_of(a.cu, lo, hi, t);
    const Span s = tree::span_of(a.cu, r, a.total);
    int64_t slot = -1;
    if (t >= s.first && t < s.first + s.count)
      slot = token_slot(a, r, clamp_length(a.lengths[r]), t - s.first, s.count, a.plan[r], top);
    a.slots[t] = slot;
  }
}

// ---------------------------------------------------------------------------
struct TrimArgs {
  const int64_t* lengths;   // [R]
  const int64_t* kept;      // [R]
  int32_t* tables;
  int32_t* free;
  int32_t* count;
  int32_t* plan;
  int64_t n_free;
  int block, columns, R, wrap;
};

// Columns [lo, hi) that request r gives back.
__device__ __forceinline__ void trim_range(const TrimArgs& a, int64_t r, int* lo, int* hi) {
  const int64_t from = used(clamp_length(a.kept[r]), a.block, a.columns, a.wrap);
  const int64_t to = used(clamp_length(a.lengths[r]), a.block, a.columns, a.wrap);
  *lo = static_cast<int>(from < a.columns ? from : a.columns);
  *hi = static_cast<int>(to < a.columns ? to : a.columns);
}

// One wave: its entries of the kDeep x 64 columns from c on; past hi none (-1).
constexpr int kDeep = 4;   // loads in flight
__device__ __forceinline__ void load_entries(const int32_t* row, int c, int hi, int32_t (&id)[kDeep]) {
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int u = 0; u < kDeep; ++u) {
    const int at = c + u * kWave + lane;
    id[u] = at < hi ? row[at] : -1;
  }
}
// One wave: the blocks in columns [lo, hi) of a row.
__device__ __forceinline__ int count_blocks(const int32_t* row, int lo, int hi) {
  int n = 0;
  for (int c = lo; c < hi; c += kDeep * kWave) {
    int32_t id[kDeep];
    load_entries(row, c, hi, id);
#pragma unroll
    for (int u = 0; u < kDeep; ++u) n += __popcll(__ballot(id[u] >= 0));
  }
  return n;
}
// One wave: they become the blocks first, first + 1, ... of the call.
__device__ __forceinline__ void give_back(const TrimArgs& a, int32_t* row, int lo, int hi, int64_t first,
                                          int64_t after) {
  const int lane = threadIdx.x & (kWave - 1);
  for (int c = lo; c < hi; c += kDeep * kWave) {
    int32_t id[kDeep];
    load_entries(row, c, hi, id);
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      const uint64_t set = __ballot(id[u] >= 0);
      const int64_t at = after - 1 - (first + __popcll(set & ((1ull << lane) - 1)));
      if (id[u] >= 0) {
        if (at >= 0 && at < a.n_free) a.free[at] = id[u];
        row[c + u * kWave + lane] = -1;
      }
      first += __popcll(set);
    }
  }
}

// One workgroup, R <= kWaves: a wave a request.
__global__ void __launch_bounds__(kThreads) trim_kernel(TrimArgs a) {
  __shared__ int s_n[kWaves];
  const int r = threadIdx.x / kWave;
  int lo, hi;
  trim_range(a, r, &lo, &hi);
  int32_t* row = a.tables + static_cast<int64_t>(r) * a.columns;
  const int n = count_blocks(row, lo, hi);
  if ((threadIdx.x & (kWave - 1)) == 0) s_n[r] = n;
  const int32_t top = clamp_count(a.count, a.n_free);
  __syncthreads();
  int64_t all = 0, first = 0;
  for (int i = 0; i < a.R; ++i) {
    first += i < r ? s_n[i] : 0;
    all += s_n[i];
  }
  if (n) give_back(a, row, lo, hi, first, top + all);
  if (threadIdx.x == 0) *a.count = static_cast<int32_t>(top + all < a.n_free ? top + all : a.n_free);
}

// More requests, or long tables: kSplit waves a request, a share of its columns each.  plan: the
// requests' counts, the waves', and the stack's height before.
constexpr int kSplit = 8;
__device__ __forceinline__ void wave_range(const TrimArgs& a, int64_t r, int* lo, int* hi) {
  trim_range(a, r, lo, hi);
  const int w = threadIdx.x / kWave, each = (max(*hi - *lo, 0) + kSplit - 1) / kSplit;
  const int from = *lo + w * each;
  *hi = min(*hi, from + each);
  *lo = from;
}

__global__ void __launch_bounds__(kSplit * kWave) trim_count_kernel(TrimArgs a) {
  __shared__ int s_n[kSplit];
  const int64_t r = blockIdx.x;
  const int w = threadIdx.x / kWave;
  int lo, hi;
  wave_range(a, r, &lo, &hi);
  const int n = count_blocks(a.tables + r * a.columns, lo, hi);
  if ((threadIdx.x & (kWave - 1)) == 0) {
    s_n[w] = n;
    a.plan[a.R + r * kSplit + w] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int all = 0;
    for (int i = 0; i < kSplit; ++i) all += s_n[i];
    a.plan[r] = all;
    if (r == 0) a.plan[static_cast<int64_t>(a.R) * (kSplit + 1)] = clamp_count(a.count, a.n_free);
  }
}

__global__ void __launch_bounds__(kSplit * kWave) trim_move_kernel(TrimArgs a) {
  __shared__ int64_t s_before[kSplit], s_all[kSplit];
  const int64_t r = blockIdx.x;
  const int w = threadIdx.x / kWave;
  int64_t before = 0, all = 0;
  for (int64_t i = threadIdx.x; i < a.R; i += kSplit * kWave) {
    const int n = a.plan[i];
    all += n;
    before += i < r ? n : 0;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    all += __shfl_xor(all, off, kWave);
    before += __shfl_xor(before, off, kWave);
  }
  if ((threadIdx.x & (kWave - 1)) == 0) {
    s_before[w] = before;
    s_all[w] = all;
  }
  __syncthreads();
  int64_t first = 0, after = a.plan[static_cast<int64_t>(a.R) * (kSplit + 1)];
#pragma unroll
  for (int i = 0; i < kSplit; ++i) {
    first += s_before[i];
    after += s_all[i];
    if (i < w) first += a.plan[a.R + r * kSplit + i];
  }
  int lo, hi;
  wave_range(a, r, &lo, &hi);
  if (a.plan[r]) give_back(a, a.tables + r * a.columns, lo, hi, first, after);
  if (r == 0 && threadIdx.x == 0) *a.count = static_cast<int32_t>(after < a.n_free ? after : a.n_free);
}

// ---------------------------------------------------------------------------
struct SlotArgs {
  const int32_t* cu;
  const int64_t* lengths;
  const int32_t* tables;
  const int32_t* parents;   // [total] or null: chains
  const int32_t* last;      // [R] or null: every node
  const uint8_t* served;    // [R] or null: all
  int64_t* slots;           // [total]
  int64_t* kept;            // [R]
  int64_t total;
  Div block, columns;
  int R, wrap;
};

// Whether request r, which ends at `end`, has its blocks: an extension served it, and a table that
// is no ring reaches as far.  Otherwise none of its nodes gets a slot: a held block would take a part
// of them, and modulo the columns they would go over the rows of its first positions.
__device__ __forceinline__ bool placed(const SlotArgs& a, int64_t r, int64_t end) {
  return (!a.served || a.served[r]) && (a.wrap || end <= static_cast<int64_t>(a.block.d) * a.columns.d);
}

__device__ __forceinline__ int64_t cache_slot(const SlotArgs& a, int64_t r, int64_t pos, int64_t end) {
  if (pos > kMaxLength || passed(pos, end, a.block, a.columns)) return -1;
  const uint32_t q = a.block.quot(static_cast<uint32_t>(pos)), in = static_cast<uint32_t>(pos) - q * a.block.d;
  const uint32_t c = q - a.columns.quot(q) * a.columns.d;
  const int32_t id = a.tables[r * a.columns.d + c];
  return id < 0 ? -1 : static_cast<int64_t>(id) * a.block.d + in;
}

// Chains (any length): a thread a token, and the first R threads a request each.
__global__ void __launch_bounds__(256) chain_slots_kernel(SlotArgs a) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (t < a.R) {
    const Span s = tree::span_of(a.cu, t, a.total);
    int64_t n = s.count;
    if (a.last) n = a.last[t] < 0 ? 0 : a.last[t] < n ? a.last[t] + 1 : n;
    const int64_t length = clamp_length(a.lengths[t]);
    a.kept[t] = placed(a, t, length + n) ? length + n : length;
  }
  if (t >= a.total) return;
  int64_t slot = -1;
  if (a.R > 0) {
    const int r = tree::request_of(a.cu, 0, a.R - 1, t);
    const Span s = tree::span_of(a.cu, r, a.total);
    const int64_t i = t - s.first;
    const int64_t n = a.last && a.last[r] < s.count ? static_cast<int64_t>(a.last[r]) + 1 : s.count;
    const int64_t length = clamp_length(a.lengths[r]);
    if (i >= 0 && i < n && placed(a, r, length + n)) slot = cache_slot(a, r, length + i, length + n);
  }
  a.slots[t] = slot;
}

// Trees: a wave a request, a lane a node; the wave after the last request
// clears the slots of rows that belong to none.
__global__ void __launch_bounds__(256) tree_slots_kernel(SlotArgs a) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
  if (r > a.R) return;
  if (r == a.R) {
    const int64_t begin = a.R > 0 ? a.cu[0] : 0, end = a.R > 0 ? a.cu[a.R] : 0;
    for (int64_t t = lane; t < a.total && t < begin; t += kWave) a.slots[t] = -1;
    for (int64_t t = (end < 0 ? 0 : end) + lane; t < a.total; t += kWave) a.slots[t] = -1;
    return;
  }
  const Span s = tree::span_of(a.cu, r, a.total);
  const int n = static_cast<int>(s.count < tree::kNodes ? s.count : tree::kNodes);
  const uint64_t set = tree::ancestors(a.parents + s.first, n);
  const int64_t length = clamp_length(a.lengths[r]);
  int64_t deep;
  bool on = lane < n;
  if (a.last) {
    const int leaf = a.last[r];
    const bool none = leaf < 0 || leaf >= n;
    const uint64_t path = __shfl(set, none ? 0 : leaf, kWave);
    on = on && !none && ((path >> lane) & 1);
    deep = none ? 0 : __popcll(path);
  } else {
    int d = on ? __popcll(set) : 0;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const int o = __shfl_xor(d, off, kWave);
      d = o > d ? o : d;
    }
    deep = d;
  }
  if (!placed(a, r, length + deep)) {
    on = false;
    deep = 0;
  }
  if (lane < n) a.slots[s.first + lane] = on ? cache_slot(a, r, length + __popcll(set) - 1, length + deep) : -1;
  for (int64_t i = n + lane; i < s.count; i += kWave) a.slots[s.first + i] = -1;
  if (lane == 0) a.kept[r] = length + deep;
}

// ---------------------------------------------------------------------------
struct WriteArgs {
  const char* k;         // [N, G, D], rows k_ts bytes apart
  const char* v;
  int64_t k_ts, v_ts;
  const int64_t* slots;  // [N], < 0: not written
  char* keys;            // [blocks, G, block, D]
  char* values;
  const int64_t* positions;   // [N] or null
  int32_t* cache_pos;         // [blocks, G, block] or null
  int64_t N, n_slots;
  Div block, pieces, row;     // slot -> block; a token's 16-byte pieces; a head's
  int G;
};

// Bound by HBM: a token's rows are read and written once, past the caches (65521
// tokens x 8 heads of 128: 106 us, 5.1 TB/s; through them 115).  A thread moves a
// 16-byte piece of the keys and of the values of kRun tokens.
constexpr int kRun = 2;

__global__ void __launch_bounds__(256) cache_write_kernel(WriteArgs a) {
  const int64_t n = a.N * a.pieces.d, at = static_cast<int64_t>(blockIdx.x) * (256 * kRun) + threadIdx.x;
  typedef unsigned u4 __attribute__((ext_vector_type(4)));
  u4 x[kRun], y[kRun];
  int64_t to[kRun];
#pragma unroll
  for (int u = 0; u < kRun; ++u) {
    const int64_t i = at + u * 256 < n ? at + u * 256 : n - 1;
    const int64_t t = i < (1ll << 31) ? a.pieces.quot(static_cast<uint32_t>(i)) : i / a.pieces.d;
    const int64_t slot = a.slots[t];
    const bool in = at + u * 256 < n && slot >= 0 && slot < a.n_slots;
    const uint32_t p = static_cast<uint32_t>(i - t * a.pieces.d), g = a.row.quot(p);
    const int64_t b = slot < (1ll << 31) ? a.block.quot(in ? static_cast<uint32_t>(slot) : 0) : slot / a.block.d;
    const int64_t head = (b * a.G + g) * a.block.d + (slot - b * a.block.d);
    to[u] = in ? (head * a.row.d + (p - g * a.row.d)) * 16 : -1;
    x[u] = y[u] = u4{0,0,0,0};
    if (in) {
      x[u] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(a.k + t * a.k_ts + static_cast<int64_t>(p) * 16));
      y[u] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(a.v + t * a.v_ts + static_cast<int64_t>(p) * 16));
      if (a.cache_pos && p == g * a.row.d) a.cache_pos[head] = static_cast<int32_t>(a.positions[t]);
    }
  }
#pragma unroll
  for (int u = 0; u < kRun; ++u)
    if (to[u] >= 0) {
      __builtin_nontemporal_store(x[u], reinterpret_cast<u4*>(a.keys + to[u]));
      __builtin_nontemporal_store(y[u], reinterpret_cast<u4*>(a.values + to[u]));
    }
}

}  // namespace
}  // namespace yh

namespace yh {
namespace {
// One launch where one workgroup can do it all: few tokens after the requests ...
bool extend_in_one(int64_t n_seqs, int64_t total) { return n_seqs <= kThreads && total <= 4096; }
// ... or a wave for every request, with columns that it takes in one step.  (us in a captured step, one launch and
// two: 1 table 5.8 and 6.6; 16 tables of 256 columns 7.6 and 7.8 with all blocks back, 6.4 and 7.5 with few; 16 of 1000
// 13.7 and 8.3 with all; a workgroup that takes 32 requests in turn 8.1 and 7.6, 128 20 and 8, 512 68 and 9.)
bool trim_in_one(int64_t n_seqs, int64_t columns) { return n_seqs <= kWaves && columns <= kDeep * kWave; }
}  // namespace
}  // namespace yh

extern "C" int64_t yh_extend_plan_bytes(int64_t n_seqs, int64_t total) {
  return n_seqs <= 0 || yh::extend_in_one(n_seqs, total) ? 0 : (n_seqs + 1) * 4;
}
extern "C" int64_t yh_trim_plan_bytes(int64_t n_seqs, int64_t columns) {
  return n_seqs <= 0 || yh::trim_in_one(n_seqs, columns) ? 0 : (n_seqs * (yh::kSplit + 1) + 1) * 4;
}

extern "C" int yh_extend_block_tables(const int64_t* lengths, const int32_t* cu_seqlens, int32_t* tables,
                                      const int32_t* free_blocks, int32_t* free_count, int64_t* slots,
                                      uint8_t* served, void* plan, int64_t n_seqs, int64_t columns, int64_t n_free,
                                      int64_t total, int64_t block, int wrap, yh_stream_t stream) {
  using namespace yh;
  YH_CHECK_ARG(n_seqs >= 0 && columns > 0 && n_free >= 0 && total >= 0 && block > 0, "extend_block_tables: bad sizes");
  YH_CHECK_ARG(n_seqs < (1ll << 31) && columns < (1ll << 31) && block < (1ll << 31) && total < (1ll << 31) &&
                   n_free < (1ll << 31),
               "extend_block_tables: sizes too large");
  if (n_seqs == 0 && total == 0) return YH_OK;
  YH_CHECK_ARG((lengths && cu_seqlens && tables && served && free_count && (plan || extend_in_one(n_seqs, total)) && (free_blocks || n_free == 0)) ||
                   n_seqs == 0,
               "extend_block_tables: null pointer");
  YH_CHECK_ARG(slots || total == 0, "extend_block_tables: null pointer");
  ExtendArgs a{lengths, cu_seqlens, tables, free_blocks, free_count, slots, served, static_cast<int32_t*>(plan), n_free,
               total, tree::make_div(static_cast<uint32_t>(block)), tree::make_div(static_cast<uint32_t>(columns)),
               static_cast<int>(n_seqs), wrap ? 1 : 0};
  hipStream_t st = static_cast<hipStream_t>(stream);
  YH_CHECK_ARG(n_seqs > 0, "extend_block_tables: tokens without requests");
  if (extend_in_one(n_seqs, total)) {
    hipLaunchKernelGGL(extend_plan_kernel<true>, dim3(1), dim3(kThreads), 0, st, a);
  } else {
    hipLaunchKernelGGL(extend_plan_kernel<false>, dim3(1), dim3(kThreads), 0, st, a);
    YH_CHECK_LAUNCH("extend_block_tables plan");
    if (total)
      hipLaunchKernelGGL(extend_slots_kernel, dim3(static_cast<unsigned>((total + kTokens - 1) / kTokens)), dim3(256), 0, st, a);
  }
  YH_CHECK_LAUNCH("extend_block_tables");
  return YH_OK;
}

extern "C" int yh_trim_block_tables(const int64_t* lengths, const int64_t* kept, int32_t* tables,
                                    int32_t* free_blocks, int32_t* free_count, void* plan, int64_t n_seqs,
                                    int64_t columns, int64_t n_free, int64_t block, int wrap, yh_stream_t stream) {
  using namespace yh;
  YH_CHECK_ARG(n_seqs >= 0 && columns > 0 && n_free >= 0 && block > 0, "trim_block_tables: bad sizes");
  YH_CHECK_ARG(n_seqs < (1ll << 23) && columns < (1ll << 31) && block < (1ll << 31) && n_free < (1ll << 31),
               "trim_block_tables: sizes too large");
  if (n_seqs == 0) return YH_OK;
  YH_CHECK_ARG(lengths && kept && tables && free_count && (plan || trim_in_one(n_seqs, columns)) &&
                   (free_blocks || n_free == 0),
               "trim_block_tables: null pointer");
  TrimArgs a{lengths, kept, tables, free_blocks, free_count, static_cast<int32_t*>(plan), n_free,
             static_cast<int>(block), static_cast<int>(columns), static_cast<int>(n_seqs), wrap ? 1 : 0};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (trim_in_one(n_seqs, columns)) {
    hipLaunchKernelGGL(trim_kernel, dim3(1), dim3(static_cast<unsigned>(n_seqs * kWave)), 0, st, a);
  } else {
    hipLaunchKernelGGL(trim_count_kernel, dim3(static_cast<unsigned>(n_seqs)), dim3(kSplit * kWave), 0, st, a);
    YH_CHECK_LAUNCH("trim_block_tables count");
    hipLaunchKernelGGL(trim_move_kernel, dim3(static_cast<unsigned>(n_seqs)), dim3(kSplit * kWave), 0, st, a);
  }
  YH_CHECK_LAUNCH("trim_block_tables");
  return YH_OK;
}

extern "C" int yh_slot_map(const int32_t* cu_seqlens, const int64_t* lengths, const int32_t* tables,
                           const int32_t* parents, const int32_t* last, int64_t* slots, int64_t* kept, int64_t n_seqs,
                           int64_t columns, int64_t total, int64_t block, yh_stream_t stream) {
  return yh_slot_map_served(cu_seqlens, lengths, tables, parents, last, nullptr, slots, kept, n_seqs, columns, total,
                            block, 1, stream);
}

extern "C" int yh_slot_map_served(const int32_t* cu_seqlens, const int64_t* lengths, const int32_t* tables,
                                  const int32_t* parents, const int32_t* last, const uint8_t* served, int64_t* slots,
                                  int64_t* kept, int64_t n_seqs, int64_t columns, int64_t total, int64_t block,
                                  int wrap, yh_stream_t stream) {
  using namespace yh;
  YH_CHECK_ARG(n_seqs >= 0 && columns > 0 && total >= 0 && block > 0, "slot_map: bad sizes");
  YH_CHECK_ARG(n_seqs < (1ll << 31) && columns < (1ll << 31) && block < (1ll << 31) && total < (1ll << 31),
               "slot_map: sizes too large");
  if (n_seqs == 0 && total == 0) return YH_OK;
  YH_CHECK_ARG((cu_seqlens && lengths && tables && kept) || n_seqs == 0, "slot_map: null pointer");
  YH_CHECK_ARG(slots || total == 0, "slot_map: null pointer");
  SlotArgs a{cu_seqlens, lengths, tables, parents, last, served, slots, kept, total,
             tree::make_div(static_cast<uint32_t>(block)), tree::make_div(static_cast<uint32_t>(columns)),
             static_cast<int>(n_seqs), wrap ? 1 : 0};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (parents) {
    hipLaunchKernelGGL(tree_slots_kernel, dim3(static_cast<unsigned>(n_seqs / 4 + 1)), dim3(256), 0, st, a);
  } else {
    const int64_t n = total > n_seqs ? total : n_seqs;
    hipLaunchKernelGGL(chain_slots_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, st, a);
  }
  YH_CHECK_LAUNCH("slot_map");
  return YH_OK;
}

extern "C" int yh_cache_write(const void* k, int64_t k_stride, const void* v, int64_t v_stride, const int64_t* slots,
                              void* keys, void* values, const int64_t* positions, int32_t* cache_pos, int64_t N,
                              int64_t blocks, int64_t G, int64_t D, int64_t block, int dtype, yh_stream_t stream) {
  using namespace yh;
  YH_CHECK_ARG(N >= 0 && blocks >= 0 && G > 0 && D > 0 && block > 0, "cache_write: bad sizes");
  YH_CHECK_ARG(is_float_dtype(dtype), "cache_write: dtype must be f32, bf16 or f16");
  const int64_t e = dtype == YH_F32 ? 4 : 2, row = D * e;
  YH_CHECK_ARG(row % 16 == 0, "cache_write: a head's row must be a multiple of 16 bytes");
  if (N == 0 || blocks == 0) return YH_OK;
  YH_CHECK_ARG(k && v && slots && keys && values, "cache_write: null pointer");
  YH_CHECK_ARG(!positions == !cache_pos, "cache_write: positions and their cache come together");
  YH_CHECK_ARG(tree::aligned16(k) && tree::aligned16(v) && tree::aligned16(keys) && tree::aligned16(values) &&
                   k_stride * e % 16 == 0 && v_stride * e % 16 == 0 && k_stride >= G * D && v_stride >= G * D,
               "cache_write: rows must be 16-byte aligned and hold whole heads");
  YH_CHECK_ARG(N < (1ll << 31) && blocks < (1ll << 31) && block < (1ll << 31) && G * row < (1ll << 31),
               "cache_write: sizes too large");
  const int64_t pieces = G * row / 16, grid = (N * pieces + 256 * kRun - 1) / (256 * kRun);
  YH_CHECK_ARG(grid < (1ll << 24), "cache_write: sizes too large");
  WriteArgs a{static_cast<const char*>(k), static_cast<const char*>(v), k_stride * e, v_stride * e, slots,
              static_cast<char*>(keys), static_cast<char*>(values), positions, cache_pos, N, blocks * block,
              tree::make_div(static_cast<uint32_t>(block)), tree::make_div(static_cast<uint32_t>(pieces)),
              tree::make_div(static_cast<uint32_t>(row / 16)), static_cast<int>(G)};
  hipLaunchKernelGGL(cache_write_kernel, dim3(static_cast<unsigned>(grid)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), a);
  YH_CHECK_LAUNCH("cache_write");
  return YH_OK;
}
