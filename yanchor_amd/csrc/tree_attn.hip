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
// A workgroup takes a request, a KV head and 128 of the rows (node, query head
// of the group): four waves of 32 rows share 64-key tiles (attn_tile.h) that
// begin at multiples of 64 positions; the nodes themselves are the last tile,
// its mask the ancestor sets.
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
};

constexpr int kNW = 4;                       // waves a workgroup
constexpr int kM = kNW * attn::kRows;        // rows a workgroup

template <int DT, int D>
__global__ void __launch_bounds__(kNW * 64, 2) tree_attention_kernel(TreeArgs a) {
  using M = attn::Mfma<DT>;
  __shared__ attn::Rows stage[4];   // two buffers of key rows, two of value rows
  __shared__ uint64_t s_set[tree::kNodes];
  __shared__ int s_deep;
  attn::Rows *ktile = stage, *vtile = stage + 2;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  const int64_t work = static_cast<int64_t>(a.R) * a.G * a.mtiles;
  if (static_cast<int64_t>(blockIdx.x) >= work) {   // rows of no request
    const int64_t end = a.R ? a.cu[a.R] : 0, row = static_cast<int64_t>(a.H) * D;
    for (int64_t i = (end < 0 ? 0 : end) * row + threadIdx.x; i < a.total * row; i += kNW * 64) a.out[i] = 0;
    return;
  }
  const int g = blockIdx.x % a.G, mt = blockIdx.x / a.G % a.mtiles, r = blockIdx.x / a.G / a.mtiles;
  const tree::Span span = tree::span_of(a.cu, r, a.total);
  const int n = static_cast<int>(span.count < a.max_nodes ? span.count : a.max_nodes);
  const int rep = a.rep.d;
  if (mt == 0) {   // nodes past the most that the call takes: not a number
    const int64_t first = span.first + n, row = static_cast<int64_t>(a.H) * D;
    for (int64_t i = threadIdx.x; i < (span.count - n) * rep * D; i += kNW * 64) {
      const int64_t t = i / (rep * D);
      a.out[(first + t) * row + static_cast<int64_t>(g) * rep * D + (i - t * rep * D)] = DT == YH_BF16 ? 0x7fc0 : 0x7e00;
    }
  }
  if (mt * kM >= n * rep) return;

  if (w == 0) {
    const uint64_t set = tree::ancestors(a.parents ? a.parents + span.first : nullptr, n);
    s_set[lane] = set;
    int d = lane < n ? __popcll(set) - 1 : 0;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) d = max(d, __shfl_xor(d, off, 64));
    if (lane == 0) s_deep = d;
  }
  __syncthreads();
  const int deep = s_deep;

  // this lane's query: row m of the request's (node, head of the group) rows
  const int m = mt * kM + w * attn::kRows + (lane & 31);
  const bool active = mt * kM + w * attn::kRows < n * rep;   // of the wave
  const bool mine = m < n * rep;
  const int node = mine ? a.rep.quot(m) : 0, head = g * rep + (mine ? m - node * rep : 0);
  uint64_t see = mine ? s_set[node] : 0;
  const int depth = mine ? __popcll(see) - 1 : 0;
  const int64_t length = a.lengths[r] < 0 ? 0 : a.lengths[r];
  const int64_t W = a.window ? a.window : (1ll << 40);
  for (int far = depth + 1; far > W; --far) see &= see - 1;   // ancestors past the window: the earliest nodes of the path
  // positions that are there and that some node sees
  const int64_t room = static_cast<int64_t>(a.columns.d) * a.block.d;
  const int64_t oldest = max(max(length - room, length - W + 1), static_cast<int64_t>(0));
  const int lo = static_cast<int>(min(oldest, length)), L = static_cast<int>(min(length, (1ll << 31) - 1));
  const int base = lo & ~(attn::kTile - 1);
  const int ctx = L > lo ? (L - base + attn::kTile - 1) / attn::kTile : 0, tiles = ctx + 1;
  // the first position that this lane's query sees, and the wave's rows' earliest
  const int from = static_cast<int>(min(max(length + depth - W + 1, static_cast<int64_t>(0)), (1ll << 31) - 1));
  int wfrom = mine ? from : 0x7fffffff;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) wfrom = min(wfrom, __shfl_xor(wfrom, off, 64));
  uint64_t wsee = see;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) wsee |= __shfl_xor(wsee, off, 64);
  const int64_t allfrom = length + deep - W + 1;   // from here on every node sees

  attn::State<DT, false, D> st;
  st.init(false);
  st.load_q(a.q + (span.first + node) * a.q_ts + static_cast<int64_t>(head) * D, mine);
  const float k2 = a.scale * 1.4426950408889634f;

  const int32_t* table = a.tables + static_cast<int64_t>(r) * a.columns.d;
  // Lane l stands for the tile's row l: its block id is loaded a tile ahead of
  // the copies, which take the row from the lane.
  auto fetch = [&](int t) {
    const int p = base + t * attn::kTile + lane;
    if (t >= ctx || p < lo || p >= L) return -1;
    const uint32_t qd = a.block.quot(p);
    return table[qd - a.columns.quot(qd) * a.columns.d];
  };
  uint64_t have = 0;   // rows of the tile that exist
  auto issue = [&](int t, int buf, int id) {
    int row = -1;   // in the cache, or the node
    if (t < ctx) {
      const int p = base + t * attn::kTile + lane;
      if (id >= 0 && id < a.NB) row = (id * a.G + g) * a.block.d + (p - a.block.quot(p) * a.block.d);
    } else if (lane < n) {
      row = lane;
    }
    have = __ballot(row >= 0);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const uint16_t* src = t < ctx ? (which ? a.values : a.keys)
                                    : (which ? a.v + span.first * a.v_ts : a.k + span.first * a.k_ts) +
                                          static_cast<int64_t>(g) * D;
      const int64_t stride = t < ctx ? D : which ? a.v_ts : a.k_ts;
      attn::load_rows<kNW>(which ? vtile[buf] : ktile[buf], [&](int rr, int e, const void* l) {
        const int x = __shfl(row, rr, 64);
        const uint16_t* p = x < 0 ? reinterpret_cast<const uint16_t*>(attn::zero_row) : src + x * stride;
        if (D == attn::kD || e < D) attn::copy16(p + e, l);
      });
    }
  };

  int t = 0, buf = 0, id = fetch(0);
  issue(0, 0, id);
  id = fetch(1);
  auto inner = [&]() { return t < ctx && have == ~0ull && base + t * attn::kTile >= allfrom; };
  auto tile = [&](auto edge) {
    const uint64_t there = have;
    attn::copy_wait();      // this wave's part of the tile has arrived
    attn::tile_barrier();   // everyone's has, and the other buffers are consumed
    if (t + 1 < tiles) issue(t + 1, buf ^ 1, id);
    id = fetch(t + 2);
    if (active) {
      attn::f32x16 c[2];
      st.scores(ktile[buf], c);
      uint64_t keep = ~0ull;
      if constexpr (edge.value) {
        uint64_t live;   // the tile's keys that the lane's query sees
        if (t < ctx) {
          const int p0 = base + t * attn::kTile;
          const int skip = min(max(from - p0, 0), 64), wskip = min(max(wfrom - p0, 0), 64);
          live = skip > 63 ? 0 : there & (~0ull << skip);
          keep = wskip > 63 ? 0 : there & (~0ull << wskip);
        } else {
          live = see;
          keep = wsee;
        }
        const uint64_t sh = live >> (4 * (lane >> 5));
        st.mask(c, [&](int key, int) { return ((key < 32 ? static_cast<uint32_t>(sh) >> key : static_cast<uint32_t>(sh >> 32) >> (key - 32)) & 1) != 0; });
      }
      st.template step<false, edge.value>(c, vtile[buf], k2, keep);
    }
    ++t;
    buf ^= 1;
  };
  // Tiles whose keys all rows see and the others take a loop each: as branches
  // of one loop they spill (the waves' conditions may differ: both loops pass
  // one barrier a tile).
  while (t < tiles) {
#pragma unroll 1
    while (t < tiles && inner()) tile(std::false_type{});
#pragma unroll 1
    while (t < tiles && !inner()) tile(std::true_type{});
  }
  if (!mine) return;

  const float inv = 1.f / (st.den + __shfl_xor(st.den, 32, 64));
  const int64_t row = span.first + node;
  uint16_t* out = a.out + (row * a.H + head) * D + 4 * (lane >> 5);
  const uint16_t* gate = a.gate ? a.gate + row * a.g_ts + head * a.g_hs + 4 * (lane >> 5) : nullptr;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int rr = 0; rr < 4; ++rr) {
      const int dim = 32 * d + 8 * rr;
      float o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = st.acc[d][4 * rr + e] * inv;
      if (gate) {
        uint16_t x[4];
        if (a.gate8) {
          const uint2 y = *reinterpret_cast<const uint2*>(gate + dim);
          x[0] = y.x & 0xffff;
          x[1] = y.x >> 16;
          x[2] = y.y & 0xffff;
          x[3] = y.y >> 16;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = gate[dim + e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= 1.f / (1.f + __expf(-M::widen(x[e])));
      }
      *reinterpret_cast<uint2*>(out + dim) = make_uint2(M::round2(o[0], o[1]), M::round2(o[2], o[3]));
    }
}

template <int DT>
void launch(const TreeArgs& a, int64_t D, unsigned grid, hipStream_t st) {
  if (D == 128)
    hipLaunchKernelGGL((tree_attention_kernel<DT, 128>), dim3(grid), dim3(kNW * 64), 0, st, a);
  else
    hipLaunchKernelGGL((tree_attention_kernel<DT, 64>), dim3(grid), dim3(kNW * 64), 0, st, a);
}

}  // namespace
}  // namespace yh

extern "C" int yh_tree_attention(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                                 int64_t v_stride, const int32_t* parents, const int32_t* cu_seqlens,
                                 const int64_t* lengths, const void* keys, const void* values, const int32_t* tables,
                                 const void* gate, int64_t gate_token_stride, int64_t gate_head_stride, void* out,
                                 int64_t n_seqs, int64_t total, int64_t blocks, int64_t columns, int64_t H, int64_t G,
                                 int64_t D, int64_t block, int64_t window, int64_t max_nodes, float scale, int dtype,
                                 yh_stream_t stream) {
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
  const int64_t rep = H / G, mtiles = (max_nodes * rep + kM - 1) / kM, work = n_seqs * G * mtiles;
  YH_CHECK_ARG(work < (1ll << 23), "tree_attention: sizes too large");
  const bool gate8 = gate && (reinterpret_cast<uintptr_t>(gate) & 7) == 0 && gate_token_stride % 4 == 0 &&
                     gate_head_stride % 4 == 0;
  TreeArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
             q_stride, k_stride, v_stride, parents, cu_seqlens, lengths, static_cast<const uint16_t*>(keys),
             static_cast<const uint16_t*>(values), tables, static_cast<const uint16_t*>(gate), gate_token_stride,
             gate_head_stride, static_cast<uint16_t*>(out), total, window,
             tree::make_div(static_cast<uint32_t>(block)), tree::make_div(static_cast<uint32_t>(columns)),
             tree::make_div(static_cast<uint32_t>(rep)), (int)n_seqs, (int)H, (int)G, (int)blocks, (int)max_nodes,
             (int)mtiles, gate8 ? 1 : 0, scale};
  const unsigned grid = static_cast<unsigned>(work + 1);   // the last clears the rows of no request
  if (dtype == YH_BF16) launch<YH_BF16>(a, D, grid, static_cast<hipStream_t>(stream));
  else launch<YH_F16>(a, D, grid, static_cast<hipStream_t>(stream));
  YH_CHECK_LAUNCH("tree_attention");
  return YH_OK;
}
