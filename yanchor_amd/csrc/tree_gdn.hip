// A GDN layer over drafted trees: the causal conv and the gated delta rule of
// every node, each continuing its own path from the request's window and state.
// Neither is written: which path stays is known only after the verification.
//
// Delta rule, with G_i the sum of the log decays g along the path to node i
// (itself included), S the request's state and every token's u_j the rank-one
// update that it leaves, S_i = e^{G_i} S + sum over the path e^{G_i - G_j} k_j u_j^T:
//   u_i = beta_i (v_i - e^{G_i} k_i S - sum_{j above i} e^{G_i - G_j} (k_i . k_j) u_j)
//   o_i = e^{G_i} q_i S + sum_{j above i, and i} e^{G_i - G_j} (q_i . k_j) u_j
// which is the chunk form of the rule with the ancestor sets in place of the
// causal triangle: the state is read once for all nodes and no state of a node
// is ever formed.
//
// A decay between two nodes is the exponential of a difference of path sums, from
// which one strong decay above both must cancel: the sums are held in 64 bits
// (in 32, g = -3e4 above a node would leave its own decay of -0.2 an error of
// 8e-4), and a g below -104, whose exponential is 0 in 32 bits, counts as -104, so
// that -inf forgets the state as it does token by token (-inf + inf would be NaN).
#include "conv_chan.h"
#include "tree.h"

namespace yh {
namespace {

struct GdnArgs {
  const void* q;           // [N, H, K]
  const void* k;
  const void* v;           // [N, HV, V]
  const void* g;           // [N, HV]
  const void* beta;
  const int32_t* parents;  // [N] or null: chains
  const int32_t* cu;       // [R + 1]
  const void* state;       // [rows, HV, K, V]
  const int32_t* rows;     // [R] or null; < 0: no request
  void* o;                 // [N, HV, V]
  int64_t total, n_rows;
  int R, H, HV, max_nodes, l2, dt, g_dt, beta_dt, state_dt;
  float scale;
};

__device__ __forceinline__ double log_decay(float g) { return g < -104.f ? -104.f : g; }   // NaN stays

// Any of the types: fp32 arithmetic on the vector unit, a workgroup a request
// and value head.
template <int K, int V>
__global__ void __launch_bounds__(256) tree_gdn_any_kernel(GdnArgs a) {
  constexpr int kN = tree::kNodes;
  __shared__ float s_q[kN][K + 1], s_k[kN][K + 1], s_low[kN][kN], s_att[kN][kN], s_u[kN][V];
  __shared__ double s_g[kN];
  __shared__ float s_beta[kN];
  __shared__ uint64_t s_set[kN];
  const int tid = threadIdx.x, lane = tid & 63;
  if (blockIdx.x >= static_cast<unsigned>(a.R * a.HV)) {   // rows of no request
    tree::clear_rows<256>(a.o, a.cu, a.R, a.total, static_cast<int64_t>(a.HV) * V * (a.dt == YH_F32 ? 4 : 2),
                          blockIdx.x - a.R * a.HV, gridDim.x - a.R * a.HV);
    return;
  }
  const int hv = blockIdx.x % a.HV, r = blockIdx.x / a.HV, h = hv / (a.HV / a.H);
  const tree::Span span = tree::span_of(a.cu, r, a.total);
  const int64_t srow = a.rows ? a.rows[r] : r;
  const bool none = srow < 0 || srow >= a.n_rows;
  const int n = none ? 0 : static_cast<int>(span.count < a.max_nodes ? span.count : a.max_nodes);
  for (int64_t i = n; i < span.count; ++i)   // no request: zeros; nodes past the most that the call takes: not a number
    for (int c = tid; c < V; c += 256) store_any(a.o, ((span.first + i) * a.HV + hv) * V + c, a.dt, none ? 0.f : NAN);
  if (n == 0) return;

  if (tid < 64) {
    const int64_t i = (span.first + (lane < n ? lane : 0)) * a.HV + hv;
    double gate = lane < n ? log_decay(load_any(a.g, i, a.g_dt)) : 0.;
    const uint64_t set = tree::ancestors(a.parents ? a.parents + span.first : nullptr, n, &gate);
    s_set[lane] = set;
    s_g[lane] = gate;
    s_beta[lane] = load_any(a.beta, i, a.beta_dt);
  }
  for (int i = tid >> 6; i < n; i += 4) {   // a wave a row: load, normalise
    const int64_t at = ((span.first + i) * a.H + h) * K;
    float x[K / 64], y[K / 64], sx = 0.f, sy = 0.f;
#pragma unroll
    for (int c = 0; c < K / 64; ++c) {
      x[c] = load_any(a.q, at + c * 64 + lane, a.dt);
      y[c] = load_any(a.k, at + c * 64 + lane, a.dt);
      sx += x[c] * x[c];
      sy += y[c] * y[c];
    }
    const float rx = a.scale * (a.l2 ? rsqrtf(wave_sum(sx) + 1e-6f) : 1.f), ry = a.l2 ? rsqrtf(wave_sum(sy) + 1e-6f) : 1.f;
#pragma unroll
    for (int c = 0; c < K / 64; ++c) {
      s_q[i][c * 64 + lane] = x[c] * rx;
      s_k[i][c * 64 + lane] = y[c] * ry;
    }
  }
  __syncthreads();
  for (int e = tid; e < n * n; e += 256) {
    const int i = e / n, j = e % n;
    float low = 0.f, att = 0.f;
    if ((s_set[i] >> j) & 1) {
      for (int c = 0; c < K; ++c) {
        low = fmaf(s_k[i][c], s_k[j][c], low);
        att = fmaf(s_q[i][c], s_k[j][c], att);
      }
      const float decay = expf(static_cast<float>(s_g[i] - s_g[j]));
      low = i == j ? 0.f : low * decay * s_beta[i];
      att *= decay;
    }
    s_low[i][j] = low;
    s_att[i][j] = att;
  }
  __syncthreads();
  for (int c = tid; c < V; c += 256) {   // a thread a column
    float s[K];
    const int64_t at = (srow * a.HV + hv) * K * V + c;
#pragma unroll
    for (int d = 0; d < K; ++d) s[d] = load_any(a.state, at + d * V, a.state_dt);
    for (int i = 0; i < n; ++i) {
      float ks = 0.f, qs = 0.f;
#pragma unroll
      for (int d = 0; d < K; ++d) {
        ks = fmaf(s_k[i][d], s[d], ks);
        qs = fmaf(s_q[i][d], s[d], qs);
      }
      const float eg = expf(static_cast<float>(s_g[i]));
      const int64_t row = ((span.first + i) * a.HV + hv) * V + c;
      float u = s_beta[i] * (load_any(a.v, row, a.dt) - eg * ks), o = eg * qs;
      for (int j = 0; j < i; ++j)
        if ((s_set[i] >> j) & 1) {
          u = fmaf(-s_low[i][j], s_u[j][c], u);
          o = fmaf(s_att[i][j], s_u[j][c], o);
        }
      s_u[i][c] = u;
      store_any(a.o, row, a.dt, fmaf(s_att[i][i], u, o));
    }
  }
}

// ---------------------------------------------------------------------------
// bf16 q / k / v with K = 128 on MFMA: a workgroup a request and value head, its
// W waves 1 / W of the value columns each.
//
// In the masks' order (a node's ancestors come before it) everything above is
// a lower triangular product over 16-node tiles, as in a chunk of a prompt:
//   low_ij = beta_i e^{G_i - G_j} (k_i . k_j), att_ij = e^{G_i - G_j} (q_i . k_j)
// where j is above i, 0 elsewhere; w_i = beta_i (v_i - e^{G_i} k_i S); then tile by
// tile u_b = (I + low_bb)^-1 (w_b - sum_{a < b} low_ba u_a), with the inverses of
// the diagonal tiles by forward substitution.
//
// q and k are exact bf16 operands, their norms and the decays go into the
// factors; float32 operands (S, low, att, w, u) enter the products as pairs hi +
// lo of bf16, which leaves 2^-16 of each product.  S is read straight into the
// operand layout: a lane holds rows 32 s + 8 (lane / 16) + 0..7 of CT
// neighbouring columns.
//
// What is not finite in one node may reach its own descendants only, but a
// product of a 0 in the mask with it would spread it: such elements enter the
// products as 0 and their bits (`bad`) turn the descendants' outputs into NaN.
//
// Bound by the chain of a workgroup's phases (the loads of q and k, the state's
// read and products, the masks' products, the inverses, the tiles one after
// another), which three workgroups a CU overlap with the read of each other's
// state: 421 MB in 110 us, 3.8 TB/s (two a CU: 156 for 136 before the phases were
// shortened).  Part of the chain are waits that the loads' order does not ask for:
// a request of fewer nodes than rows zeroes q and k behind each load, which waits
// for it, and with four tiles, V = 128 and a float32 state 5 registers spill, three
// of them just loaded.  Of up to 16 nodes, one tile, 71 us; float16 state 105.
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef float f32x2v __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4v mma32(bf16x8_t a, bf16x8_t b, f32x4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4v mma16(uint2 a, uint2 b, f32x4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4_t, a), __builtin_bit_cast(s16x4_t, b), c, 0,
                                                   0, 0);
}
// Two values as bf16 hi (to nearest) and lo = bf16(x - hi), packed in pairs.
__device__ __forceinline__ void pair2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2v){x, y}, bf16x2_t));
  lo = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2v){x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u)}, bf16x2_t));
}
// One value as a word hi << 16 | lo, and back.
__device__ __forceinline__ uint32_t split1(float x) {
  const uint16_t hi = f32_to_bf16(x);
  return static_cast<uint32_t>(hi) << 16 | f32_to_bf16(x - bf16_to_f32(hi));
}
__device__ __forceinline__ float join1(uint32_t w) { return __uint_as_float(w & 0xffff0000u) + __uint_as_float(w << 16); }
// Four such words as the hi and the lo operand.
__device__ __forceinline__ void unzip4(uint4 w, uint2& hi, uint2& lo) {
  hi = make_uint2(__builtin_amdgcn_perm(w.y, w.x, 0x07060302), __builtin_amdgcn_perm(w.w, w.z, 0x07060302));
  lo = make_uint2(__builtin_amdgcn_perm(w.y, w.x, 0x05040100), __builtin_amdgcn_perm(w.w, w.z, 0x05040100));
}
__device__ __forceinline__ f32x4v mma16x3(uint4 a, uint2 bhi, uint2 blo, f32x4v c) {
  uint2 hi, lo;
  unzip4(a, hi, lo);
  c = mma16(lo, bhi, c);
  c = mma16(hi, blo, c);
  return mma16(hi, bhi, c);
}

template <int ST, int V, int T, int W>
__global__ void __launch_bounds__(64 * W, T == 4 ? 3 : 4) tree_gdn_mfma_kernel(GdnArgs a) {
  constexpr int kN = 16 * T, K = 128, CT = V / (16 * W), SF = kN + 4, TH = 64 * W;   // CT columns a lane
  // q and k: rows of 16 pieces, piece p of row r at p ^ (r % 16).  Once every wave
  // has its products of them, split1 words of -low (below the diagonal tiles) and
  // att: 41 KB in all for 64 nodes, three workgroups a CU.
  __shared__ union {
    uint4 qk[2][kN * 16];
    struct {
      uint32_t low[kN][SF], att[kN][SF];
    };
  } s_m;
  auto& s_q = s_m.qk[0];
  auto& s_k = s_m.qk[1];
  auto& s_low = s_m.low;
  auto& s_att = s_m.att;
  __shared__ float s_diag[kN][20];   // -low's diagonal tiles transposed, then their inverses as split1 words
  __shared__ double s_g[64];
  __shared__ float s_beta[64], s_rk[kN], s_rq[kN];
  __shared__ uint64_t s_set[64];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15, quad = lane >> 4;
  uint16_t* out = static_cast<uint16_t*>(a.o);
  if (blockIdx.x >= static_cast<unsigned>(a.R * a.HV)) {   // rows of no request
    tree::clear_rows<TH>(out, a.cu, a.R, a.total, static_cast<int64_t>(a.HV) * V * 2, blockIdx.x - a.R * a.HV,
                         gridDim.x - a.R * a.HV);
    return;
  }
  const int hv = blockIdx.x % a.HV, r = blockIdx.x / a.HV, h = hv / (a.HV / a.H);
  const tree::Span span = tree::span_of(a.cu, r, a.total);
  const int64_t srow = a.rows ? a.rows[r] : r;
  const bool none = srow < 0 || srow >= a.n_rows;
  const int most = a.max_nodes < kN ? a.max_nodes : kN;
  const int n = none ? 0 : static_cast<int>(span.count < most ? span.count : most);
  for (int64_t i = n; i < span.count; ++i)   // no request: zeros; nodes past the most that the call takes: not a number
    for (int c = tid; c < V; c += TH) out[((span.first + i) * a.HV + hv) * V + c] = none ? 0 : 0x7fc0;
  if (n == 0) return;
  const int nt = (n + 15) >> 4;

  // q and k rows (a thread a piece of a row), then the state
  constexpr int kRows = TH / 16, kLoads = (kN + kRows - 1) / kRows;
  uint4 rq[kLoads], rk[kLoads];
#pragma unroll
  for (int t = 0; t < kLoads; ++t) {
    const int i = kRows * t + (tid >> 4);
    const int64_t at = ((span.first + (i < n ? i : 0)) * a.H + h) * K + (tid & 15) * 8;
    rq[t] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + at);
    rk[t] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.k) + at);
    if (i >= n) rq[t] = rk[t] = make_uint4(0, 0, 0, 0);
  }
  const int64_t gat = (span.first + (lane < n ? lane : 0)) * a.HV + hv;
  float gate = 0.f, beta = 0.f;
  int up = -1;
  if (w == 0) {
    if (lane < n) up = a.parents ? a.parents[span.first + lane] : lane - 1;
    gate = lane < n ? load_any(a.g, gat, a.g_dt) : 0.f;
    beta = lane < n ? load_any(a.beta, gat, a.beta_dt) : 0.f;
  }
  const int col = w * 16 * CT + n16 * CT;
  float sv[4][8][CT];
  const int64_t sat = (srow * a.HV + hv) * K * V + col;
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t at = sat + (32 * s + 8 * quad + j) * V;
      if constexpr (ST == YH_F32) {
        typedef float ldv __attribute__((ext_vector_type(CT)));
        const ldv x = __builtin_nontemporal_load(reinterpret_cast<const ldv*>(static_cast<const float*>(a.state) + at));
#pragma unroll
        for (int c = 0; c < CT; ++c) sv[s][j][c] = x[c];
      } else {
        typedef _Float16 ldv __attribute__((ext_vector_type(CT)));
        const ldv x = __builtin_nontemporal_load(reinterpret_cast<const ldv*>(static_cast<const _Float16*>(a.state) + at));
#pragma unroll
        for (int c = 0; c < CT; ++c) sv[s][j][c] = static_cast<float>(x[c]);
      }
    }
  typedef uint16_t vcol __attribute__((ext_vector_type(CT)));
  vcol vv[T][4];   // the lane's values
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 16 * t + 4 * quad + e;
      vv[t][e] = *reinterpret_cast<const vcol*>(static_cast<const uint16_t*>(a.v) + ((span.first + (i < n ? i : 0)) * a.HV + hv) * V + col);
    }
  if (w == 0) {
    double sum = log_decay(gate);
    s_set[lane] = tree::ancestors_of(up, &sum);
    s_g[lane] = sum;
    s_beta[lane] = beta;
  }
#pragma unroll
  for (int t = 0; t < kLoads; ++t) {
    const int i = kRows * t + (tid >> 4), p = i * 16 + ((tid & 15) ^ (i & 15));
    if (kN % kRows && i >= kN) break;
    s_q[p] = rq[t];
    s_k[p] = rk[t];
    float sums[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint4 y = x ? rk[t] : rq[t];
      const uint32_t word[4] = {y.x, y.y, y.z, y.w};
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float lo = __uint_as_float(word[e] << 16), hi = __uint_as_float(word[e] & 0xffff0000u);
        sum = fmaf(lo, lo, fmaf(hi, hi, sum));
      }
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
      sums[x] = a.l2 ? rsqrtf(sum + 1e-6f) : 1.f;
    }
    if ((tid & 15) == 0) {
      s_rq[i] = a.scale * sums[0];
      s_rk[i] = sums[1];
    }
  }
  __syncthreads();

  auto operand = [&](const uint4* m, int t, int s) {   // rows of tile t, columns 32 s + 8 quad ..
    return __builtin_bit_cast(bf16x8_t, m[(16 * t + n16) * 16 + ((4 * s + quad) ^ n16)]);
  };
  // k S and q S
  f32x4v ks[T][CT], qs[T][CT];
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int c = 0; c < CT; ++c) ks[t][c] = qs[t][c] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    bf16x8_t hi[CT], lo[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      uint32_t x[4], y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) pair2(sv[s][2 * j][c], sv[s][2 * j + 1][c], x[j], y[j]);
      hi[c] = __builtin_bit_cast(bf16x8_t, make_uint4(x[0], x[1], x[2], x[3]));
      lo[c] = __builtin_bit_cast(bf16x8_t, make_uint4(y[0], y[1], y[2], y[3]));
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {
      if (t >= nt) break;
      const bf16x8_t k8 = operand(s_k, t, s), q8 = operand(s_q, t, s);
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        ks[t][c] = mma32(k8, lo[c], ks[t][c]);
        ks[t][c] = mma32(k8, hi[c], ks[t][c]);
        qs[t][c] = mma32(q8, lo[c], qs[t][c]);
        qs[t][c] = mma32(q8, hi[c], qs[t][c]);
      }
    }
  }
  // The branches above end right behind matrix instructions, and where they meet the
  // compiler (LLVM 22) misses the wait for their results: nothing reads them before this.
  asm volatile("s_nop 7\n\ts_nop 7");
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int c = 0; c < CT; ++c) asm volatile("" : "+v"(ks[t][c]), "+v"(qs[t][c]));
  // k k^T and q k^T, a wave every W-th pair of tiles
  constexpr int kPairs = T * (T + 1) / 2, kMine = (kPairs + W - 1) / W;
  f32x4v kk[kMine], qk[kMine];
  auto tile_a = [](int pair) { return (pair >= 1) + (pair >= 3) + (pair >= 6); };
#pragma unroll
  for (int x = 0; x < kMine; ++x) {
    const int pair = W * x + w, ta = tile_a(pair), tb = pair - ta * (ta + 1) / 2;
    kk[x] = qk[x] = f32x4v{0.f, 0.f, 0.f, 0.f};
    if (pair >= kPairs || ta >= nt) continue;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const bf16x8_t b = operand(s_k, tb, s);
      kk[x] = mma32(operand(s_k, ta, s), b, kk[x]);
      qk[x] = mma32(operand(s_q, ta, s), b, qk[x]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < kMine; ++x) {
    const int pair = W * x + w, ta = tile_a(pair), tb = pair - ta * (ta + 1) / 2;
    if (pair >= kPairs || ta >= nt) continue;
    const int j = 16 * tb + n16;
    const float rkj = s_rk[j];
    const double gj = s_g[j];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 16 * ta + 4 * quad + e;
      const bool above = (s_set[i] >> j) & 1;
      const float f = above ? __expf(static_cast<float>(s_g[i] - gj)) * rkj : 0.f;
      kk[x][e] = above && i != j ? -s_beta[i] * s_rk[i] * f * kk[x][e] : 0.f;
      if (ta != tb) s_low[i][j] = split1(kk[x][e]);
      s_att[i][j] = above ? split1(s_rq[i] * f * qk[x][e]) : 0u;
    }
    if (ta == tb) *reinterpret_cast<f32x4v*>(&s_diag[16 * ta + n16][4 * quad]) = kk[x];
  }
  __syncthreads();
  if (w == 0 && quad < nt) {   // the diagonal tiles' inverses: a lane a column
    const int b = 16 * quad;
    float x[16];
    f32x4v l[2][4];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = i == n16 ? 1.f : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) l[0][i] = *reinterpret_cast<const f32x4v*>(&s_diag[b][4 * i]);
#pragma unroll
    for (int m = 0; m < 15; ++m) {
#pragma unroll
      for (int i = (m + 2) / 4; i < 4; ++i) l[(m + 1) & 1][i] = *reinterpret_cast<const f32x4v*>(&s_diag[b + m + 1][4 * i]);
      // what is not finite stays in its row, whose u then marks the descendants
      const float f = fabsf(x[m]) < INFINITY ? x[m] : 0.f;
#pragma unroll
      for (int i = m + 1; i < 16; ++i) x[i] = fmaf(l[m & 1][i >> 2][i & 3], f, x[i]);
      asm volatile("" ::: "memory");   // one column ahead, not all
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s_diag[b + i][n16] = __uint_as_float(split1(x[i]));
  }
  __syncthreads();

  uint2 uhi[T][CT], ulo[T][CT];
  uint64_t bad[CT] = {};
#pragma unroll
  for (int b = 0; b < T; ++b) {
    if (b >= nt) break;
    float ge[4], bt[4];
    f32x4v x[CT];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 16 * b + 4 * quad + e;
      ge[e] = __expf(static_cast<float>(s_g[i]));
      bt[e] = s_beta[i];
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const float y = bt[e] * (bf16_to_f32(vv[b][e][c]) - ge[e] * s_rk[i] * ks[b][c][e]);
        x[c][e] = i < n ? y : 0.f;
      }
    }
#pragma unroll
    for (int ta = 0; ta < b; ++ta) {
      const uint4 l = *reinterpret_cast<const uint4*>(&s_low[16 * b + n16][16 * ta + 4 * quad]);
#pragma unroll
      for (int c = 0; c < CT; ++c) x[c] = mma16x3(l, uhi[ta][c], ulo[ta][c], x[c]);
    }
    // elements that are not finite: 0, and their bit
    auto pack = [&](f32x4v& y, int c, uint2& hi, uint2& lo) {
      uint32_t off = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!(fabsf(y[e]) < INFINITY)) {
          off |= 1u << e;
          y[e] = 0.f;
        }
      bad[c] |= static_cast<uint64_t>(off) << (16 * b + 4 * quad);
      pair2(y[0], y[1], hi.x, lo.x);
      pair2(y[2], y[3], hi.y, lo.y);
    };
    const uint4 inv = *reinterpret_cast<const uint4*>(&s_diag[16 * b + n16][4 * quad]);
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      uint2 hi, lo;
      pack(x[c], c, hi, lo);
      f32x4v u = mma16x3(inv, hi, lo, f32x4v{0.f, 0.f, 0.f, 0.f});
      pack(u, c, uhi[b][c], ulo[b][c]);
    }
    uint64_t any = bad[0];
    if constexpr (CT == 2) any |= bad[1];
    bool lost[CT][4] = {};
    if (__any(any != 0)) {
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        bad[c] |= __shfl_xor(bad[c], 16, 64);
        bad[c] |= __shfl_xor(bad[c], 32, 64);
#pragma unroll
        for (int e = 0; e < 4; ++e) lost[c][e] = (bad[c] & s_set[16 * b + 4 * quad + e]) != 0;
      }
    }
    f32x4v o[CT];
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int c = 0; c < CT; ++c) o[c][e] = ge[e] * s_rq[16 * b + 4 * quad + e] * qs[b][c][e];
#pragma unroll
    for (int ta = 0; ta <= b; ++ta) {
      const uint4 l = *reinterpret_cast<const uint4*>(&s_att[16 * b + n16][16 * ta + 4 * quad]);
#pragma unroll
      for (int c = 0; c < CT; ++c) o[c] = mma16x3(l, uhi[ta][c], ulo[ta][c], o[c]);
    }
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[c][e] = lost[c][e] ? NAN : o[c][e];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 16 * b + 4 * quad + e;
      if (i >= n) continue;
      uint16_t* to = out + ((span.first + i) * a.HV + hv) * V + col;
      if constexpr (CT == 2)
        *reinterpret_cast<uint32_t*>(to) = attn::Mfma<YH_BF16>::round2(o[0][e], o[1][e]);
      else
        *to = f32_to_bf16(o[0][e]);
    }
  }
}

template <int ST, int V>
void launch_mfma(const GdnArgs& a, unsigned grid, hipStream_t st) {
  // Up to 32 nodes a wave takes 16 columns.  Past them V / 4: eight waves of four tiles each spill (128 requests of up
  // to 64 nodes x 32 heads: 213 us for 110).
  if (a.max_nodes <= 16) hipLaunchKernelGGL((tree_gdn_mfma_kernel<ST, V, 1, V / 16>), dim3(grid), dim3(V * 4), 0, st, a);
  else if (a.max_nodes <= 32) hipLaunchKernelGGL((tree_gdn_mfma_kernel<ST, V, 2, V / 16>), dim3(grid), dim3(V * 4), 0, st, a);
  else hipLaunchKernelGGL((tree_gdn_mfma_kernel<ST, V, 4, 4>), dim3(grid), dim3(256), 0, st, a);
}

// ---------------------------------------------------------------------------
struct ConvTreeArgs {
  const uint16_t* proj;     // [N, P], the first C columns
  int64_t P;
  const uint16_t* window;   // [R, 3, C], oldest first
  const uint16_t* w;        // [C, 4]
  const int32_t* parents;   // [N] or null: chains
  const int32_t* cu;
  uint16_t* y;              // [C / Cp, N, Cp]
  int64_t C, Cp, total;
  int R;
};

// y_i = silu(sum_j w_j x(3 - j steps up the path of node i)).  Bound by HBM: a
// workgroup takes 32 VEC channels of a request, brings the window and the nodes'
// inputs into LDS once (every row is read by up to four nodes: from L1 and L2
// that took 73 us for 50, 4.7 TB/s, at 128 requests of 8 to 64 nodes x 12288
// channels), and each eighth of it a node at a time, a lane VEC channels.
template <int VEC>
__global__ void __launch_bounds__(256) conv_tree_kernel(ConvTreeArgs a) {
  using Ch = Chan<VEC>;
  typedef typename Ch::T T;
  constexpr int kN = tree::kNodes, kGroups = 8;
  __shared__ T s_x[kN + 3][32];      // the nodes, then the window
  __shared__ int s_up[3][kN];        // rows of s_x 1, 2 and 3 steps up
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5, r = blockIdx.y;
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * 32 + lane) * VEC;
  const bool in = c < a.C;
  const int64_t plane = c / a.Cp;
  T* dst = reinterpret_cast<T*>(a.y + plane * a.total * a.Cp + (c - plane * a.Cp));
  const int64_t yc = a.Cp / VEC, sp = a.P / VEC, sc = a.C / VEC;
  if (r == a.R) {   // rows of no request
    const int64_t end = a.R ? a.cu[a.R] : 0;
    if (in)
      for (int64_t i = (end < 0 ? 0 : end) + grp; i < a.total; i += kGroups) dst[i * yc] = T{};
    return;
  }
  const tree::Span span = tree::span_of(a.cu, r, a.total);
  const int n = static_cast<int>(span.count < kN ? span.count : kN);
  if (n == 0) return;
  const T* src = reinterpret_cast<const T*>(a.proj + span.first * a.P + c);
  T x[kN / kGroups];
#pragma unroll
  for (int u = 0; u < kN / kGroups; ++u)
    if (in && u * kGroups + grp < n) x[u] = src[(u * kGroups + grp) * sp];
  if (in && grp < 3) s_x[kN + grp][lane] = reinterpret_cast<const T*>(a.window + static_cast<int64_t>(r) * 3 * a.C + c)[grp * sc];
  if (threadIdx.x < 64) {
    const int node = threadIdx.x;
    int up = -1;
    if (node < n) up = a.parents ? a.parents[span.first + node] : node - 1;
    if (up >= node || up < 0) up = -1;
    int two = __shfl(up, up < 0 ? 0 : up, 64);
    if (up < 0) two = up - 1;
    int three = __shfl(up, two < 0 ? 0 : two, 64);
    if (two < 0) three = two - 1;
    s_up[0][node] = up < 0 ? kN + 3 + up : up;   // -1, -2, -3: the window from its end
    s_up[1][node] = two < 0 ? kN + 3 + two : two;
    s_up[2][node] = three < 0 ? kN + 3 + three : three;
  }
  uint2 wr[VEC];
  if (in)
#pragma unroll
    for (int i = 0; i < VEC; ++i) wr[i] = reinterpret_cast<const uint2*>(a.w)[c + i];
#pragma unroll
  for (int u = 0; u < kN / kGroups; ++u)
    if (u * kGroups + grp < n) s_x[u * kGroups + grp][lane] = x[u];
  __syncthreads();
  if (!in) return;
  float wt[4][VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    wt[0][i] = __uint_as_float(wr[i].x << 16);
    wt[1][i] = __uint_as_float(wr[i].x & 0xffff0000u);
    wt[2][i] = __uint_as_float(wr[i].y << 16);
    wt[3][i] = __uint_as_float(wr[i].y & 0xffff0000u);
  }
#pragma unroll
  for (int u = 0; u < kN / kGroups; ++u) {
    const int i = u * kGroups + grp;
    if (i >= n) break;
    float y[VEC];
    T t[3];
#pragma unroll
    for (int j = 0; j < 3; ++j) t[j] = s_x[s_up[2 - j][i]][lane];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      float acc = Ch::f32(t[0], v) * wt[0][v];
      acc = fmaf(Ch::f32(t[1], v), wt[1][v], acc);
      acc = fmaf(Ch::f32(t[2], v), wt[2][v], acc);
      acc = fmaf(Ch::f32(x[u], v), wt[3][v], acc);
      // silu on the hardware's exp2 and reciprocal (1 ulp each, far below the rounding to bf16)
      y[v] = acc * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(acc * -1.4426950408889634f));
    }
    dst[(span.first + i) * yc] = Ch::pack(y);
  }
  float nan[VEC];   // nodes past the most: not a number
#pragma unroll
  for (int v = 0; v < VEC; ++v) nan[v] = NAN;
  for (int64_t i = n + grp; i < span.count; i += kGroups) dst[(span.first + i) * yc] = Ch::pack(nan);
}

}  // namespace
}  // namespace yh

extern "C" int yh_tree_gated_delta_rule(const void* q, const void* k, const void* v, const void* g, const void* beta,
                                        const int32_t* parents, const int32_t* cu_seqlens, const void* state,
                                        int state_dtype, const int32_t* state_indices, void* o, int64_t n_seqs,
                                        int64_t total, int64_t H, int64_t HV, int64_t K, int64_t V,
                                        int64_t n_state_rows, int64_t max_nodes, float scale, int use_qk_l2norm,
                                        int qkv_dtype, int g_dtype, int beta_dtype, yh_stream_t stream) {
  using namespace yh;
  YH_CHECK_ARG(n_seqs >= 0 && total >= 0 && n_state_rows >= 0 && H > 0 && HV > 0, "tree_gated_delta_rule: bad sizes");
  YH_CHECK_ARG(HV % H == 0, "tree_gated_delta_rule: HV must be a multiple of H");
  YH_CHECK_ARG((K == 64 || K == 128) && (V == 64 || V == 128), "tree_gated_delta_rule: K and V must be 64 or 128");
  YH_CHECK_ARG(max_nodes > 0 && max_nodes <= tree::kNodes, "tree_gated_delta_rule: max_nodes must be 1 to %d",
               tree::kNodes);
  YH_CHECK_ARG(is_float_dtype(qkv_dtype) && is_float_dtype(g_dtype) && is_float_dtype(beta_dtype),
               "tree_gated_delta_rule: dtypes must be f32, bf16 or f16");
  YH_CHECK_ARG(state_dtype == YH_F32 || state_dtype == YH_F16, "tree_gated_delta_rule: state must be f32 or f16");
  if (total == 0) return YH_OK;
  YH_CHECK_ARG(q && k && v && g && beta && o && (cu_seqlens || n_seqs == 0) && (state || n_state_rows == 0),
               "tree_gated_delta_rule: null pointer");
  YH_CHECK_ARG(state_indices || n_state_rows >= n_seqs, "tree_gated_delta_rule: fewer state rows than requests");
  YH_CHECK_ARG(total < (1ll << 31) && HV < (1ll << 20) && n_seqs * HV < (1ll << 23),
               "tree_gated_delta_rule: sizes too large");
  GdnArgs a{q, k, v, g, beta, parents, cu_seqlens, state, state_indices, o, total, n_state_rows, (int)n_seqs, (int)H,
            (int)HV, (int)max_nodes, use_qk_l2norm ? 1 : 0, qkv_dtype, g_dtype, beta_dtype, state_dtype, scale};
  const unsigned grid = static_cast<unsigned>(n_seqs * HV + tree::clearing(total, HV * V * (qkv_dtype == YH_F32 ? 4 : 2)));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool mfma = K == 128 && qkv_dtype == YH_BF16 && tree::aligned16(q) && tree::aligned16(k) &&
                    tree::aligned16(state) && ((reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(o)) & 3) == 0;
  if (mfma && state_dtype == YH_F32 && V == 128) launch_mfma<YH_F32, 128>(a, grid, st);
  else if (mfma && state_dtype == YH_F32) launch_mfma<YH_F32, 64>(a, grid, st);
  else if (mfma && V == 128) launch_mfma<YH_F16, 128>(a, grid, st);
  else if (mfma) launch_mfma<YH_F16, 64>(a, grid, st);
  else if (K == 128 && V == 128) hipLaunchKernelGGL((tree_gdn_any_kernel<128, 128>), dim3(grid), dim3(256), 0, st, a);
  else if (K == 128) hipLaunchKernelGGL((tree_gdn_any_kernel<128, 64>), dim3(grid), dim3(256), 0, st, a);
  else if (V == 128) hipLaunchKernelGGL((tree_gdn_any_kernel<64, 128>), dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((tree_gdn_any_kernel<64, 64>), dim3(grid), dim3(256), 0, st, a);
  YH_CHECK_LAUNCH("tree_gated_delta_rule");
  return YH_OK;
}

extern "C" int yh_conv_tree(const void* proj, int64_t proj_stride, const void* window, const void* conv_w,
                            const int32_t* parents, const int32_t* cu_seqlens, int64_t n_seqs, int64_t total,
                            int64_t channels, int64_t planes, void* out, int dtype, yh_stream_t stream) {
  using namespace yh;
  YH_CHECK_ARG(n_seqs >= 0 && total >= 0 && channels > 0 && proj_stride >= channels, "conv_tree: bad sizes");
  YH_CHECK_ARG(dtype == YH_BF16, "conv_tree: activations must be bfloat16");
  YH_CHECK_ARG(planes > 0 && channels % planes == 0, "conv_tree: planes must divide the channels");
  if (total == 0) return YH_OK;
  YH_CHECK_ARG(proj && out && conv_w && ((window && cu_seqlens) || n_seqs == 0), "conv_tree: null pointer");
  YH_CHECK_ARG(total < (1ll << 31) && n_seqs < 65535 && channels < (1ll << 24), "conv_tree: sizes too large");
  YH_CHECK_ARG((reinterpret_cast<uintptr_t>(conv_w) & 7) == 0, "conv_tree: conv_w must be 8-byte aligned");
  const bool vec = channels / planes % 8 == 0 && proj_stride % 8 == 0 && tree::aligned16(proj) &&
                   tree::aligned16(window) && tree::aligned16(out);
  const int64_t per_block = 32 * (vec ? 8 : 1), cb = (channels + per_block - 1) / per_block;
    ConvTreeArgs a{static_cast<const uint16_t*>(proj), proj_stride, static_cast<const uint16_t*>(window),
                 static_cast<const uint16_t*>(conv_w), parents, cu_seqlens, static_cast<uint16_t*>(out), channels,
                 channels / planes, total, (int)n_seqs};
  const dim3 grid(static_cast<unsigned>(cb), static_cast<unsigned>(n_seqs + 1));   // neighbours read on in the same rows
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (vec) hipLaunchKernelGGL(conv_tree_kernel<8>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(conv_tree_kernel<1>, grid, dim3(256), 0, st, a);
  YH_CHECK_LAUNCH("conv_tree");
  return YH_OK;
}
