// Norms of query and key heads with rotary positions of several axes, one pass.
//
//   y = x / sqrt(mean(x^2) + eps) * (1 + w)                      (a head of D)
//   (y_j, y_{j + R/2}) turned by the angle p_{axis(j)} f_j,      j < R / 2
// with positions p [axes, N] (time, height, width, ...) and frequencies f.  Axis a
// has sections[a] of the R / 2 pairs, one section behind the other, or interleaved:
// pair j is of axis j mod axes while that axis has pairs left, of axis 0 otherwise.
//
// Everything is float32 and rounded once, but for the angle: a position of a
// million times a frequency of one leaves float32 an error of 0.06, so the product
// and its reduction to one turn are float64, and sine and cosine take the turn's
// rest in float32 (2^-25 of a turn).
//
// Bound by HBM, heads are read and written once: 65521 tokens of 40 heads of 128 in
// 231 us, 5.8 TB/s.  A wave takes heads of one token, eight elements a lane; its lanes
// form the token's angles, one or two each, once, and exchange them through LDS.
// (296 us with a square root and a division a head, weights and angles applied one
// after the other, sums by LDS shuffles and one load ahead: 210 instructions for four
// heads, of which the memory leaves time for about 150.)
#include "attn_tile.h"
#include "tree.h"

namespace yh {
namespace {

constexpr int kAxes = 4;
constexpr int kWaves = 4;
constexpr int kPairs = 128;     // most pairs of a head

typedef unsigned u4 __attribute__((ext_vector_type(4)));

struct RopeArgs {
  const uint16_t* q;
  const uint16_t* k;
  int64_t q_ts, q_hs, k_ts, k_hs;      // token and head strides
  const uint16_t* q_w;                 // [D], or null: no norm
  const uint16_t* k_w;
  const int64_t* positions;            // [axes, N]
  const float* freq;                   // [R / 2]
  uint16_t* q_out;                     // dense [N, H, D], [N, G, D]
  uint16_t* k_out;
  int64_t N;
  int H, G, half, plus_one, shares;
  uint64_t axis[kPairs / 32];          // of each pair, two bits
  float eps;
};

template <int DT>
__device__ __forceinline__ void wide8(uint4 x, float* y) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[2 * i] = DT == YH_BF16 ? __uint_as_float(w[i] << 16) : f16_to_f32(w[i] & 0xffff);
    y[2 * i + 1] = DT == YH_BF16 ? __uint_as_float(w[i] & 0xffff0000u) : f16_to_f32(w[i] >> 16);
  }
}
template <int DT>
__device__ __forceinline__ uint4 narrow8(const float* y) {
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = attn::Mfma<DT>::round2(y[2 * i], y[2 * i + 1]);
  return make_uint4(o[0], o[1], o[2], o[3]);
}

template <int CTRL>
__device__ __forceinline__ float lanes_add(float x) {
  return x + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, true));
}
// Sum over the L lanes of a head.
template <int L>
__device__ __forceinline__ float head_sum(float x) {
  x = lanes_add<0xB1>(x);     // quad_perm [1, 0, 3, 2]
  x = lanes_add<0x4E>(x);     // quad_perm [2, 3, 0, 1]
  x = lanes_add<0x141>(x);    // row_half_mirror
  if constexpr (L >= 16) x = lanes_add<0x140>(x);    // row_mirror
  if constexpr (L == 32) x += __shfl_xor(x, 16, kWave);
  return x;
}

// Groups first, first + shares, ... of `count` heads, kWave / L heads each, kAhead of them loaded before the first is
// used.  With c, s cosine and signed sine, w the weights, o_i = r (x_i c_i w_i + x_p s_i w_p), p the other of the pair:
// the products of c, s and w are the token's.
template <int DT, int D>
__device__ __forceinline__ void turn_heads(const RopeArgs& a, const uint16_t* src, int64_t stride, uint16_t* dst, int count,
                                           int first, const uint16_t* weight, const float (&c)[8], const float (&s)[8],
                                           bool rot, bool upper, int from) {
  constexpr int L = D / 8, kHeads = kWave / L, kAhead = 4;
  const int groups = (count + kHeads - 1) / kHeads;
  if (first >= groups) return;
  const int lane = threadIdx.x & (kWave - 1), li = lane % L, e0 = 8 * li;
  float cw[8], sw[8];
  if (weight) {
    float w[8], wp[8];
    wide8<DT>(*reinterpret_cast<const uint4*>(weight + e0), w);
    wide8<DT>(*reinterpret_cast<const uint4*>(weight + (rot ? (upper ? e0 - a.half : e0 + a.half) : e0)), wp);
    const float one = a.plus_one ? 1.f : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      cw[i] = c[i] * (one + w[i]);
      sw[i] = s[i] * (one + wp[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      cw[i] = c[i];
      sw[i] = s[i];
    }
  }
  for (int g0 = first; g0 < groups; g0 += kAhead * a.shares) {
    uint4 x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int h = (g0 + u * a.shares) * kHeads + lane / L;
      x[u] = make_uint4(0, 0, 0, 0);
      if (h < count) {
        const u4 y = __builtin_nontemporal_load(reinterpret_cast<const u4*>(src + h * stride + e0));
        x[u] = make_uint4(y[0], y[1], y[2], y[3]);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int h = (g0 + u * a.shares) * kHeads + lane / L;
      if ((g0 + u * a.shares) >= groups) break;
      float y[8], p[8];
      wide8<DT>(x[u], y);
      uint4 xp;
      xp.x = __shfl(x[u].x, from, kWave);
      xp.y = __shfl(x[u].y, from, kWave);
      xp.z = __shfl(x[u].z, from, kWave);
      xp.w = __shfl(x[u].w, from, kWave);
      if (!rot) xp = make_uint4(0, 0, 0, 0);
      wide8<DT>(xp, p);
      float r = 1.f;
      if (weight) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(y[i], y[i], sum);
        r = rsqrtf(head_sum<L>(sum) * (1.f / D) + a.eps);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = fmaf(p[i], sw[i], y[i] * cw[i]) * r;
      if (h < count) {
        const uint4 o = narrow8<DT>(y);
        __builtin_nontemporal_store(u4{o.x, o.y, o.z, o.w}, reinterpret_cast<u4*>(dst + static_cast<int64_t>(h) * D + e0));
      }
    }
  }
}

template <int DT, int D>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(RopeArgs a) {
  constexpr int L = D / 8, kHeads = kWave / L;       // lanes of a head, heads of a wave
  __shared__ float2 turns[kWaves][kPairs];
  const int lane = threadIdx.x & (kWave - 1), w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kWaves + w;
  const int64_t n = a.shares == 1 ? item : item / a.shares;
  if (n >= a.N) return;
  const int share = static_cast<int>(item - n * a.shares);
  float2* turn = turns[w];
#pragma unroll
  for (int k = 0; k < D / 128 + (D < 128); ++k) {
    const int j = lane + k * kWave;
    if (j < a.half) {
      const int axis = static_cast<int>((lane < 32 ? a.axis[2 * k] : a.axis[2 * k + 1]) >> (2 * (lane & 31))) & 3;
      const double rev = static_cast<double>(a.positions[axis * a.N + n]) * static_cast<double>(a.freq[j]) *
                         0.15915494309189533577;
      float s, c;
      sincospif(2.f * static_cast<float>(rev - rint(rev)), &s, &c);
      turn[j] = make_float2(c, s);
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const int e0 = 8 * (lane % L);
  const bool rot = e0 < 2 * a.half, upper = e0 >= a.half;
  const int step = a.half / 8, from = rot ? (upper ? lane - step : lane + step) : lane;
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 t = rot ? turn[e0 + i - (upper ? a.half : 0)] : make_float2(1.f, 0.f);
    c[i] = t.x;
    s[i] = upper ? t.y : -t.y;
  }
  // groups of heads in a row, the queries' and then the keys', go round the token's waves
  turn_heads<DT, D>(a, a.q + n * a.q_ts, a.q_hs, a.q_out + n * a.H * D, a.H, share, a.q_w, c, s, rot, upper, from);
  const int before = (a.H + kHeads - 1) / kHeads % a.shares;
  turn_heads<DT, D>(a, a.k + n * a.k_ts, a.k_hs, a.k_out + n * a.G * D, a.G,
                    share >= before ? share - before : share - before + a.shares, a.k_w, c, s, rot, upper, from);
}

template <int DT>
void launch(const RopeArgs& a, int64_t D, unsigned grid, hipStream_t st) {
  if (D == 64) hipLaunchKernelGGL((qk_norm_rope_kernel<DT, 64>), dim3(grid), dim3(kWaves * kWave), 0, st, a);
  else if (D == 128) hipLaunchKernelGGL((qk_norm_rope_kernel<DT, 128>), dim3(grid), dim3(kWaves * kWave), 0, st, a);
  else hipLaunchKernelGGL((qk_norm_rope_kernel<DT, 256>), dim3(grid), dim3(kWaves * kWave), 0, st, a);
}

}  // namespace
}  // namespace yh

extern "C" int yh_qk_norm_rope(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                               int64_t k_token_stride, int64_t k_head_stride, const void* q_w, const void* k_w,
                               const int64_t* positions, const float* freq, const int64_t* sections, int64_t axes,
                               int interleaved, void* q_out, void* k_out, int64_t N, int64_t H, int64_t G, int64_t D,
                               int64_t rotary_dim, float eps, int plus_one, int dtype, yh_stream_t stream) {
  using namespace yh;
  YH_CHECK_ARG(N >= 0 && H >= 0 && G >= 0, "qk_norm_rope: bad sizes");
  YH_CHECK_ARG(D == 64 || D == 128 || D == 256, "qk_norm_rope: head dim must be 64, 128 or 256");
  YH_CHECK_ARG(rotary_dim >= 0 && rotary_dim <= D && rotary_dim % 16 == 0,
               "qk_norm_rope: rotary dims must be a multiple of 16 up to the head dim");
  YH_CHECK_ARG(axes >= 1 && axes <= kAxes, "qk_norm_rope: 1 to %d axes", kAxes);
  YH_CHECK_ARG(eps >= 0.f && eps < INFINITY, "qk_norm_rope: eps must not be negative");
  if (dtype != YH_BF16 && dtype != YH_F16) {
    set_error("qk_norm_rope: dtype must be bf16 or fp16");
    return YH_ERR_UNSUPPORTED;
  }
  RopeArgs a{};
  const int64_t half = rotary_dim / 2;
  YH_CHECK_ARG(sections || axes == 1, "qk_norm_rope: several axes need their sections");
  int64_t begin[kAxes + 1] = {};
  for (int i = 0; i < axes; ++i) {
    const int64_t n = axes == 1 ? half : sections[i];
    YH_CHECK_ARG(n >= 0 && n <= half, "qk_norm_rope: bad section");
    YH_CHECK_ARG(!interleaved || i == 0 || n == 0 || i + axes * (n - 1) < half,
                 "qk_norm_rope: an interleaved section reaches past the pairs");
    begin[i + 1] = begin[i] + n;
  }
  YH_CHECK_ARG(begin[axes] == half, "qk_norm_rope: the sections must add up to half of the rotary dims");
  for (int64_t j = 0; j < half; ++j) {
    int64_t x = 0;
    if (interleaved) x = j < axes * (begin[j % axes + 1] - begin[j % axes]) ? j % axes : 0;
    else while (j >= begin[x + 1]) ++x;
    a.axis[j / 32] |= static_cast<uint64_t>(x) << (2 * (j % 32));
  }
  if (N == 0 || H + G == 0) return YH_OK;
  YH_CHECK_ARG((q && q_out) || H == 0, "qk_norm_rope: null pointer");
  YH_CHECK_ARG((k && k_out) || G == 0, "qk_norm_rope: null pointer");
  YH_CHECK_ARG((positions && freq) || half == 0, "qk_norm_rope: null pointer");
  YH_CHECK_ARG(tree::aligned16(q) && tree::aligned16(k) && tree::aligned16(q_w) && tree::aligned16(k_w) &&
                   tree::aligned16(q_out) && tree::aligned16(k_out) && q_token_stride % 8 == 0 &&
                   q_head_stride % 8 == 0 && k_token_stride % 8 == 0 && k_head_stride % 8 == 0,
               "qk_norm_rope: heads must be 16-byte aligned");
  YH_CHECK_ARG(N < (1ll << 31) && H < (1ll << 20) && G < (1ll << 20), "qk_norm_rope: sizes too large");
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.q_ts = q_token_stride;
  a.q_hs = q_head_stride;
  a.k_ts = k_token_stride;
  a.k_hs = k_head_stride;
  a.q_w = static_cast<const uint16_t*>(q_w);
  a.k_w = static_cast<const uint16_t*>(k_w);
  a.positions = positions;
  a.freq = freq;
  a.q_out = static_cast<uint16_t*>(q_out);
  a.k_out = static_cast<uint16_t*>(k_out);
  a.N = N;
  a.H = static_cast<int>(H);
  a.G = static_cast<int>(G);
  a.half = static_cast<int>(half);
  a.plus_one = plus_one ? 1 : 0;
  a.eps = eps;
  // heads of a token over as many waves as there are for few tokens, one wave for many
  const int64_t each = 512 / D, rounds = (H + each - 1) / each + (G + each - 1) / each, few = 4096 / N;
  a.shares = static_cast<int>(few < 1 ? 1 : few < rounds ? few : rounds);
  const int64_t grid = (N * a.shares + kWaves - 1) / kWaves;
  YH_CHECK_ARG(grid < (1ll << 24), "qk_norm_rope: sizes too large");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == YH_BF16) launch<YH_BF16>(a, D, static_cast<unsigned>(grid), st);
  else launch<YH_F16>(a, D, static_cast<unsigned>(grid), st);
  YH_CHECK_LAUNCH("qk_norm_rope");
  return YH_OK;
}
