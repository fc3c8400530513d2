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
// Bound by HBM: heads are read and written once.  A wave takes heads of one token,
// eight elements a lane; its lanes form the token's angles, one or two each, once.
#include "common.h"
#include "tree.h"

namespace yh {
namespace {

constexpr int kAxes = 4;
constexpr int kWaves = 4;
constexpr int kPairs = 128;     // most pairs of a head

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
  int H, G, half, axes, interleaved, plus_one, shares;
  int begin[kAxes + 1];                // sections: the first pair of each axis
  float eps;
};

__device__ __forceinline__ int axis_of(const RopeArgs& a, int j) {
  if (a.axes == 1) return 0;
  if (a.interleaved) {
    const int x = j % a.axes;
    return j < a.axes * (a.begin[x + 1] - a.begin[x]) ? x : 0;
  }
  int x = 0;
#pragma unroll
  for (int i = 1; i < kAxes; ++i) x += i < a.axes && j >= a.begin[i];
  return x;
}

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
  for (int i = 0; i < 4; ++i)
    o[i] = DT == YH_BF16 ? f32_to_bf16(y[2 * i]) | static_cast<uint32_t>(f32_to_bf16(y[2 * i + 1])) << 16
                         : f32_to_f16(y[2 * i]) | static_cast<uint32_t>(f32_to_f16(y[2 * i + 1])) << 16;
  return make_uint4(o[0], o[1], o[2], o[3]);
}

template <int DT, int D>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(RopeArgs a) {
  constexpr int L = D / 8, kHeads = kWave / L;       // lanes of a head, heads of a wave
  __shared__ float2 turns[kWaves][kPairs];
  const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kWaves + w;
  const int64_t n = item / a.shares;
  if (n >= a.N) return;
  const int share = static_cast<int>(item - n * a.shares);
  float2* turn = turns[w];
  for (int j = lane; j < a.half; j += kWave) {
    const double rev = static_cast<double>(a.positions[axis_of(a, j) * a.N + n]) * static_cast<double>(a.freq[j]) *
                       0.15915494309189533577;
    float s, c;
    sincospif(2.f * static_cast<float>(rev - rint(rev)), &s, &c);
    turn[j] = make_float2(c, s);
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const int li = lane % L, e0 = 8 * li;
  const bool rot = e0 < 2 * a.half, upper = e0 >= a.half;
  const int step = a.half / 8, from = rot ? (upper ? lane - step : lane + step) : lane;
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 t = rot ? turn[e0 + i - (upper ? a.half : 0)] : make_float2(1.f, 0.f);
    c[i] = t.x;
    s[i] = upper ? t.y : -t.y;
  }
  float wq[8], wk[8];
  if (a.q_w) wide8<DT>(*reinterpret_cast<const uint4*>(a.q_w + e0), wq);
  if (a.k_w) wide8<DT>(*reinterpret_cast<const uint4*>(a.k_w + e0), wk);
  const float one = a.plus_one ? 1.f : 0.f;
  for (int h0 = share * kHeads; h0 < a.H + a.G; h0 += a.shares * kHeads) {
    const bool in = h0 + lane / L < a.H + a.G;
    const int h = in ? h0 + lane / L : 0;
    const bool key = h >= a.H;
    const int hh = key ? h - a.H : h;
    const uint16_t* src = key ? a.k + n * a.k_ts + hh * a.k_hs : a.q + n * a.q_ts + hh * a.q_hs;
    float y[8];
    wide8<DT>(*reinterpret_cast<const uint4*>(src + e0), y);
    if (key ? a.k_w != nullptr : a.q_w != nullptr) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(y[i], y[i], sum);
#pragma unroll
      for (int off = 1; off < L; off <<= 1) sum += __shfl_xor(sum, off, kWave);
      const float r = 1.f / sqrtf(sum / D + a.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * r * (one + (key ? wk[i] : wq[i]));
    }
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float p = __shfl(y[i], from, kWave);
      o[i] = rot ? fmaf(p, s[i], y[i] * c[i]) : y[i];
    }
    uint16_t* dst = key ? a.k_out + (n * a.G + hh) * D : a.q_out + (n * a.H + hh) * D;
    if (in) *reinterpret_cast<uint4*>(dst + e0) = narrow8<DT>(o);
  }
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
  for (int i = 0; i < axes; ++i) {
    const int64_t n = axes == 1 ? half : sections[i];
    YH_CHECK_ARG(n >= 0 && n <= half, "qk_norm_rope: bad section");
    YH_CHECK_ARG(!interleaved || i == 0 || n == 0 || i + axes * (n - 1) < half,
                 "qk_norm_rope: an interleaved section reaches past the pairs");
    a.begin[i + 1] = a.begin[i] + static_cast<int>(n);
  }
  YH_CHECK_ARG(a.begin[axes] == half, "qk_norm_rope: the sections must add up to half of the rotary dims");
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
  a.axes = static_cast<int>(axes);
  a.interleaved = interleaved ? 1 : 0;
  a.plus_one = plus_one ? 1 : 0;
  a.eps = eps;
  // heads of a token over as many waves as there are for few tokens, one wave for many
  const int64_t rounds = (H + G + 512 / D - 1) / (512 / D), few = 4096 / N;
  a.shares = static_cast<int>(few < 1 ? 1 : few < rounds ? few : rounds);
  const int64_t grid = (N * a.shares + kWaves - 1) / kWaves;
  YH_CHECK_ARG(grid < (1ll << 24), "qk_norm_rope: sizes too large");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == YH_BF16) launch<YH_BF16>(a, D, static_cast<unsigned>(grid), st);
  else launch<YH_F16>(a, D, static_cast<unsigned>(grid), st);
  YH_CHECK_LAUNCH("qk_norm_rope");
  return YH_OK;
}
