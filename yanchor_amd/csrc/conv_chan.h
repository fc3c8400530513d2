// Channels of the depthwise conv: 16-byte groups and the SiLU, shared by the
// prompt and the drafted-tree form.
#pragma once
#include "attn_tile.h"

namespace yh {

__device__ __forceinline__ float silu(float x) { return x / (1.f + expf(-x)); }

// VEC consecutive bf16 channels of a row: 16 bytes in one access (VEC = 8),
// or one element where a row does not keep 16-byte alignment (VEC = 1).
template <int VEC>
struct Chan;
template <>
struct Chan<8> {
  typedef uint4 T;
  static __device__ __forceinline__ float f32(const T& x, int i) {
    const uint32_t w = i < 2 ? x.x : i < 4 ? x.y : i < 6 ? x.z : x.w;
    return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ T pack(const float (&y)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = attn::Mfma<YH_BF16>::round2(y[2 * i], y[2 * i + 1]);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Chan<1> {
  typedef uint16_t T;
  static __device__ __forceinline__ float f32(const T& x, int) { return bf16_to_f32(x); }
  static __device__ __forceinline__ T pack(const float (&y)[1]) { return f32_to_bf16(y[0]); }
};

}  // namespace yh
