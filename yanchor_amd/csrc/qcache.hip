// Rows into a quantised block cache, and rows of a cache back (qcache.h).
//
// Write: s = the smallest byte with max |x| <= M 2^(s - 127) over a run of 32
// values, M the largest code; code = round_to_nearest_even(x 2^(127 - s)).  No
// value saturates, and since scales are powers of two both the product and what
// is read back are exact but for that one rounding (half a step: 2^-4 of an e4m3
// value, 1/4 of the code's power of two of an e2m1 value).
// Read: value = code 2^(s - 127), rounded to the output's type.
#include "qcache.h"
#include "tree.h"

namespace yh {
namespace {

using namespace qcache;
using tree::Div;

struct Args {
  const uint16_t* k;       // write: rows in, tokens ks / vs apart
  const uint16_t* v;
  int64_t ks, vs;
  uint16_t* k_out;         // read: rows out, dense
  uint16_t* v_out;
  const int64_t* slots;    // [N]
  char* keys;
  char* values;
  uint8_t* key_scales;
  uint8_t* value_scales;
  int64_t N, n_slots;      // n_slots = blocks * block
  Div block, pieces, row;  // a row's pieces of eight values; a head's
  int G;
};

// Where piece p of token t lies: its slot, head and dim, or slot < 0.
struct Place {
  int64_t token, head;     // head: (block id * G + g) * block rows + row, in rows
  int64_t run;             // of its scale byte
  uint32_t p, dim;
  bool in;
};
__device__ __forceinline__ Place place(const Args& a, int64_t i, int64_t n) {
  Place w;
  const int64_t j = i < n ? i : n - 1;
  w.token = j < (1ll << 31) ? a.pieces.quot(static_cast<uint32_t>(j)) : j / a.pieces.d;
  const int64_t slot = a.slots[w.token];
  w.in = i < n && slot >= 0 && slot < a.n_slots;
  w.p = static_cast<uint32_t>(j - w.token * a.pieces.d);
  const uint32_t g = a.row.quot(w.p);
  w.dim = (w.p - g * a.row.d) * 8;
  const int64_t sl = w.in ? slot : 0;
  const int64_t b = sl < (1ll << 31) ? a.block.quot(static_cast<uint32_t>(sl)) : sl / a.block.d;
  const int64_t row = sl - b * a.block.d;
  w.head = (b * a.G + g) * a.block.d + row;
  w.run = ((b * a.G + g) * (a.row.d / 4) + w.dim / kRun) * a.block.d + row;
  return w;
}

template <int DT>
__device__ __forceinline__ void widen8(uint4 x, float* y) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[2 * i] = DT == YH_BF16 ? __uint_as_float(w[i] << 16) : f16_to_f32(w[i] & 0xffff);
    y[2 * i + 1] = DT == YH_BF16 ? __uint_as_float(w[i] & 0xffff0000u) : f16_to_f32(w[i] >> 16);
  }
}

// Eight values into their codes and, by the first of a run's four lanes, its scale.
template <int DT, int FMT>
__device__ __forceinline__ void put8(const Args& a, const Place& w, uint4 x, char* codes, uint8_t* scales) {
  float y[8], top = 0.f;
  widen8<DT>(x, y);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // a NaN has the largest bit pattern of all magnitudes
    const float m = __uint_as_float(__float_as_uint(y[i]) & 0x7fffffffu);
    top = __float_as_uint(m) > __float_as_uint(top) ? m : top;
  }
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    const uint32_t other = __shfl_xor(__float_as_uint(top), off, kWave);
    top = other > __float_as_uint(top) ? __uint_as_float(other) : top;
  }
  const int s = scale_of<FMT>(top);
  const float inv = s == kNotANumber ? 0.f : scale_inverse(s);   // such a run reads back as NaN by its scale
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = s == kNotANumber ? 0.f : y[i] * inv;
  if (!w.in) return;
  if constexpr (FMT == kFp8) {
    uint2 c;
    c.x = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    c.x = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c.x, true);
    c.y = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
    c.y = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], c.y, true);
    *reinterpret_cast<uint2*>(codes + w.head * (a.row.d * 8) + w.dim) = c;
  } else {
    uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[0], y[1], 1.f, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[2], y[3], 1.f, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[4], y[5], 1.f, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[6], y[7], 1.f, 3);
    *reinterpret_cast<uint32_t*>(codes + w.head * (a.row.d * 4) + w.dim / 2) = c;
  }
  if (w.dim % kRun == 0) scales[w.run] = static_cast<uint8_t>(s);
}

// Bound by HBM.  A thread takes eight values of the keys and of the values.
template <int DT, int FMT>
__global__ void __launch_bounds__(256) write_kernel(Args a) {
  const int64_t n = a.N * a.pieces.d, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const Place w = place(a, i, n);
  uint4 x = make_uint4(0, 0, 0, 0), y = x;
  if (w.in) {
    x = *reinterpret_cast<const uint4*>(a.k + w.token * a.ks + w.p * 8);
    y = *reinterpret_cast<const uint4*>(a.v + w.token * a.vs + w.p * 8);
  }
  put8<DT, FMT>(a, w, x, a.keys, a.key_scales);
  put8<DT, FMT>(a, w, y, a.values, a.value_scales);
}

template <int DT, int FMT>
__device__ __forceinline__ uint4 get8(const Args& a, const Place& w, const char* codes, const uint8_t* scales) {
  if (!w.in) return make_uint4(0, 0, 0, 0);
  if constexpr (FMT == k16) {
    return *reinterpret_cast<const uint4*>(codes + (w.head * (a.row.d * 8) + w.dim) * 2);
  } else {
    const float s = scale_value(scales[w.run]);
    float y[8];
    if constexpr (FMT == kFp8) {
      const uint2 c = *reinterpret_cast<const uint2*>(codes + w.head * (a.row.d * 8) + w.dim);
      const auto p0 = __builtin_amdgcn_cvt_pk_f32_fp8(c.x, false), p1 = __builtin_amdgcn_cvt_pk_f32_fp8(c.x, true);
      const auto p2 = __builtin_amdgcn_cvt_pk_f32_fp8(c.y, false), p3 = __builtin_amdgcn_cvt_pk_f32_fp8(c.y, true);
      y[0] = p0[0]; y[1] = p0[1]; y[2] = p1[0]; y[3] = p1[1];
      y[4] = p2[0]; y[5] = p2[1]; y[6] = p3[0]; y[7] = p3[1];
    } else {
      const uint32_t c = *reinterpret_cast<const uint32_t*>(codes + w.head * (a.row.d * 4) + w.dim / 2);
      const auto p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 0);
      const auto p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 1);
      const auto p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 2);
      const auto p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 3);
      y[0] = p0[0]; y[1] = p0[1]; y[2] = p1[0]; y[3] = p1[1];
      y[4] = p2[0]; y[5] = p2[1]; y[6] = p3[0]; y[7] = p3[1];
    }
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float lo = y[2 * i] * s, hi = y[2 * i + 1] * s;
      o[i] = DT == YH_BF16 ? f32_to_bf16(lo) | static_cast<uint32_t>(f32_to_bf16(hi)) << 16
                           : f32_to_f16(lo) | static_cast<uint32_t>(f32_to_f16(hi)) << 16;
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
  }
}

template <int DT, int FMT>
__global__ void __launch_bounds__(256) read_kernel(Args a) {
  const int64_t n = a.N * a.pieces.d, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const Place w = place(a, i, n);
  const uint4 x = get8<DT, FMT>(a, w, a.keys, a.key_scales), y = get8<DT, FMT>(a, w, a.values, a.value_scales);
  if (i >= n) return;
  *reinterpret_cast<uint4*>(a.k_out + i * 8) = x;
  *reinterpret_cast<uint4*>(a.v_out + i * 8) = y;
}

int check_cache(const char* what, const void* keys, const void* values, const uint8_t* key_scales,
                const uint8_t* value_scales, const int64_t* slots, int64_t N, int64_t blocks, int64_t G, int64_t D,
                int64_t block, int bits) {
  YH_CHECK_ARG(N >= 0 && blocks >= 0 && G > 0 && D > 0 && block > 0, "%s: bad sizes", what);
  YH_CHECK_ARG(bits == 4 || bits == 8 || bits == 16, "%s: a cache holds 4, 8 or 16 bits a value", what);
  YH_CHECK_ARG(D % (bits == 16 ? 8 : kRun) == 0, "%s: the head dim must be a multiple of %d", what, bits == 16 ? 8 : kRun);
  YH_CHECK_ARG(N < (1ll << 31) && blocks < (1ll << 31) && block < (1ll << 31) && G < (1ll << 31) && D < (1ll << 31) &&
                   G * D < (1ll << 31) && blocks * block < (1ll << 40),
               "%s: sizes too large", what);
  YH_CHECK_ARG((N * (G * D / 8) + 255) / 256 < (1ll << 24), "%s: sizes too large", what);
  if (N == 0) return YH_OK;
  YH_CHECK_ARG(slots && ((keys && values && (bits == 16 || (key_scales && value_scales))) || blocks == 0),
               "%s: null pointer", what);
  YH_CHECK_ARG(tree::aligned16(keys) && tree::aligned16(values), "%s: the cache must be 16-byte aligned", what);
  return YH_OK;
}

Args args_of(const int64_t* slots, const void* keys, const void* values, const uint8_t* key_scales,
             const uint8_t* value_scales, int64_t N, int64_t blocks, int64_t G, int64_t D, int64_t block) {
  Args a{};
  a.slots = slots;
  a.keys = static_cast<char*>(const_cast<void*>(keys));
  a.values = static_cast<char*>(const_cast<void*>(values));
  a.key_scales = const_cast<uint8_t*>(key_scales);
  a.value_scales = const_cast<uint8_t*>(value_scales);
  a.N = N;
  a.n_slots = blocks * block;
  a.block = tree::make_div(static_cast<uint32_t>(block));
  a.pieces = tree::make_div(static_cast<uint32_t>(G * D / 8));
  a.row = tree::make_div(static_cast<uint32_t>(D / 8));
  a.G = static_cast<int>(G);
  return a;
}

}  // namespace
}  // namespace yh

extern "C" int yh_cache_write_quantized(const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                                        const int64_t* slots, void* keys, void* values, uint8_t* key_scales,
                                        uint8_t* value_scales, int64_t N, int64_t blocks, int64_t G, int64_t D,
                                        int64_t block, int bits, int dtype, yh_stream_t stream) {
  using namespace yh;
  YH_CHECK_ARG(bits == 4 || bits == 8, "cache_write_quantized: a quantised cache holds 4 or 8 bits a value");
  YH_CHECK_ARG(dtype == YH_BF16 || dtype == YH_F16, "cache_write_quantized: dtype must be bf16 or f16");
  const int rc = check_cache("cache_write_quantized", keys, values, key_scales, value_scales, slots, N, blocks, G, D,
                             block, bits);
  if (rc != YH_OK || N == 0 || blocks == 0) return rc;
  YH_CHECK_ARG(k && v, "cache_write_quantized: null pointer");
  YH_CHECK_ARG(tree::aligned16(k) && tree::aligned16(v) && k_stride % 8 == 0 && v_stride % 8 == 0 &&
                   k_stride >= G * D && v_stride >= G * D,
               "cache_write_quantized: rows must be 16-byte aligned and hold whole heads");
  Args a = args_of(slots, keys, values, key_scales, value_scales, N, blocks, G, D, block);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.ks = k_stride;
  a.vs = v_stride;
  const dim3 grid(static_cast<unsigned>((N * a.pieces.d + 255) / 256));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == YH_BF16) {
    if (bits == 8) hipLaunchKernelGGL((write_kernel<YH_BF16, kFp8>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((write_kernel<YH_BF16, kFp4>), grid, dim3(256), 0, st, a);
  } else {
    if (bits == 8) hipLaunchKernelGGL((write_kernel<YH_F16, kFp8>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((write_kernel<YH_F16, kFp4>), grid, dim3(256), 0, st, a);
  }
  YH_CHECK_LAUNCH("cache_write_quantized");
  return YH_OK;
}

extern "C" int yh_cache_read(const int64_t* slots, const void* keys, const void* values, const uint8_t* key_scales,
                             const uint8_t* value_scales, void* k, void* v, int64_t N, int64_t blocks, int64_t G,
                             int64_t D, int64_t block, int bits, int dtype, yh_stream_t stream) {
  using namespace yh;
  YH_CHECK_ARG(dtype == YH_BF16 || dtype == YH_F16, "cache_read: dtype must be bf16 or f16");
  const int rc = check_cache("cache_read", keys, values, key_scales, value_scales, slots, N, blocks, G, D, block, bits);
  if (rc != YH_OK || N == 0) return rc;
  YH_CHECK_ARG(k && v, "cache_read: null pointer");
  YH_CHECK_ARG(tree::aligned16(k) && tree::aligned16(v), "cache_read: the rows must be 16-byte aligned");
  Args a = args_of(slots, keys, values, key_scales, value_scales, N, blocks, G, D, block);
  a.k_out = static_cast<uint16_t*>(k);
  a.v_out = static_cast<uint16_t*>(v);
  const dim3 grid(static_cast<unsigned>((N * a.pieces.d + 255) / 256));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (bits == 16) {
    hipLaunchKernelGGL((read_kernel<YH_BF16, k16>), grid, dim3(256), 0, st, a);   // 16 bits move as they are
  } else if (dtype == YH_BF16) {
    if (bits == 8) hipLaunchKernelGGL((read_kernel<YH_BF16, kFp8>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((read_kernel<YH_BF16, kFp4>), grid, dim3(256), 0, st, a);
  } else {
    if (bits == 8) hipLaunchKernelGGL((read_kernel<YH_F16, kFp8>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((read_kernel<YH_F16, kFp4>), grid, dim3(256), 0, st, a);
  }
  YH_CHECK_LAUNCH("cache_read");
  return YH_OK;
}
