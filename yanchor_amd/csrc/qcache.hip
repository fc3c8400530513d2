// Rows into a quantised block cache, and rows of a cache back (qcache.h).
//
// Write: s = the smallest byte with max |x| <= M 2^(s - 127) over a run of 32
// values, M the largest code; code = round_to_nearest_even(x 2^(127 - s)).  No
// value saturates, and since scales are powers of two both the product and what
// is read back are exact but for that one rounding (half a step: 2^-4 of an e4m3
// value, 1/4 of the code's power of two of an e2m1 value).
// Read: value = code 2^(s - 127), rounded to the output's type.
//
// Bound by HBM and, where slots are scattered, by its granules: 65521 tokens of 8
// heads of 128 into scattered rows of 4 bits 92 us for 340 MB, of which the scale
// bytes, each in a granule of its own, take 23 and the 64-byte rows 14 (the input is
// 43 at a copy's rate); back 79; 154000 tokens in order of 8 bits back 177 us, 5.4
// TB/s.  Rows in and out pass the caches (101 and 91 us through them); codes of 4 bits
// do not, as two rows share a granule (79 us for 91).
#include "qcache.h"
#include "tree.h"

namespace yh {
namespace {

using namespace qcache;
using tree::Div;
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));

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
  Div block, per, row;     // per: a token's pieces of eight values, kThreads at most; row: a head's
  uint32_t pieces;         // all of a token's
  uint32_t tokens;         // that a workgroup takes at a time
  int G;
};

constexpr int kThreads = 256;
// Tokens that a thread takes where there are many (U = 1 for few), so that what lies where in a row is found once.
// (us of the prefixes in order back: one 187, two 184, four 177, eight 174, but eight write in 100 for 92.)
constexpr int kMany = 4;

// Piece p of a token's row: its bytes from the block's begin on, of FMT, and its scale's.
template <int FMT>
struct Piece {
  uint32_t code, scale, row;   // row: bytes of a head's row
  __device__ __forceinline__ Piece(const Args& a, uint32_t p) {
    const uint32_t g = a.row.quot(p), dim = (p - g * a.row.d) * 8;
    row = FMT == k16 ? a.row.d * 16 : FMT == kFp8 ? a.row.d * 8 : a.row.d * 4;
    code = g * a.block.d * row + (FMT == k16 ? dim * 2 : FMT == kFp8 ? dim : dim / 2);
    scale = (g * (a.row.d / 4) + dim / kRun) * a.block.d;
  }
};
// Where the row of slot s begins, or that it is none.
struct Slot {
  int64_t block;
  uint32_t row;
  bool in;
};
__device__ __forceinline__ Slot slot_of(const Args& a, int64_t t) {
  const int64_t s = t < a.N ? a.slots[t] : -1;
  const bool in = s >= 0 && s < a.n_slots;
  const int64_t x = in ? s : 0;
  const int64_t b = x < (1ll << 31) ? a.block.quot(static_cast<uint32_t>(x)) : x / a.block.d;
  return {b, static_cast<uint32_t>(x - b * a.block.d), in};
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
__device__ __forceinline__ void put8(uint4 x, bool in, bool first, char* codes, uint8_t* scale) {
  float y[8];
  widen8<DT>(x, y);
  uint32_t top = 0;      // of the magnitudes, as bits: a NaN's are the largest
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(y[i]) & 0x7fffffffu);
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1, kWave)));
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 2, kWave)));
  const int s = scale_of<FMT>(__uint_as_float(top));
  const float inv = scale_inverse(s);
  // a run that is not finite reads back as NaN by its scale
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = s == kNotANumber ? 0.f : y[i] * inv;
  if (!in) return;
  if constexpr (FMT == kFp8) {
    u2 c;
    c[0] = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    c[0] = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c[0], true);
    c[1] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
    c[1] = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], c[1], true);
    *reinterpret_cast<u2*>(codes) = c;
  } else {
    uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[0], y[1], 1.f, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[2], y[3], 1.f, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[4], y[5], 1.f, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, y[6], y[7], 1.f, 3);
    *reinterpret_cast<uint32_t*>(codes) = c;
  }
  if (first) *scale = static_cast<uint8_t>(s);
}

__device__ __forceinline__ uint4 stream_load(const void* p) {
  const u4 x = __builtin_nontemporal_load(static_cast<const u4*>(p));
  return make_uint4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void stream_store(void* p, uint4 x) {
  __builtin_nontemporal_store(u4{x.x, x.y, x.z, x.w}, static_cast<u4*>(p));
}

// Both kernels: thread (token of the workgroup's, piece), U tokens a thread, and more pieces where a row has more than
// the workgroup has threads.
template <int DT, int FMT, int U>
__global__ void __launch_bounds__(kThreads) write_kernel(Args a) {
  const uint32_t sub = a.per.quot(threadIdx.x), p0 = threadIdx.x - sub * a.per.d;
  if (sub >= a.tokens) return;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * (U * a.tokens) + sub;
  const int64_t block_codes = static_cast<int64_t>(a.G) * a.block.d * (a.row.d * (FMT == kFp8 ? 8 : 4));
  const int64_t block_scales = static_cast<int64_t>(a.G) * a.block.d * (a.row.d / 4);
  Slot slot[U];
#pragma unroll
  for (int u = 0; u < U; ++u) slot[u] = slot_of(a, t0 + u * a.tokens);
  for (uint32_t p = p0; p < a.pieces; p += kThreads) {
    const Piece<FMT> at(a, p);
    uint4 x[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[u] = y[u] = make_uint4(0, 0, 0, 0);
      if (slot[u].in) {
        x[u] = stream_load(a.k + (t0 + u * a.tokens) * a.ks + p * 8);
        y[u] = stream_load(a.v + (t0 + u * a.tokens) * a.vs + p * 8);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t code = slot[u].block * block_codes + at.code + static_cast<uint64_t>(slot[u].row) * at.row;
      const int64_t scale = slot[u].block * block_scales + at.scale + slot[u].row;
      put8<DT, FMT>(x[u], slot[u].in, p % 4 == 0, a.keys + code, a.key_scales + scale);
      put8<DT, FMT>(y[u], slot[u].in, p % 4 == 0, a.values + code, a.value_scales + scale);
    }
  }
}

// Eight values as they are stored, and their scale.
struct Raw {
  uint4 codes;
  uint32_t scale;
};
template <int FMT>
__device__ __forceinline__ Raw fetch8(bool in, const char* codes, const uint8_t* scale) {
  Raw r{};
  if (!in) return r;
  if constexpr (FMT == k16) {
    r.codes = stream_load(codes);
  } else {
    r.scale = *scale;
    if constexpr (FMT == kFp8) {
      const u2 c = __builtin_nontemporal_load(reinterpret_cast<const u2*>(codes));
      r.codes.x = c[0];
      r.codes.y = c[1];
    } else {
      r.codes.x = *reinterpret_cast<const uint32_t*>(codes);
    }
  }
  return r;
}
template <int DT, int FMT>
__device__ __forceinline__ uint4 decode8(Raw r) {
  if constexpr (FMT == k16) {
    return r.codes;
  } else {
    const float s = scale_value(r.scale);
    float y[8];
    if constexpr (FMT == kFp8) {
      const auto p0 = __builtin_amdgcn_cvt_pk_f32_fp8(r.codes.x, false), p1 = __builtin_amdgcn_cvt_pk_f32_fp8(r.codes.x, true);
      const auto p2 = __builtin_amdgcn_cvt_pk_f32_fp8(r.codes.y, false), p3 = __builtin_amdgcn_cvt_pk_f32_fp8(r.codes.y, true);
      y[0] = p0[0]; y[1] = p0[1]; y[2] = p1[0]; y[3] = p1[1];
      y[4] = p2[0]; y[5] = p2[1]; y[6] = p3[0]; y[7] = p3[1];
    } else {
      const auto p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r.codes.x, 1.f, 0);
      const auto p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r.codes.x, 1.f, 1);
      const auto p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r.codes.x, 1.f, 2);
      const auto p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r.codes.x, 1.f, 3);
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

template <int DT, int FMT, int U>
__global__ void __launch_bounds__(kThreads) read_kernel(Args a) {
  const uint32_t sub = a.per.quot(threadIdx.x), p0 = threadIdx.x - sub * a.per.d;
  if (sub >= a.tokens) return;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * (U * a.tokens) + sub;
  const int64_t block_codes = static_cast<int64_t>(a.G) * a.block.d * (a.row.d * (FMT == k16 ? 16 : FMT == kFp8 ? 8 : 4));
  const int64_t block_scales = static_cast<int64_t>(a.G) * a.block.d * (a.row.d / 4);
  Slot slot[U];
#pragma unroll
  for (int u = 0; u < U; ++u) slot[u] = slot_of(a, t0 + u * a.tokens);
  for (uint32_t p = p0; p < a.pieces; p += kThreads) {
    const Piece<FMT> at(a, p);
    Raw x[U], y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t code = slot[u].block * block_codes + at.code + static_cast<uint64_t>(slot[u].row) * at.row;
      const int64_t scale = slot[u].block * block_scales + at.scale + slot[u].row;
      x[u] = fetch8<FMT>(slot[u].in, a.keys + code, a.key_scales + scale);
      y[u] = fetch8<FMT>(slot[u].in, a.values + code, a.value_scales + scale);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = t0 + u * a.tokens;
      if (t >= a.N) break;
      stream_store(a.k_out + (t * a.pieces + p) * 8, decode8<DT, FMT>(x[u]));
      stream_store(a.v_out + (t * a.pieces + p) * 8, decode8<DT, FMT>(y[u]));
    }
  }
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
  YH_CHECK_ARG(G * D * block * 2 < (1ll << 32) && N * (G * D / 8) < (1ll << 32), "%s: sizes too large", what);
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
  a.pieces = static_cast<uint32_t>(G * D / 8);
  a.per = tree::make_div(a.pieces < kThreads ? a.pieces : kThreads);
  a.tokens = kThreads / a.per.d;
  a.row = tree::make_div(static_cast<uint32_t>(D / 8));
  a.G = static_cast<int>(G);
  return a;
}

// Whether each thread takes several tokens: where that still leaves four workgroups a CU.
bool many(const Args& a) { return a.N >= static_cast<int64_t>(1024) * kMany * a.tokens; }
unsigned grid_of(const Args& a) {
  const int64_t each = (many(a) ? kMany : 1) * static_cast<int64_t>(a.tokens);
  return static_cast<unsigned>((a.N + each - 1) / each);
}
template <int DT, int FMT>
void launch_write(const Args& a, hipStream_t st) {
  if (many(a)) hipLaunchKernelGGL((write_kernel<DT, FMT, kMany>), dim3(grid_of(a)), dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((write_kernel<DT, FMT, 1>), dim3(grid_of(a)), dim3(kThreads), 0, st, a);
}
template <int DT, int FMT>
void launch_read(const Args& a, hipStream_t st) {
  if (many(a)) hipLaunchKernelGGL((read_kernel<DT, FMT, kMany>), dim3(grid_of(a)), dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((read_kernel<DT, FMT, 1>), dim3(grid_of(a)), dim3(kThreads), 0, st, a);
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
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == YH_BF16) {
    if (bits == 8) launch_write<YH_BF16, kFp8>(a, st);
    else launch_write<YH_BF16, kFp4>(a, st);
  } else {
    if (bits == 8) launch_write<YH_F16, kFp8>(a, st);
    else launch_write<YH_F16, kFp4>(a, st);
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
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (bits == 16) {
    launch_read<YH_BF16, k16>(a, st);   // 16 bits move as they are
  } else if (dtype == YH_BF16) {
    if (bits == 8) launch_read<YH_BF16, kFp8>(a, st);
    else launch_read<YH_BF16, kFp4>(a, st);
  } else {
    if (bits == 8) launch_read<YH_F16, kFp8>(a, st);
    else launch_read<YH_F16, kFp4>(a, st);
  }
  YH_CHECK_LAUNCH("cache_read");
  return YH_OK;
}
