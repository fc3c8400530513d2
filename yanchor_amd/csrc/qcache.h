// Quantised block caches: runs of 32 values of a row share a power of two
// 2^(s - 127), s a byte; the values are e4m3 codes (8 bits) or e2m1 codes (4 bits,
// two a byte, the even dim in the low half).
//   codes  [blocks, G, block, D] or [blocks, G, block, D / 2] bytes
//   scales [blocks, G, D / 32, block] bytes
// A row's scales lie a run apart, so that the rows of one run, which an attention
// reads together, are neighbouring bytes.
#pragma once
#include "common.h"

namespace yh {
namespace qcache {

constexpr int kRun = 32;        // values that share a scale
// The least scale, 2^-111: the smallest code of either type is then no
// subnormal of float32 or bf16, wherever it is multiplied.
constexpr int kLeast = 16;
constexpr int kNotANumber = 255;   // the scale of a run that holds a NaN or an infinity

enum Format { k16 = 0, kFp8 = 1, kFp4 = 2 };

// The scale byte of a run whose largest magnitude is `top`: the smallest at which
// top is no larger than the largest code, 448 = 1.75 x 2^8 or 6 = 1.5 x 2^2.
// Adding the rest of the mantissa's range carries into the exponent exactly where
// top's mantissa is past 1.75 (1.5).
template <int FMT>
__device__ __forceinline__ int scale_of(float top) {
  const uint32_t bits = __float_as_uint(top);
  if (bits >= 0x7f800000u) return kNotANumber;
  const int s = FMT == kFp8 ? static_cast<int>((bits + 0x1fffffu) >> 23) - 8
                            : static_cast<int>((bits + 0x3fffffu) >> 23) - 2;
  return s < kLeast ? kLeast : s;
}
// 2^(s - 127), a NaN for 255; of 0, which the write does not make, the subnormal 2^-127.
__device__ __forceinline__ float scale_value(int s) {
  return s == kNotANumber ? __uint_as_float(0x7fc00000u) : __uint_as_float(s == 0 ? 1u << 22 : static_cast<uint32_t>(s) << 23);
}
// 2^(127 - s) for s in [kLeast, 253], the inverse of a finite run's scale (up to 247 in 8 bits, 253 in 4); of 255, NaN.
__device__ __forceinline__ float scale_inverse(int s) {
  return s == kNotANumber ? __uint_as_float(0x7fc00000u) : __uint_as_float(static_cast<uint32_t>(254 - s) << 23);
}

}  // namespace qcache
}  // namespace yh
