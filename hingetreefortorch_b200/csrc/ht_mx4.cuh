// Weights held as microscaled 4-bit numbers (ht_mx4.cu, ht_linear_mx4.cu): MXFP4 of the Open Compute Project's Microscaling Formats
// specification v1.0.  32 neighbouring features share a power of two, byte b for 2^(b - 127), 255 for no number; each of them is one of
// 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (2 bits of exponent, 1 of mantissa), two to a byte, the first in the low half.
//   codes  [outputs, 16 blocks]   scales [outputs, blocks]   blocks = features / 32, rounded up; codes behind the last feature are 0
#pragma once

#include "ht_dense.cuh"

namespace ht {
namespace mx4 {

constexpr int kBlock = 32;
__host__ __device__ inline int64_t blocks_of(int64_t features) { return (features + kBlock - 1) / kBlock; }

// 8 codes of a word as bf16: word i of the four has codes i and i + 4.  The 3 bits of a magnitude in the lowest bits of the exponent and the
// highest of the mantissa are the number times 2^-126, subnormal ones too, so one multiplication gives number and scale.  Operands are held as
// 2^-4 of their values: from 2^-132, a subnormal number of bf16, up to 6 2^123 all are exact, where 6 2^127 is beyond it; what they are summed to is
// multiplied by kHeld.
//   first: 2^126 2^(b - 127) / kHeld, for b up to 132;  more: what is missing beyond (1 otherwise)
constexpr float kHeld = 16.0f;
struct Scale {
  uint32_t first, more;  // twice the same bf16
  bool beyond;
};
__device__ __forceinline__ Scale scale_of(uint32_t b) {
  Scale s;
  const uint32_t f = b == 255u ? 0x7fc0u : min(b + 122u, 254u) << 7, m = b > 132u && b != 255u ? (b - 5u) << 7 : 0x3f80u;
  s.first = f | f << 16;
  s.more = m | m << 16;
  s.beyond = b > 132u;
  return s;
}
__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ void numbers_of(uint32_t w, uint32_t (&v)[4]) {
  constexpr uint32_t kMagnitude = 0x01c001c0u, kSign = 0x80008000u;
  v[0] = ((w << 6) & kMagnitude) | ((w << 12) & kSign);
  v[1] = ((w << 2) & kMagnitude) | ((w << 8) & kSign);
  v[2] = ((w >> 2) & kMagnitude) | ((w << 4) & kSign);
  v[3] = ((w >> 6) & kMagnitude) | (w & kSign);
}

}  // namespace mx4
}  // namespace ht
