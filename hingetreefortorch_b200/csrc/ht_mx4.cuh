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

// Codes as bf16 numbers.  A byte permutation whose selectors are the codes looks up 4 of them at a time: its fourth selector bit, the sign, turns
// a byte whose highest bit is 0 into 0, so one look-up gives the positive numbers, another, with the signs inverted, the negative ones, and
// their sum is 32 + 4 v.  Behind 0x42 that is the bf16 number 40 + v, and (40 + v) s - 40 s is v s without rounding.  s = 2^(b - 127) / kHeld: from
// 2^-133, the smallest subnormal number of bf16, up to 40 2^122 all of it is in bf16's range, where 6 2^127 is not; what operands
// are summed to is multiplied by kHeld.
// Permutations, shifts and logic run at half the rate of the rest: 11 of them for 8 codes, where moving sign and magnitude to their places
// by shifts took 19 (8192 x 1024 to 50000 of bf16 846 us instead of 885, with all else as it was then).
constexpr float kHeld = 32.0f;
struct Scale {
  uint32_t s, offset;  // twice the same bf16: s and -40 s
};
__device__ __forceinline__ Scale scale_of(uint32_t b) {
  uint32_t s = b < 6u ? 2u << b : (b - 5u) << 7, offset = b == 0u ? 0x8050u : 0x8020u | b << 7;
  if (b == 255u) s = 0x7fc0u;
  return {s | s << 16, offset | offset << 16};
}
__device__ __forceinline__ uint32_t permute(uint32_t a, uint32_t b, uint32_t selectors) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(selectors));
  return r;
}
// 8 codes of a word as 4 words of two neighbours.  `one` is 1 in a register: a sum by multiplication, which runs at the full rate.
__device__ __forceinline__ void weights_of(uint32_t w, const Scale &scale, uint32_t one, uint32_t *out) {
  const uint32_t n = w ^ 0x88888888u;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t positive = permute(0x26242220u, 0x38302c28u, h == 0 ? w : w >> 16), negative = permute(0x1a1c1e20u, 0x08101418u, h == 0 ? n : n >> 16);
    uint32_t bytes;
    asm("mad.lo.u32 %0, %1, %2, %3;" : "=r"(bytes) : "r"(positive), "r"(one), "r"(negative));
#pragma unroll
    for (int i = 0; i < 2; ++i)
      asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(out[2 * h + i]) : "r"(__byte_perm(bytes, 0x42424242u, i == 0 ? 0x4140u : 0x4342u)), "r"(scale.s), "r"(scale.offset));
  }
}
// 1 where the compiler does not know it.
__device__ __forceinline__ uint32_t opaque_one() {
  uint32_t one;
  asm volatile("mov.u32 %0, 1;" : "=r"(one));
  return one;
}

}  // namespace mx4
}  // namespace ht
