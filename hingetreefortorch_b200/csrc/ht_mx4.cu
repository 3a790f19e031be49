// Weights into microscaled 4-bit numbers (ht_mx4.cuh) and back.
//
//     b = max(floor(log2 max|w|) - 2, -127) + 127 over a block (255 where it holds an infinity or no number)
//     code = w 2^(127 - b), to the nearest of the eight magnitudes, of two as near the one with the even code, 6 at the most
//
// Both are bound by memory: a thread takes 8 features, 4 threads a block, and two of those at a time, so that their loads are under way together; a
// place's row comes by a multiplication (a division by the row's length took a third of the time).  Measured: 50000 x 1024 of fp32 packed in 35 us
// (6.6 TB/s), unpacked to bf16 in 26.5 (4.9; issue slots 80 % in use, the sign of zeros is 1.2 of them); 10007 x 771 of fp16, whose rows start on 2 bytes,
// 7.7 and 10.2 (value by value 24 and 30).
#include "ht_mx4.cuh"

namespace ht {
namespace mx4 {
namespace {

using dense::after_previous_kernel;
using dense::load_plain;
using dense::to_float;

constexpr int kThreads = 256, kItems = 1024;  // of a CTA at a time, about

struct Shape {
  int64_t outputs, features, stride;
  int per_row;   // items of 8 features, four for each block
  int rows;      // of a CTA at a time
  uint32_t magic;  // item i of a CTA is in its row i magic / 2^32
  bool whole;    // rows start on 16 bytes
};

// 8 values of a row from k on, zeros behind its end.  16-bit rows that start on 2 or 4 bytes are read by words, 5 of them on odd starts, as long as
// a value follows the last one (`followed`).
template <typename T>
__device__ __forceinline__ void load_values(const T *from, int64_t left, bool whole, bool followed, float (&v)[8]) {
  constexpr int kPer = 16 / (int)sizeof(T);
  if (whole && left >= 8) {
#pragma unroll
    for (int j = 0; j < 8; j += kPer) {
      T t[kPer];
      *reinterpret_cast<uint4 *>(t) = load_plain(reinterpret_cast<const uint4 *>(from + j));
#pragma unroll
      for (int n = 0; n < kPer; ++n) v[j + n] = to_float(t[n]);
    }
    return;
  }
  if constexpr (sizeof(T) == 2) {
    if (left > 8 || (left == 8 && followed)) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(from);
      const uint32_t *words = reinterpret_cast<const uint32_t *>(at & ~(uintptr_t)3);
      const bool odd = (at & 2u) != 0;
      uint32_t q[5];
#pragma unroll
      for (int j = 0; j < 5; ++j) q[j] = j < 4 || odd ? load_plain(words + j) : 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t pair = odd ? __funnelshift_r(q[j], q[j + 1], 16) : q[j];
        T t[2];
        *reinterpret_cast<uint32_t *>(t) = pair;
        v[2 * j] = to_float(t[0]), v[2 * j + 1] = to_float(t[1]);
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < left ? to_float(from[j]) : 0.0f;
}
template <typename T>
__device__ __forceinline__ void store_values(T *to, int64_t left, bool whole, const T (&t)[8]) {
  constexpr int kPer = 16 / (int)sizeof(T);
  if (whole && left >= 8) {
#pragma unroll
    for (int j = 0; j < 8; j += kPer) *reinterpret_cast<uint4 *>(to + j) = *reinterpret_cast<const uint4 *>(t + j);
    return;
  }
  if constexpr (sizeof(T) == 2) {
    if (left >= 8) {  // words from the first even address on
      const bool odd = (reinterpret_cast<uintptr_t>(to) & 2u) != 0;
      const uint32_t *pairs = reinterpret_cast<const uint32_t *>(t);
      if (!odd) {
#pragma unroll
        for (int j = 0; j < 4; ++j) reinterpret_cast<uint32_t *>(to)[j] = pairs[j];
      } else {
        to[0] = t[0];
#pragma unroll
        for (int j = 0; j < 3; ++j) reinterpret_cast<uint32_t *>(to + 1)[j] = __funnelshift_r(pairs[j], pairs[j + 1], 16);
        to[7] = t[7];
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) to[j] = t[j];
}

// Codes of 8 values, the first in the lowest bits.
__device__ __forceinline__ uint32_t codes_of(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Items of a CTA's rows, kAtOnce of them a thread at a time: their loads are under way together.
constexpr int kAtOnce = 2;
template <typename T>
__global__ void __launch_bounds__(kThreads) pack_kernel(const Shape a, const T *w, uint32_t *codes, uint8_t *scales) {
  after_previous_kernel();
  for (int64_t row0 = (int64_t)blockIdx.x * a.rows; row0 < a.outputs; row0 += (int64_t)gridDim.x * a.rows) {
    const uint32_t items = (uint32_t)min((int64_t)a.rows, a.outputs - row0) * (uint32_t)a.per_row;  // (a multiple of 4: the lanes of a block go together)
    for (uint32_t i0 = threadIdx.x; i0 < items; i0 += kAtOnce * kThreads) {
      float v[kAtOnce][8];
      uint32_t q[kAtOnce];
      int64_t row[kAtOnce];
#pragma unroll
      for (int n = 0; n < kAtOnce; ++n) {
        const uint32_t i = i0 + n * kThreads, r = __umulhi(i, a.magic);
        q[n] = i - r * (uint32_t)a.per_row;
        row[n] = row0 + r;
        const int64_t k = (int64_t)q[n] * 8, left = i < items ? a.features - k : 0;
        load_values(w + (left > 0 ? row[n] * a.stride + k : 0), left, a.whole, row[n] + 1 < a.outputs, v[n]);
      }
#pragma unroll
      for (int n = 0; n < kAtOnce; ++n) {
        if (i0 + n * kThreads >= items) break;
        float largest = fabsf(v[n][0]);
#pragma unroll
        for (int j = 1; j < 8; ++j) asm("max.NaN.f32 %0, %1, %2;" : "=f"(largest) : "f"(largest), "f"(fabsf(v[n][j])));
        uint32_t top = __float_as_uint(largest);  // bits: no number is above infinity
        const uint32_t lanes = 0xfu << (threadIdx.x & 28u);
        top = max(top, __shfl_xor_sync(lanes, top, 1));
        top = max(top, __shfl_xor_sync(lanes, top, 2));
        const uint32_t field = top >> 23, b = field == 255u ? 255u : field > 2u ? field - 2u : 0u;
        const float factor = __uint_as_float((254u - b) << 23);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[n][j] *= factor;
        codes[row[n] * a.per_row + q[n]] = b == 255u ? 0u : codes_of(v[n]);
        if ((q[n] & 3u) == 0u) scales[row[n] * (a.per_row / 4) + q[n] / 4] = (uint8_t)b;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) unpack_kernel(const Shape a, const uint32_t *codes, const uint8_t *scales, T *w) {
  after_previous_kernel();
  const uint32_t one = opaque_one();
  for (int64_t row0 = (int64_t)blockIdx.x * a.rows; row0 < a.outputs; row0 += (int64_t)gridDim.x * a.rows) {
    const uint32_t items = (uint32_t)min((int64_t)a.rows, a.outputs - row0) * (uint32_t)a.per_row;
    for (uint32_t i0 = threadIdx.x; i0 < items; i0 += kAtOnce * kThreads) {
      uint32_t c[kAtOnce], b[kAtOnce], q[kAtOnce];
      int64_t row[kAtOnce];
#pragma unroll
      for (int n = 0; n < kAtOnce; ++n) {
        const uint32_t i = i0 + n * kThreads, r = __umulhi(i, a.magic);
        q[n] = i - r * (uint32_t)a.per_row;
        row[n] = row0 + r;
        c[n] = i < items ? load_plain(codes + row[n] * a.per_row + q[n]) : 0u;
        b[n] = i < items ? load_plain(scales + row[n] * (a.per_row / 4) + q[n] / 4) : 0u;
      }
#pragma unroll
      for (int n = 0; n < kAtOnce; ++n) {
        const int64_t k = (int64_t)q[n] * 8;
        if (i0 + n * kThreads >= items || k >= a.features) continue;
        alignas(16) T t[8];
        if (b[n] < 250u) {  // 40 2^(b - 127) is a number of bf16
          const uint32_t s = b[n] == 0u ? 0x40u : b[n] << 7, offset = 0x8020u | (b[n] + 5u) << 7;
          uint32_t w4[4];
          weights_of(c[n], Scale{s | s << 16, offset | offset << 16}, one, w4);
#pragma unroll
          for (int j = 0; j < 4; ++j)  // (40 + v) s - 40 s is 0 for both zeros: the sign is the code's
            w4[j] |= __byte_perm(c[n] << 4, c[n], 0x4000u + 0x1010u * (uint32_t)j) & 0x80008000u;
          if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            *reinterpret_cast<uint4 *>(t) = make_uint4(w4[0], w4[1], w4[2], w4[3]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              t[2 * j] = dense::from_float<T>(__uint_as_float(w4[j] << 16));
              t[2 * j + 1] = dense::from_float<T>(__uint_as_float(w4[j] & 0xffff0000u));
            }
          }
          store_values(w + row[n] * a.stride + k, a.features - k, a.whole, t);
          continue;
        }
        const float scale = b[n] == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(b[n] << 23);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t code = c[n] >> (4 * j);
          const float number = __uint_as_float((code & 7u) << 22) * 0x1p126f * scale;
          t[j] = dense::from_float<T>(__uint_as_float(__float_as_uint(number) | (code & 8u) << 28));
        }
        store_values(w + row[n] * a.stride + k, a.features - k, a.whole, t);
      }
    }
  }
}

int shape_of(int dtype, int64_t outputs, int64_t features, int64_t stride, const void *w, Shape *s) {
  if (dtype != HT_DTYPE_F32 && dtype != HT_DTYPE_BF16 && dtype != HT_DTYPE_F16) return HT_ERR_INVALID_ARGUMENT;
  if (outputs < 0 || features < 1 || stride < features) return HT_ERR_INVALID_ARGUMENT;
  if (features > 0x3fffff00 || outputs > 0x3fffff00) return HT_ERR_UNSUPPORTED;
  const int64_t size = dtype == HT_DTYPE_F32 ? 4 : 2;
  s->outputs = outputs, s->features = features, s->stride = stride;
  s->per_row = (int)(4 * blocks_of(features));
  s->rows = std::max(kItems / s->per_row, 1);
  // (exact where both items and their number in a row are below 2^16; a row alone is row 0)
  s->magic = s->rows > 1 ? (uint32_t)((0x100000000ull + (uint64_t)s->per_row - 1) / (uint64_t)s->per_row) : 0u;
  s->whole = (reinterpret_cast<uintptr_t>(w) & 15u) == 0 && stride * size % 16 == 0;
  return HT_OK;
}

template <typename F>
int by_type(int dtype, F &&f) {
  return dtype == HT_DTYPE_F32 ? f(float()) : dtype == HT_DTYPE_BF16 ? f(__nv_bfloat16()) : f(__half());
}

}  // namespace
}  // namespace mx4
}  // namespace ht

using namespace ht;
using namespace ht::mx4;

extern "C" int ht_mx4_pack(int dtype, const void *w, int64_t w_stride, int64_t outputs, int64_t features, void *codes, void *scales, ht_stream_t stream) {
  Shape s = {};
  HT_TRY(shape_of(dtype, outputs, features, w_stride, w, &s));
  if (outputs == 0) return HT_OK;
  if (w == nullptr || codes == nullptr || scales == nullptr) return HT_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(codes) & 15u) != 0) return HT_ERR_UNSUPPORTED;
  return by_type(dtype, [&](auto zero) -> int {
    typedef decltype(zero) T;
    return dense::launch_next<pack_kernel<T>>(dim3(dense::blocks_for(outputs, s.rows, 148 * 64)), kThreads, 0, 0, reinterpret_cast<cudaStream_t>(stream), 1, s,
                                              static_cast<const T *>(w), static_cast<uint32_t *>(codes), static_cast<uint8_t *>(scales));
  });
}

extern "C" int ht_mx4_unpack(int dtype, const void *codes, const void *scales, int64_t outputs, int64_t features, void *w, int64_t w_stride,
                             ht_stream_t stream) {
  Shape s = {};
  HT_TRY(shape_of(dtype, outputs, features, w_stride, w, &s));
  if (outputs == 0) return HT_OK;
  if (w == nullptr || codes == nullptr || scales == nullptr) return HT_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(codes) & 15u) != 0) return HT_ERR_UNSUPPORTED;
  return by_type(dtype, [&](auto zero) -> int {
    typedef decltype(zero) T;
    return dense::launch_next<unpack_kernel<T>>(dim3(dense::blocks_for(outputs, s.rows, 148 * 64)), kThreads, 0, 0, reinterpret_cast<cudaStream_t>(stream), 1,
                                                s, static_cast<const uint32_t *>(codes), static_cast<const uint8_t *>(scales), static_cast<T *>(w));
  });
}
