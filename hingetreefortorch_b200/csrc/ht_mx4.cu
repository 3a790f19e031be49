// Weights into microscaled 4-bit numbers (ht_mx4.cuh) and back.
//
//     b = max(floor(log2 max|w|) - 2, -127) + 127 over a block (255 where it holds an infinity or no number)
//     code = w 2^(127 - b), to the nearest of the eight magnitudes, of two as near the one with the even code, 6 at the most
//
// Both are bound by memory: a thread takes 8 features, 4 threads a block.
#include "ht_mx4.cuh"

namespace ht {
namespace mx4 {
namespace {

using dense::after_previous_kernel;
using dense::load_plain;
using dense::to_float;

constexpr int kThreads = 256, kItems = 2048;  // of a CTA at a time, about

struct Shape {
  int64_t outputs, features, stride;
  int per_row;   // items of 8 features, four for each block
  int rows;      // of a CTA at a time
  bool whole;    // rows start on 16 bytes
};

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

template <typename T>
__global__ void __launch_bounds__(kThreads) pack_kernel(const Shape a, const T *w, uint32_t *codes, uint8_t *scales) {
  after_previous_kernel();
  constexpr int kPer = 16 / (int)sizeof(T);
  for (int64_t row0 = (int64_t)blockIdx.x * a.rows; row0 < a.outputs; row0 += (int64_t)gridDim.x * a.rows) {
    const uint32_t items = (uint32_t)min((int64_t)a.rows, a.outputs - row0) * (uint32_t)a.per_row;  // (a multiple of 4: the lanes of a block go together)
    for (uint32_t i = threadIdx.x; i < items; i += kThreads) {
      const uint32_t r = i / (uint32_t)a.per_row, q = i - r * (uint32_t)a.per_row;
      const int64_t row = row0 + r, k = (int64_t)q * 8;
      const T *from = w + row * a.stride + k;
      float v[8];
      if (a.whole && k + 8 <= a.features) {
#pragma unroll
        for (int j = 0; j < 8; j += kPer) {
          T t[kPer];
          *reinterpret_cast<uint4 *>(t) = load_plain(reinterpret_cast<const uint4 *>(from + j));
#pragma unroll
          for (int n = 0; n < kPer; ++n) v[j + n] = to_float(t[n]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = k + j < a.features ? to_float(from[j]) : 0.0f;
      }
      uint32_t top = 0;  // the largest magnitude's bits: no number is above infinity
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
      const uint32_t lanes = 0xfu << (threadIdx.x & 28u);
      top = max(top, __shfl_xor_sync(lanes, top, 1));
      top = max(top, __shfl_xor_sync(lanes, top, 2));
      const uint32_t field = top >> 23, b = field == 255u ? 255u : field > 2u ? field - 2u : 0u;
      const float factor = __uint_as_float((254u - b) << 23);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= factor;
      codes[row * a.per_row + q] = b == 255u ? 0u : codes_of(v);
      if ((q & 3u) == 0u) scales[row * (a.per_row / 4) + q / 4] = (uint8_t)b;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) unpack_kernel(const Shape a, const uint32_t *codes, const uint8_t *scales, T *w) {
  after_previous_kernel();
  constexpr int kPer = 16 / (int)sizeof(T);
  for (int64_t row0 = (int64_t)blockIdx.x * a.rows; row0 < a.outputs; row0 += (int64_t)gridDim.x * a.rows) {
    const uint32_t items = (uint32_t)min((int64_t)a.rows, a.outputs - row0) * (uint32_t)a.per_row;
    for (uint32_t i = threadIdx.x; i < items; i += kThreads) {
      const uint32_t r = i / (uint32_t)a.per_row, q = i - r * (uint32_t)a.per_row;
      const int64_t row = row0 + r, k = (int64_t)q * 8;
      if (k >= a.features) continue;
      const uint32_t c = load_plain(codes + row * a.per_row + q), b = load_plain(scales + row * (a.per_row / 4) + q / 4);
      const float scale = b == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(b == 0u ? 0x00400000u : b << 23);
      T t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t code = c >> (4 * j);
        const float number = __uint_as_float((code & 7u) << 22) * 0x1p126f * scale;
        t[j] = dense::from_float<T>(__uint_as_float(__float_as_uint(number) | (code & 8u) << 28));
      }
      T *to = w + row * a.stride + k;
      if (a.whole && k + 8 <= a.features) {
#pragma unroll
        for (int j = 0; j < 8; j += kPer) *reinterpret_cast<uint4 *>(to + j) = *reinterpret_cast<const uint4 *>(t + j);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (k + j < a.features) to[j] = t[j];
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
    return dense::launch_next<pack_kernel<T>>(dim3(dense::blocks_for(outputs, s.rows, 148 * 8)), kThreads, 0, 0, reinterpret_cast<cudaStream_t>(stream), 1, s,
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
    return dense::launch_next<unpack_kernel<T>>(dim3(dense::blocks_for(outputs, s.rows, 148 * 8)), kThreads, 0, 0, reinterpret_cast<cudaStream_t>(stream), 1,
                                                s, static_cast<const uint32_t *>(codes), static_cast<const uint8_t *>(scales), static_cast<T *>(w));
  });
}
