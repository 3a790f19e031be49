// What the dense layers around a forest share (ht_gated_linear.cu, ht_class_loss.cu): element types, the layout of operands for the tile
// product, stores of a thread's 32 columns, column sums, the kernel for few rows, and the two products of a backward pass.
#pragma once

#include "ht_dense_tile.cuh"

namespace ht {
namespace dense {

// Element types of a call: fp32 is held as three bf16 planes for the tensor cores.
template <typename T>
struct Kind;
template <>
struct Kind<float> {
  static constexpr int kPlanes = 3;
  typedef __nv_bfloat16 Operand;
};
template <>
struct Kind<__nv_bfloat16> {
  static constexpr int kPlanes = 1;
  typedef __nv_bfloat16 Operand;
};
template <>
struct Kind<__half> {
  static constexpr int kPlanes = 1;
  typedef __half Operand;
};

// What gradients of scores or projections are held as, and the other operand of the products that they enter.  fp16 has neither the range nor,
// by one scale for all, room for rows of different sizes (u act'(a) beyond 65504, one row a million times the next): two bf16
// numbers, 2^-17 of a value of any size, with x and the weights, 11 bits each, exact in two as well.  Three products for one: 8192 x 784 to
// 12700 takes 2.3 ms a training step where bf16 takes 1.3.
template <typename T>
struct GradKind : Kind<T> {};
template <>
struct GradKind<__half> {
  static constexpr int kPlanes = 2;
  typedef __nv_bfloat16 Operand;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ uint32_t pack_pair(float a, float b, const __nv_bfloat16 *) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t pack_pair(float a, float b, const __half *) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// v = p0 + p1 + p2, each the rounding to bf16 of what the ones before leave: 24 bits; two values at a time, to a word each.  The first rounding
// does not leave the finite numbers; of an infinity the rest is one as well, and the third number none.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t &p0, uint32_t &p1, uint32_t &p2) {
  asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(p0) : "f"(b), "f"(a));
  const float rest_a = a - __uint_as_float(p0 << 16), rest_b = b - __uint_as_float(p0 & 0xffff0000u);
  p1 = pack_pair(rest_a, rest_b, static_cast<const __nv_bfloat16 *>(nullptr));
  p2 = pack_pair(rest_a - __uint_as_float(p1 << 16), rest_b - __uint_as_float(p1 & 0xffff0000u), static_cast<const __nv_bfloat16 *>(nullptr));
}

// n numbers of one row, contiguous; all lanes read the same ones.
template <typename T>
__device__ __forceinline__ void load_columns(const T *in, float (&v)[32], int n) {
  if (n >= 32) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 32; i += kPer) {
      T t[kPer];
      *reinterpret_cast<uint4 *>(t) = load_plain(reinterpret_cast<const uint4 *>(in + i));
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[i + j] = to_float(t[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = i < n ? to_float(in[i]) : 0.0f;
  }
}

__device__ __forceinline__ void store_32_bytes(void *to, const uint32_t (&q)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3]), "r"(q[4]),
               "r"(q[5]), "r"(q[6]), "r"(q[7])
               : "memory");
}
__device__ __forceinline__ void load_32_bytes(const void *from, uint32_t (&q)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7])
               : "l"(from)
               : "memory");
}

// A warp's 32 rows of 32 columns between registers (a lane has a row) and a matrix: `first` points at the first row's first column of
// the box, `rows` and `cols` of the box are inside the matrix (32 or fewer), `align` is the power of two of bytes that every row starts on
// (32 at the most).  Rows on 32 bytes go lane by lane in whole sectors; others through the warp's shared memory, so that neighbouring lanes
// read or write neighbouring addresses, `align` bytes each (rows of 12700 bf16, written two bytes a lane and row, took 5 times the
// product's time).
template <int BYTES>
struct Word;
template <>
struct Word<2> {
  typedef uint16_t type;
};
template <>
struct Word<4> {
  typedef uint32_t type;
};
template <>
struct Word<8> {
  typedef uint2 type;
};
template <>
struct Word<16> {
  typedef uint4 type;
};
// 16-byte piece q of row r of the box
template <typename T>
__device__ __forceinline__ uint32_t box_offset(uint32_t r, uint32_t q) {
  return sizeof(T) == 4 ? 128u * r + 16u * (q ^ (r & 7u)) : 64u * r + 16u * (q ^ ((r >> 1) & 3u));
}
template <typename T, int BYTES, bool STORE>
__device__ __forceinline__ void move_box(uint32_t box, T *first, size_t pitch, int rows, int cols, int lane) {
  typedef typename Word<BYTES>::type W;
  constexpr int kPerRow = 32 * (int)sizeof(T) / BYTES, kRows = 32 / kPerRow, kValues = BYTES / (int)sizeof(T);
  const int piece = lane % kPerRow, c = piece * kValues;
#pragma unroll 4
  for (int r = lane / kPerRow; r < 32; r += kRows) {
    if (r >= rows || c >= cols) continue;
    const uint32_t at = box + box_offset<T>((uint32_t)r, (uint32_t)(piece * BYTES / 16)) + (uint32_t)(piece * BYTES % 16);
    W *const shared = reinterpret_cast<W *>(__cvta_shared_to_generic(at));
    T *const global = first + (size_t)r * pitch + c;
    if (c + kValues <= cols) {
      if (STORE)
        *reinterpret_cast<W *>(global) = *shared;
      else
        *shared = load_plain(reinterpret_cast<const W *>(global));
    } else {
      T *const each = reinterpret_cast<T *>(shared);
      for (int j = 0; j < cols - c; ++j) {
        if (STORE)
          global[j] = each[j];
        else
          each[j] = global[j];
      }
    }
  }
}
// Whole boxes of 16-bit rows that start on 2 bytes, to memory: two values at a time from the first even address on, out of two words of the
// box where the row starts on an odd one, whose first and last value go alone.
template <typename T>
__device__ __forceinline__ void store_odd_box(uint32_t box, T *first, size_t pitch, int rows, int lane) {
  auto word = [&](uint32_t r, uint32_t i) { return lds_b32(box + box_offset<T>(r, i >> 2) + (i & 3u) * 4u); };
  const uint32_t i = (uint32_t)lane & 15u;
#pragma unroll 4
  for (uint32_t r = (uint32_t)lane >> 4; r < 32u; r += 2u) {
    T *const row = first + (size_t)r * pitch;
    const bool odd = (reinterpret_cast<uintptr_t>(row) & 2u) != 0;
    const uint32_t low = word(r, i), high = word(r, min(i + 1u, 15u));
    if ((int)r < rows && !(odd && i == 15u)) *reinterpret_cast<uint32_t *>(row + 2 * i + (odd ? 1 : 0)) = odd ? __funnelshift_r(low, high, 16) : low;
  }
  T *const own = first + (size_t)lane * pitch;
  if (lane < rows && (reinterpret_cast<uintptr_t>(own) & 2u) != 0) {
    *reinterpret_cast<uint16_t *>(own) = (uint16_t)word((uint32_t)lane, 0u);
    *reinterpret_cast<uint16_t *>(own + 31) = (uint16_t)(word((uint32_t)lane, 15u) >> 16);
  }
}
template <typename T, bool STORE>
__device__ __forceinline__ void move_box_by(uint32_t box, T *first, size_t pitch, int rows, int cols, int align, int lane) {
  if (align >= 16)
    move_box<T, 16, STORE>(box, first, pitch, rows, cols, lane);
  else if (align == 8)
    move_box<T, 8, STORE>(box, first, pitch, rows, cols, lane);
  else if (align == 4 || sizeof(T) == 4)
    move_box<T, 4, STORE>(box, first, pitch, rows, cols, lane);
  else if constexpr (sizeof(T) == 2) {
    if (STORE && cols >= 32)
      store_odd_box<T>(box, first, pitch, rows, lane);
    else
      move_box<T, 2, STORE>(box, first, pitch, rows, cols, lane);
  }
}

template <typename T>
__device__ __forceinline__ void to_words(const float (&v)[32], int from, uint32_t (&q)[8]) {  // 32 bytes
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(T) == 4)
      q[i] = __float_as_uint(v[from + i]);
    else
      q[i] = pack_pair(v[from + 2 * i], v[from + 2 * i + 1], static_cast<const T *>(nullptr));
  }
}
template <typename T>
__device__ __forceinline__ void from_words(const uint32_t (&q)[8], int from, float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[from + i] = __uint_as_float(q[i]);
    } else {
      T pair[2];
      *reinterpret_cast<uint32_t *>(pair) = q[i];
      v[from + 2 * i] = to_float(pair[0]);
      v[from + 2 * i + 1] = to_float(pair[1]);
    }
  }
}

template <typename T>
__device__ __forceinline__ void store_box(const Where &w, T *first, size_t pitch, int rows, int cols, int align, const float (&v)[32]) {
  constexpr int kStep = 32 / (int)sizeof(T);
  if (align >= 32 && cols >= 32) {
    if (w.lane < rows) {
      T *to = first + (size_t)w.lane * pitch;
#pragma unroll
      for (int i = 0; i < 32; i += kStep) {
        uint32_t q[8];
        to_words<T>(v, i, q);
        store_32_bytes(to + i, q);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 32; i += kStep) {
    uint32_t q[8];
    to_words<T>(v, i, q);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(w.box + box_offset<T>((uint32_t)w.lane, (uint32_t)(i / kStep * 2 + h))),
                   "r"(q[4 * h]), "r"(q[4 * h + 1]), "r"(q[4 * h + 2]), "r"(q[4 * h + 3])
                   : "memory");
  }
  __syncwarp();
  move_box_by<T, true>(w.box, first, pitch, rows, cols, align, w.lane);
  __syncwarp();
}
// (columns and rows outside the matrix come as what the box held before)
template <typename T>
__device__ __forceinline__ void load_box(const Where &w, const T *first, size_t pitch, int rows, int cols, int align, float (&v)[32]) {
  constexpr int kStep = 32 / (int)sizeof(T);
  if (align >= 32 && cols >= 32) {
    const T *from = first + (size_t)min(w.lane, rows - 1) * pitch;
#pragma unroll
    for (int i = 0; i < 32; i += kStep) {
      uint32_t q[8];
      load_32_bytes(from + i, q);
      from_words<T>(q, i, v);
    }
    return;
  }
  move_box_by<T, false>(w.box, const_cast<T *>(first), pitch, rows, cols, align, w.lane);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 32; i += kStep) {
    uint32_t q[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 t = lds_b128(w.box + box_offset<T>((uint32_t)w.lane, (uint32_t)(i / kStep * 2 + h)));
      q[4 * h] = t.x, q[4 * h + 1] = t.y, q[4 * h + 2] = t.z, q[4 * h + 3] = t.w;
    }
    from_words<T>(q, i, v);
  }
  __syncwarp();
}
// load_box in two halves: begun early (cp.async, for rows on 4 bytes at least; others wait for the second half), and finished into
// registers: `last`, or another box has been begun since.  A box takes 1024 sizeof(T) bytes at `at`.
template <typename T, int BYTES>
__device__ __forceinline__ void fetch_box(uint32_t at, const T *first, size_t pitch, int rows, int cols, int lane) {
  constexpr int kPerRow = 32 * (int)sizeof(T) / BYTES, kRows = 32 / kPerRow, kValues = BYTES / (int)sizeof(T);
  const int piece = lane % kPerRow, c = piece * kValues;
  if (c >= cols) return;
  const int bytes = min(BYTES, (cols - c) * (int)sizeof(T));
#pragma unroll 4
  for (int r = lane / kPerRow; r < rows; r += kRows) {
    const uint32_t to = at + box_offset<T>((uint32_t)r, (uint32_t)(piece * BYTES / 16)) + (uint32_t)(piece * BYTES % 16);
    const T *from = first + (size_t)r * pitch + c;
    if constexpr (BYTES == 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
    else
      asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(to), "l"(from), "r"(bytes), "n"(BYTES) : "memory");
  }
}
template <typename T>
__device__ __forceinline__ void begin_box(uint32_t at, const T *first, size_t pitch, int rows, int cols, int align, int lane) {
  if (align >= 16)
    fetch_box<T, 16>(at, first, pitch, rows, cols, lane);
  else if (align == 8)
    fetch_box<T, 8>(at, first, pitch, rows, cols, lane);
  else if (align == 4)
    fetch_box<T, 4>(at, first, pitch, rows, cols, lane);
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <typename T>
__device__ __forceinline__ void finish_box(uint32_t at, const T *first, size_t pitch, int rows, int cols, int align, int lane, bool last, float (&v)[32]) {
  constexpr int kStep = 32 / (int)sizeof(T);
  if (align >= 4) {
    if (last)
      asm volatile("cp.async.wait_all;" ::: "memory");
    else
      asm volatile("cp.async.wait_group 1;" ::: "memory");
  } else
  
    move_box_by<T, false>(at, const_cast<T *>(first), pitch, rows, cols, align, lane);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 32; i += kStep) {
    uint32_t q[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 t = lds_b128(at + box_offset<T>((uint32_t)lane, (uint32_t)(i / kStep * 2 + h)));
      q[4 * h] = t.x, q[4 * h + 1] = t.y, q[4 * h + 2] = t.z, q[4 * h + 3] = t.w;
    }
    from_words<T>(q, i, v);
  }
  __syncwarp();
}

// The alignment of a matrix's rows for the functions above.
inline int row_alignment(const void *data, int64_t row_bytes) {
  const uint64_t bits = (uint64_t)reinterpret_cast<uintptr_t>(data) | (uint64_t)row_bytes | 32u;
  return (int)(bits & (~bits + 1));
}

// The same as operands of a later product: [planes][rows][pitch], rows of a multiple of 64 elements; a lane's row.
template <typename T>
__device__ __forceinline__ void store_operand(typename GradKind<T>::Operand *out, size_t plane, const float (&v)[32]) {
  typedef typename GradKind<T>::Operand O;
#pragma unroll
  for (int i = 0; i < 32; i += 16) {
    uint32_t q[8];
    if constexpr (GradKind<T>::kPlanes == 1) {
      to_words<O>(v, i, q);
      store_32_bytes(out + i, q);
    } else {
      uint32_t q1[8], q2[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) split_pair(v[i + 2 * j], v[i + 2 * j + 1], q[j], q1[j], q2[j]);
      store_32_bytes(out + i, q);
      store_32_bytes(out + plane + i, q1);
      if constexpr (GradKind<T>::kPlanes == 3) store_32_bytes(out + 2 * plane + i, q2);
    }
  }
}

// The sum over the warp's 32 rows of column `lane`: every step halves the columns that a lane holds.
__device__ __forceinline__ float sum_rows(const float (&v)[32], int lane) {
  float h[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const bool up = (lane & 16) != 0;
    h[i] = (up ? v[i + 16] : v[i]) + __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + 16], 16);
  }
#pragma unroll
  for (int s = 8; s >= 1; s >>= 1) {
    const bool up = (lane & s) != 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < s) h[i] = (up ? h[i + s] : h[i]) + __shfl_xor_sync(0xffffffffu, up ? h[i] : h[i + s], s);
  }
  return h[0];
}

// What gradients are multiplied by when they leave: a number on the device (over a count that is there as well, 0 for none), or 1.
struct Scale {
  const float *number = nullptr, *count = nullptr;
  __device__ __forceinline__ float value() const {
    if (number == nullptr) return 1.0f;
    const float n = load_plain(number), c = count != nullptr ? load_plain(count) : 1.0f;
    return c > 0.0f ? n / c : 0.0f;
  }
};

// ---- epilogue: the products themselves, scaled -----------------------------------------------------------------------
// out = alpha (acc + products): `sum` holds what earlier pieces of k have given, in fp32; `keep`: the sum goes on (then all rows go to one matrix).
template <typename T>
struct StoreEpilogue {
  static constexpr bool kPair = false;
  struct State {
    float alpha;
  };
  int rows, cols;
  T *out, *out2;       // [part, cols] each: of the products' rows, those from `split` (a multiple of 32) on go to out2
  int split, part;
  Scale scale;
  float *sum;          // [rows, cols] or null
  bool begins, keep;   // the first piece of a sum, not the last one
  int align, sum_align;
  float *parts;        // [parts of k][rows][pitch]: sums that another kernel adds, or null
  int parts_pitch;
  __device__ __forceinline__ void begin(State &s, const Where &, bool) const { s.alpha = scale.value(); }
  __device__ __forceinline__ void unit(State &s, const Where &w, int col, float (&v)[32]) const {
    const int top = w.row - w.lane, row = top < split ? top : top - split;
    const int m = min(32, min(part - row, rows - top)), n = min(32, cols - col);
    if (m <= 0 || n <= 0) return;
    if (parts != nullptr) {  // rows of 32 bytes: whole boxes, in their pitch
      store_box(w, parts + ((size_t)w.part * (size_t)rows + (size_t)top) * (size_t)parts_pitch + col, (size_t)parts_pitch, m, min(32, parts_pitch - col), 32, v);
      return;
    }
    if (sum != nullptr) {
      float *acc = sum + (size_t)top * (size_t)cols + col;
      if (!begins) {
        float before[32];
        load_box(w, acc, (size_t)cols, m, n, sum_align, before);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] += before[i];
      }
      if (keep) {
        store_box(w, acc, (size_t)cols, m, n, sum_align, v);
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= s.alpha;
    store_box(w, (top < split ? out : out2) + (size_t)row * (size_t)cols + col, (size_t)cols, m, n, align, v);
  }
  __device__ __forceinline__ void end(State &, const Where &) const {}
};

// out = alpha sum_part parts[part], parts ascending; 4 columns a thread.  Reads 4 bytes a value and part, at the memory's or L2's speed.
template <typename T>
__global__ void __launch_bounds__(256) add_parts_kernel(const StoreEpilogue<T> e, int count) {
  after_previous_kernel();
  const float alpha = e.scale.value();
  const int quads = e.parts_pitch / 4;
  const int64_t n = (int64_t)e.rows * quads, step = (int64_t)gridDim.x * 256;
  const size_t plane = (size_t)e.rows * (size_t)e.parts_pitch;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += step) {
    const int r = (int)(i / quads), c = (int)(i - (int64_t)r * quads) * 4, row = r < e.split ? r : r - e.split;
    if (c >= e.cols || row >= e.part) continue;
    const float *from = e.parts + (size_t)r * (size_t)e.parts_pitch + c;
    float4 sum = load_plain(reinterpret_cast<const float4 *>(from));
#pragma unroll 4
    for (int p = 1; p < count; ++p) {
      const float4 q = load_plain(reinterpret_cast<const float4 *>(from + (size_t)p * plane));
      sum.x += q.x, sum.y += q.y, sum.z += q.z, sum.w += q.w;
    }
    T *to = (r < e.split ? e.out : e.out2) + (size_t)row * (size_t)e.cols + c;
    const float v[4] = {alpha * sum.x, alpha * sum.y, alpha * sum.z, alpha * sum.w};
    if (e.align >= 4 * (int)sizeof(T) && c + 4 <= e.cols) {
      if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4 *>(to) = make_float4(v[0], v[1], v[2], v[3]);
      else
        *reinterpret_cast<uint2 *>(to) = make_uint2(pack_pair(v[0], v[1], to), pack_pair(v[2], v[3], to));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < e.cols) to[j] = from_float<T>(v[j]);
    }
  }
}

// ---- operands ---------------------------------------------------------------------------------------------------------

constexpr int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Memory handed out of a workspace in pieces of 256 bytes; with no base it only counts.
struct Arena {
  char *base;
  size_t used = 0;
  explicit Arena(void *at) : base(static_cast<char *>(at)) {}
  template <typename P>
  P *take(int64_t count) {
    P *p = base == nullptr ? nullptr : reinterpret_cast<P *>(base + used);
    used += align_up((size_t)std::max<int64_t>(count, 0) * sizeof(P), 256);
    return p;
  }
};

// A matrix as the tile product reads it, K = Kind or GradKind of its type: itself, or laid out anew (`copy`).  What K splits is split into
// planes, 16-bit rows that do not start on 16 bytes are padded, and rows whose target is `ignore` come as zeros where `target` is given.
template <typename T, typename K = Kind<T>>
struct Operand {
  Matrix m;
  typename K::Operand *copy = nullptr;
  const T *source = nullptr;
  int64_t stride = 0;
  const int64_t *target = nullptr;
  int64_t ignore = 0;
  static bool direct(int64_t stride) { return K::kPlanes == 1 && stride % 8 == 0; }
  bool ready = false;  // the copy has been made by an earlier call
  // `skips`: rows whose target is the ignored one come as zeros, in a copy.
  void set(Arena &arena, const T *data, int64_t rows, int64_t cols, int64_t row_stride, bool skips = false, const int64_t *skip = nullptr,
           int64_t skipped = 0) {
    source = data, stride = row_stride, target = skip, ignore = skipped;
    m.rows = rows, m.cols = cols, m.planes = K::kPlanes;
    if (direct(row_stride) && !skips) {
      m.data = data, m.pitch = row_stride;
      return;
    }
    m.pitch = round_up(cols, 8);
    m.plane = rows * m.pitch;
    copy = arena.template take<typename K::Operand>(m.plane * m.planes);
    m.data = copy;
  }
};
// The other operand of the products that a gradient enters, where that is not what the forward reads.
template <typename T>
struct GradOperand : Operand<T, GradKind<T>> {
  // `rows` rows from `first` on, out of the matrix, or out of its copy where an earlier call has made one (whose rows start on 16 bytes).
  void from(const Operand<T> &o, int64_t first, int64_t rows) {
    const bool again = o.copy != nullptr && o.ready;
    this->source = (again ? reinterpret_cast<const T *>(o.copy) : o.source) + first * (again ? o.m.pitch : o.stride);
    this->stride = again ? o.m.pitch : o.stride;
    this->m.rows = rows;
  }
};
template <typename T>
constexpr bool kSameOperands = Kind<T>::kPlanes == GradKind<T>::kPlanes;

// The copies of a call's operands, all in one launch.
template <typename T>
struct LayOut {
  struct Job {
    const T *source;
    void *copy;
    int64_t rows, cols, stride, pitch, plane, ignore;
    const int64_t *target;
    int planes;
    bool whole;  // rows of the source start on 16 bytes
  } jobs[6];
  unsigned count;
  template <typename K>
  void add(const Operand<T, K> &o) {
    if (o.copy == nullptr || o.ready || o.m.rows == 0) return;
    const bool whole = (reinterpret_cast<uintptr_t>(o.source) & 15u) == 0 && o.stride * (int64_t)sizeof(T) % 16 == 0;
    jobs[count++] = {o.source, o.copy, o.m.rows, o.m.cols, o.stride, o.m.pitch, o.m.plane, o.ignore, o.target, o.m.planes, whole};
  }
};

// 8 columns a thread.  x is read once, the copy written once: 10 bytes a value from fp32, 4 from 16 bits (6 into two planes); 8192 x 1024 of fp32 in 13 us
// (6.3 TB/s), 10007 x 771 of fp16, whose rows start on odd addresses, in 9 (3.4 TB/s: loads of single values).
template <typename T>
__global__ void __launch_bounds__(256) lay_out_kernel(const __grid_constant__ LayOut<T> all) {
  after_previous_kernel();
  const typename LayOut<T>::Job &a = all.jobs[blockIdx.y];
  const int64_t per_row = a.pitch / 8, n = a.rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / per_row, c = (i - r * per_row) * 8;
    float v[8];
    const T *from = a.source + r * a.stride + c;
    if (a.target != nullptr && load_plain(a.target + r) == a.ignore) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    } else if (a.whole && c + 8 <= a.cols) {
      T t[8];
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<uint4 *>(t) = load_plain(reinterpret_cast<const uint4 *>(from));
        *reinterpret_cast<uint4 *>(t + 4) = load_plain(reinterpret_cast<const uint4 *>(from + 4));
      } else {
        *reinterpret_cast<uint4 *>(t) = load_plain(reinterpret_cast<const uint4 *>(from));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_float(t[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < a.cols ? to_float(from[j]) : 0.0f;
    }
    if (Kind<T>::kPlanes == 1 && a.planes == 1) {
      typename Kind<T>::Operand *to = static_cast<typename Kind<T>::Operand *>(a.copy) + r * a.pitch + c;
      *reinterpret_cast<uint4 *>(to) = make_uint4(pack_pair(v[0], v[1], to), pack_pair(v[2], v[3], to), pack_pair(v[4], v[5], to), pack_pair(v[6], v[7], to));
    } else if constexpr (GradKind<T>::kPlanes > 1) {
      constexpr int kPlanes = GradKind<T>::kPlanes;  // (two: the third one of 11 bits is 0)
      __nv_bfloat16 *to = static_cast<__nv_bfloat16 *>(a.copy) + r * a.pitch + c;
      uint32_t p[3][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) split_pair(v[2 * j], v[2 * j + 1], p[0][j], p[1][j], p[2][j]);
#pragma unroll
      for (int q = 0; q < kPlanes; ++q) *reinterpret_cast<uint4 *>(to + q * a.plane) = make_uint4(p[q][0], p[q][1], p[q][2], p[q][3]);
    }
  }
}

inline unsigned blocks_for(int64_t work, int64_t per_block, int64_t most) {
  return (unsigned)std::min<int64_t>(std::max<int64_t>((work + per_block - 1) / per_block, 1), most);
}

template <typename T>
int lay_out(const LayOut<T> &all, cudaStream_t stream) {
  if (all.count == 0) return HT_OK;
  int64_t most = 0;
  for (unsigned i = 0; i < all.count; ++i) most = std::max(most, all.jobs[i].rows * (all.jobs[i].pitch / 8));
  return launch_next<lay_out_kernel<T>>(dim3(blocks_for(most, 256, 148 * 16), all.count), 256, 0, 0, stream, 1, all);
}
template <typename T, typename... Operands>
int lay_out(cudaStream_t stream, const Operands &...operands) {
  LayOut<T> all = {};
  (all.add(operands), ...);
  return lay_out(all, stream);
}

// Sums of 32 rows that an epilogue leaves for these rows: of every tile's, inside the matrix or not.
inline int64_t row_sum_count(int64_t rows, const TileShape &shape) { return (rows + shape.rows() - 1) / shape.rows() * shape.rows() / 32; }

// Column sums from the sums of 32 rows each that the epilogues leave: out[c] = alpha sum_r partial[r, c], r in 32 strands,
// ascending in each, that are added in order.  32 columns a block; columns from `second` on go to out2.  256 sums of 1000 columns 6 us, latency.
template <typename T>
__global__ void __launch_bounds__(1024) column_sums_kernel(const float *partial, int64_t rows, int64_t pitch, int64_t cols, int64_t second,
                                                          Scale scale, T *out, T *out2) {
  after_previous_kernel();
  __shared__ float strand[32][33];
  const int lane = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane, part = c < second ? c : c - second;
  T *const to = c < second ? out : out2;
  const bool inside = part < cols && to != nullptr;
  float sum = 0.0f;
  if (inside)
#pragma unroll 4
    for (int64_t r = y; r < rows; r += 32) sum += load_plain(partial + r * pitch + c);
  strand[y][lane] = sum;
  __syncthreads();
  if (y == 0 && inside) {
#pragma unroll
    for (int i = 1; i < 32; ++i) sum += strand[i][lane];
    to[part] = from_float<T>(scale.value() * sum);
  }
}

// (out2: the sums from column `second` on; null, or one of the two null: those are not wanted)
template <typename T>
int column_sums(const float *partial, int64_t rows, int64_t pitch, int64_t cols, const Scale &scale, T *out, T *out2, int64_t second, cudaStream_t stream) {
  return launch_next<column_sums_kernel<T>>(dim3((unsigned)(((out2 != nullptr ? second : 0) + cols + 31) / 32)), 1024, 0, 0, stream, 1, partial, rows, pitch, cols,
                     second, scale, out, out2);
}

// Outputs of a piece where `most` fit the bound: all of them, or pieces of whole tiles, about equal, 256 at the least.
inline int64_t piece_of(int64_t outputs, int64_t most) {
  if (most >= outputs) return outputs;
  const int64_t whole = std::max<int64_t>(most / 256 * 256, 256), pieces = (outputs + whole - 1) / whole;
  return std::min(outputs, round_up((outputs + pieces - 1) / pieces, 256));
}

// The two products of a backward pass (ht_dense_products.cu): dx (+)= g w over a piece of the outputs, dw = g^T x.  `parts`: room for
// product_parts() floats, or null; what a product with few tiles is cut into along k is summed there.
constexpr int kMostParts = 16;
inline TileShape product_shape(int64_t rows, int64_t cols, int64_t k, int planes, bool in_parts) {
  return tile_shape(rows, cols, k, planes, false, in_parts ? kMostParts : 1);
}
inline int64_t product_parts(int64_t rows, int64_t cols, int64_t k, int planes) {
  const int split = product_shape(rows, cols, k, planes, true).split;
  return split > 1 ? split * rows * round_up(cols, 8) : 0;
}
template <typename T>
int product_dx(const TileProblem &p, StoreEpilogue<T> e, float *parts, int sms, cudaStream_t stream);
template <typename T>
int product_dw(const TileProblem &p, StoreEpilogue<T> e, float *parts, int sms, cudaStream_t stream);

}  // namespace dense
}  // namespace ht
