// y = x W^T + bias under weights held as microscaled 4-bit numbers (ht_mx4.cuh).
//
// A weight is exact in bf16, so that x alone decides the products: one of bf16 values, two of fp16 (two bf16 numbers a value, exact), three of
// fp32 (three numbers, 24 bits), summed in fp32.
#include "ht_mx4_tile.cuh"

namespace ht {
namespace mx4 {
namespace {

using dense::after_previous_kernel;
using dense::to_float;

// x's bf16 numbers a value.
template <typename T>
constexpr int kNumbers = std::is_same<T, __nv_bfloat16>::value ? 1 : std::is_same<T, __half>::value ? 2 : 3;

// ---- few rows ---------------------------------------------------------------------------------------------------------
// A warp takes 16 outputs (the 16 rows of mma.sync's first operand) and 128 features, of which a lane has a block of 32 of two outputs: their codes
// are 16 contiguous bytes each, read straight into registers, some groups of outputs ahead.  x, the other operand, is in registers for good where
// one warp's share of the features never changes: up to 16 warps share a group of outputs, and their sums meet in shared memory, those of four
// groups at a time.
// What bounds it: latency.  The bytes alone take 4.2 us, decoding (11 instructions of half rate for 8 weights) 3.9; issue slots are 48 % and the
// ALU pipe 47 % in use, and an instruction waits for loads for 2.1 of its 7 cycles, with one CTA of 16 warps an SM, 8 warps to 1024
// features of 16 outputs, whose sums have to meet, and 11 such groups a team, which are three uneven turns.  Measured, 1024 to 50000: 1 to 8 rows of bf16
// 12.6 us, 16 rows 15.4, 8 rows of fp16 14.4, of fp32 18.5 (the unpacked layer as torch's bf16 product: 1 row 22.7, 16 rows 23.1); 784 to 12700, 1 row
// 5.5, most of it the launch.  Beyond 2048 features x does not stay in registers but is loaded for every 16 outputs: 2048 to 50000 24.5 us for 1 to 8 rows
// and 28 for 16, 4096 to 50000 83 to 89 and 124, of which 17 rows take 55 as a tile.
constexpr int kFewThreads = 512, kFewWarps = kFewThreads / 32;

template <typename T>
struct FewArgs {
  const T *x, *bias;
  const uint8_t *codes, *scales;
  T *y;
  int64_t x_stride;
  int rows, features, outputs, blocks;
  int chunks;  // of 4 blocks of features
  int sharing; // warps that share a group of outputs
  bool whole;  // rows of x start on 16 bytes
};

// A lane's 32 features of one row of x as pairs of neighbours, number by number.
template <typename T>
__device__ __forceinline__ void load_x(const FewArgs<T> &a, int row, int k, uint32_t (&x)[kNumbers<T>][16]) {
  constexpr int kPer = 16 / (int)sizeof(T);
  const T *from = a.x + (int64_t)row * a.x_stride + k;
  const bool there = row < a.rows;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float v[8];
    if (there && a.whole && k + 8 * q + 8 <= a.features) {
#pragma unroll
      for (int j = 0; j < 8; j += kPer) {
        T t[kPer];
        *reinterpret_cast<uint4 *>(t) = load_plain(reinterpret_cast<const uint4 *>(from + 8 * q + j));
#pragma unroll
        for (int n = 0; n < kPer; ++n) v[j + n] = to_float(t[n]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = there && k + 8 * q + j < a.features ? to_float(from[8 * q + j]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kNumbers<T> == 1) {
        x[0][4 * q + i] = dense::pack_pair(v[2 * i], v[2 * i + 1], static_cast<const __nv_bfloat16 *>(nullptr));
      } else {
        uint32_t third;
        dense::split_pair(v[2 * i], v[2 * i + 1], x[0][4 * q + i], x[1][4 * q + i], third);
        if constexpr (kNumbers<T> == 3) x[2][4 * q + i] = third;
      }
    }
  }
}

struct Codes {  // a lane's of two outputs
  uint4 a, b;
  uint8_t scale_a, scale_b;  // (as they are loaded: what touches them waits for them)
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T, int NT, int AHEAD>
__global__ void __launch_bounds__(kFewThreads, 1) few_rows_kernel(const FewArgs<T> a) {
  constexpr int P = kNumbers<T>;
  extern __shared__ __align__(16) float few_sums[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, j = lane & 3;
  const int team = warp / a.sharing, part = warp - team * a.sharing, teams = kFewWarps / a.sharing;
  const int row0 = (int)blockIdx.y * (8 * NT);
  const int groups = (a.outputs + 15) / 16, first = team * (int)gridDim.x + (int)blockIdx.x, stride = teams * (int)gridDim.x;
  after_previous_kernel();
  if (team >= teams) return;

  const uint32_t number = opaque_one();
  uint32_t x[NT][P][16];
  auto fragments = [&](int chunk) {
#pragma unroll
    for (int n = 0; n < NT; ++n) load_x(a, row0 + 8 * n + g, (4 * chunk + j) * kBlock, x[n]);
  };
  // The codes of a chunk of two outputs of a group.
  auto fetch = [&](int group, int chunk) {
    Codes c = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u), 127, 127};
    const int block = 4 * chunk + j, o = group * 16 + g;
    const int64_t at = (int64_t)o * a.blocks + block, bt = at + 8 * (int64_t)a.blocks;
    if (o < a.outputs && block < a.blocks) {
      c.a = load_plain(reinterpret_cast<const uint4 *>(a.codes) + at);
      c.scale_a = load_plain(a.scales + at);
    }
    if (o + 8 < a.outputs && block < a.blocks) {
      c.b = load_plain(reinterpret_cast<const uint4 *>(a.codes) + bt);
      c.scale_b = load_plain(a.scales + bt);
    }
    return c;
  };
  auto multiply = [&](const Codes &c, float (&sum)[NT][4]) {
    const Scale sa = scale_of(c.scale_a), sb = scale_of(c.scale_b);
    const uint32_t wa[4] = {c.a.x, c.a.y, c.a.z, c.a.w}, wb[4] = {c.b.x, c.b.y, c.b.z, c.b.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t va[4], vb[4];
      weights_of(wa[q], sa, number, va);
      weights_of(wb[q], sb, number, vb);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if constexpr (P == 1) {
#pragma unroll
          for (int h = 0; h < 4; h += 2) mma_bf16(sum[n], va[h], vb[h], va[h + 1], vb[h + 1], x[n][0][4 * q + h], x[n][0][4 * q + h + 1]);
        } else {  // the tensor core truncates what it adds to: short sums, the small ones first, added in fp32
          float fresh[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int p = P - 1; p >= 0; --p)
#pragma unroll
            for (int h = 0; h < 4; h += 2) mma_bf16(fresh, va[h], vb[h], va[h + 1], vb[h + 1], x[n][p][4 * q + h], x[n][p][4 * q + h + 1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[n][i] += fresh[i];
        }
      }
    }
  };
  // The warps' sums of AHEAD groups meet: [AHEAD][warps][NT][32] of 4, twice, so that the next ones need not wait for these to have been read.
  constexpr int kGroupSums = kFewWarps * NT * 32;
  float4 *const sums = reinterpret_cast<float4 *>(few_sums);
  uint32_t buffer = 0;
  auto leave = [&](int d, const float (&sum)[NT][4]) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
      sums[(buffer * AHEAD + d) * kGroupSums + (warp * NT + n) * 32 + lane] = make_float4(sum[n][0], sum[n][1], sum[n][2], sum[n][3]);
  };
  auto finish = [&](int base, int count) {
    if (a.sharing > 1)
      asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(a.sharing * 32) : "memory");
    else
      __syncwarp();
    for (int f = part * 32 + lane; f < count * NT * 32; f += a.sharing * 32) {
      const int of = f & 31, n = f / 32 % NT, d = f / (32 * NT);
      const float4 *from = sums + (buffer * AHEAD + d) * kGroupSums + (team * a.sharing * NT + n) * 32 + of;
      float4 v = from[0];
      for (int p = 1; p < a.sharing; ++p) {
        const float4 q = from[p * NT * 32];
        v.x += q.x, v.y += q.y, v.z += q.z, v.w += q.w;
      }
      // number i of four is output g + 8 (i / 2) and row 2 j + i % 2 of the lane whose they are
      const int o = (base + d * stride) * 16 + (of >> 2), row = row0 + 8 * n + 2 * (of & 3);
      const float each[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int to = o + 8 * (i >> 1), at = row + (i & 1);
        if (at >= a.rows || to >= a.outputs) continue;
        float y = each[i] * kHeld;
        if (a.bias != nullptr) y += to_float(a.bias[to]);
        a.y[(int64_t)at * a.outputs + to] = dense::from_float<T>(y);
      }
    }
    buffer ^= 1u;  // (the next sums go to the other half, and those after them come after the next barrier)
  };

  if (a.chunks <= a.sharing) {
    Codes ahead[AHEAD];
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) ahead[d] = fetch(first + d * stride, part);
    fragments(part);
    for (int base = first; base < groups; base += AHEAD * stride) {
      int count = 0;
#pragma unroll
      for (int d = 0; d < AHEAD; ++d) {
        const int group = base + d * stride;
        if (group >= groups) break;
        const Codes c = ahead[d];
        ahead[d] = fetch(group + AHEAD * stride, part);
        float sum[NT][4] = {};
        multiply(c, sum);
        leave(d, sum);
        ++count;
      }
      finish(base, count);
    }
  } else {
    for (int group = first; group < groups; group += stride) {
      float sum[NT][4] = {};
      Codes next = fetch(group, part);
      for (int chunk = part; chunk < a.chunks; chunk += a.sharing) {
        const Codes c = next;
        if (chunk + a.sharing < a.chunks) next = fetch(group, chunk + a.sharing);
        fragments(chunk);
        multiply(c, sum);
      }
      leave(0, sum);
      finish(group, 1);
    }
  }
}

int screen(const ht_dense_problem *p) {
  if (p == nullptr || p->rows < 0 || p->features < 1 || p->outputs < 1 || p->x_stride < p->features) return HT_ERR_INVALID_ARGUMENT;
  if (p->dtype != HT_DTYPE_F32 && p->dtype != HT_DTYPE_BF16 && p->dtype != HT_DTYPE_F16) return HT_ERR_INVALID_ARGUMENT;
  if (p->rows > 0x7fffff00 || p->features > 0x3fffff00 || p->outputs > 0x3fffff00) return HT_ERR_UNSUPPORTED;
  return HT_OK;
}

template <typename T, int NT, int AHEAD>
int launch_few(const FewArgs<T> &a, cudaStream_t stream) {
  const int groups = (a.outputs + 15) / 16;
  constexpr size_t kBytes = sizeof(float) * 2 * AHEAD * kFewWarps * NT * 128;
  const dim3 grid((unsigned)std::min(groups, 148), (unsigned)((a.rows + 8 * NT - 1) / (8 * NT)));
  return dense::launch_next<few_rows_kernel<T, NT, AHEAD>>(grid, kFewThreads, kBytes, kBytes, stream, 1, a);
}

// Whether the rows are few enough for the kernel above: 17 rows of bf16, 1024 to 50000, take 16.8 us as a tile, 16 rows 15.4 here; 9 rows of fp16 21.8
// and of fp32 22.1 as a tile, 8 rows 14.5 and 18.7 here (two groups of 8 rows would read the weights twice).
template <typename T>
bool few_rows(int64_t rows) {
  return rows <= (kNumbers<T> == 1 ? 16 : 8);
}

// ---- many rows of bf16 ------------------------------------------------------------------------------------------------
// Weights decoded once, into memory, as the tile kernel's operands are (2^-5 of their values), and the pair kernel of ht_dense_tile.cuh.  Decoding is
// bound by memory: 27 MB in and 102 out for 50000 x 1024, 25 us.
__global__ void __launch_bounds__(256) decode_kernel(const uint32_t *codes, const uint8_t *scales, uint4 *out, int64_t words) {
  after_previous_kernel();
  const uint32_t one = opaque_one();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
    uint32_t v[4];
    weights_of(dense::load_plain(codes + i), scale_of(dense::load_plain(scales + i / 4)), one, v);
    out[i] = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

template <typename T>
struct ScoresEpilogue {
  static constexpr bool kPair = false;
  struct State {};
  int rows, cols;
  const T *bias;
  T *y;  // [rows, cols], `pitch` from row to row
  int64_t pitch;
  int align;
  __device__ __forceinline__ void begin(State &, const dense::Where &, bool) const {}
  __device__ __forceinline__ void unit(State &, const dense::Where &w, int col, float (&v)[32]) const {
    const int n = cols - col, top = w.row - w.lane;
    if (n <= 0 || top >= rows) return;
    float b[32];
    if (bias != nullptr)
      dense::load_columns(bias + col, b, n);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = fmaf(v[i], kHeld, bias != nullptr ? b[i] : 0.0f);
    dense::store_box(w, y + (size_t)top * (size_t)pitch + col, (size_t)pitch, min(32, rows - top), min(32, n), align, v);
  }
  __device__ __forceinline__ void end(State &, const dense::Where &) const {}
};

// Whether that is the way.  us, decoded for every tile and decoded once, in long loops: 8192 x 1024 to 50000 788 and 660, 1024 rows of it 127 and 112, 512
// rows 66 and 75; 8192 x 784 to 4096 76 and 53; 8192 x 2048 to 1000 38 and 34; 4096 x 200 to 20000 75 and 73; 8192 x 333 to 1001 19 and 26; 1024 x
// 1024 to 1000 8 and 13.  fp16 and fp32 rows are not among them: the pair kernel has as many numbers a value on both sides, 3 products for two
// and 6 for three, where weights of one number take 2 and 3.
template <typename T>
bool many_rows(const ht_dense_problem &p, int64_t outputs) {
  return kNumbers<T> == 1 && p.rows >= 1024 && (double)p.rows * (double)p.features * (double)outputs >= 1e10;
}
// Outputs that are decoded at a time: what the caller's limit holds of them, whole tiles; 0 where that is not the way, or where a piece is
// too little work for it.
constexpr int64_t kDecodedBytes = (int64_t)512 << 20;
template <typename T>
int64_t decoded_outputs(const ht_dense_problem &p) {
  const int64_t limit = p.scratch_limit > 0 ? std::min(p.scratch_limit, kDecodedBytes) : kDecodedBytes;
  const int64_t most = limit / (blocks_of(p.features) * kBlock * (int64_t)sizeof(__nv_bfloat16));
  const int64_t piece = p.outputs <= most ? p.outputs : most / 256 * 256;
  return many_rows<T>(p, piece) ? piece : 0;
}

template <typename T>
struct Plan {
  dense::Operand<T, dense::GradKind<T>> x;
  dense::Matrix w;  // decoded, where the rows are many: all outputs or a piece of them
  size_t bytes = 0;
  Plan(const ht_dense_problem &p, const void *xp, void *ws) {
    dense::Arena arena(ws);
    if (!few_rows<T>(p.rows)) x.set(arena, static_cast<const T *>(xp), p.rows, p.features, p.x_stride);
    const int64_t piece = decoded_outputs<T>(p);
    if (piece > 0) {
      w.rows = piece, w.cols = p.features, w.pitch = blocks_of(p.features) * kBlock;
      w.data = arena.template take<__nv_bfloat16>(w.rows * w.pitch);
    }
    bytes = arena.used;
  }
};

template <typename T>
int forward(const ht_dense_problem &p, const void *x, const void *codes, const void *scales, const void *bias, void *y, void *ws, size_t ws_bytes,
            uint32_t *status_word, cudaStream_t stream) {
  static_assert(kNumbers<T> == dense::GradKind<T>::kPlanes, "the operand's planes are x's numbers");
  if (!few_rows<T>(p.rows)) {
    Plan<T> plan(p, x, ws);
    if (plan.bytes > ws_bytes || (plan.bytes > 0 && ws == nullptr)) return HT_ERR_WORKSPACE;
    int sms = 0;
    HT_TRY(dense::sm_count(&sms));
    HT_TRY(dense::lay_out<T>(stream, plan.x));
    if constexpr (kNumbers<T> == 1)
      if (plan.w.data != nullptr) {
        const int64_t piece = plan.w.rows, per_output = blocks_of(p.features) * 4;
        for (int64_t first = 0; first < p.outputs; first += piece) {
          const int64_t count = std::min(piece, p.outputs - first), words = count * per_output;
          HT_TRY((dense::launch_next<decode_kernel>(dim3(dense::blocks_for(words, 1024, 148 * 16)), 256, 0, 0, stream, 1,
                                                    static_cast<const uint32_t *>(codes) + first * per_output,
                                                    static_cast<const uint8_t *>(scales) + first * per_output / 4,
                                                    static_cast<uint4 *>(const_cast<void *>(plan.w.data)), words)));
          dense::TileProblem t;
          t.a[0] = plan.x.m;
          t.b[0] = plan.w;
          t.b[0].rows = count;
          t.rows = p.rows, t.cols = count, t.k = p.features;
          t.status_word = status_word;
          T *const to = static_cast<T *>(y) + first;
          const ScoresEpilogue<T> e = {(int)p.rows, (int)count, bias != nullptr ? static_cast<const T *>(bias) + first : nullptr, to, p.outputs,
                                       dense::row_alignment(to, p.outputs * (int64_t)sizeof(T))};
          HT_TRY((dense::launch_tiles<1, false, false>(t, e, dense::tile_shape(p.rows, count, p.features, 1, false), sms, stream)));
        }
        return HT_OK;
      }
    return launch_tiles<T, kNumbers<T>>(plan.x.m, codes, static_cast<const uint8_t *>(scales), static_cast<const T *>(bias), static_cast<T *>(y), p.rows,
                                        p.features, p.outputs, status_word, sms, stream);
  }
  FewArgs<T> a = {};
  a.x = static_cast<const T *>(x), a.bias = static_cast<const T *>(bias), a.y = static_cast<T *>(y);
  a.codes = static_cast<const uint8_t *>(codes), a.scales = static_cast<const uint8_t *>(scales);
  a.x_stride = p.x_stride;
  a.rows = (int)p.rows, a.features = (int)p.features, a.outputs = (int)p.outputs, a.blocks = (int)blocks_of(p.features);
  a.chunks = (a.blocks + 3) / 4;
  a.sharing = std::min(a.chunks, kFewWarps);
  a.whole = p.x_stride * (int64_t)sizeof(T) % 16 == 0 || p.rows == 1;
  if constexpr (kNumbers<T> == 1) {
    return p.rows <= 8 ? launch_few<T, 1, 4>(a, stream) : launch_few<T, 2, 4>(a, stream);
  } else {
    return launch_few<T, 1, 4>(a, stream);
  }
}

template <typename F>
int by_type(int dtype, F &&f) {
  return dtype == HT_DTYPE_F32 ? f(float()) : dtype == HT_DTYPE_BF16 ? f(__nv_bfloat16()) : f(__half());
}

bool aligned(std::initializer_list<const void *> pointers) {
  uintptr_t all = 0;
  for (const void *p : pointers) all |= reinterpret_cast<uintptr_t>(p);
  return (all & 15u) == 0;
}

}  // namespace
}  // namespace mx4
}  // namespace ht

using namespace ht;
using namespace ht::mx4;

extern "C" size_t ht_linear_mx4_workspace_bytes(const ht_dense_problem *p) {
  if (screen(p) != HT_OK || p->rows == 0) return 0;
  size_t bytes = 0;
  by_type(p->dtype, [&](auto zero) -> int {
    bytes = Plan<decltype(zero)>(*p, nullptr, nullptr).bytes;
    return HT_OK;
  });
  return bytes;
}

extern "C" int ht_linear_mx4(const ht_dense_problem *p, const void *x, const void *codes, const void *scales, const void *bias, void *y, void *workspace,
                             size_t workspace_bytes, uint32_t *status_word, ht_stream_t stream) {
  const int rc = screen(p);
  if (rc != HT_OK) return rc;
  if (p->rows == 0) return HT_OK;
  if (x == nullptr || codes == nullptr || scales == nullptr || y == nullptr) return HT_ERR_INVALID_ARGUMENT;
  if (!aligned({x, codes, scales, bias, y})) return HT_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return HT_ERR_WORKSPACE;
  return by_type(p->dtype, [&](auto zero) -> int {
    return forward<decltype(zero)>(*p, x, codes, scales, bias, y, workspace, workspace_bytes, status_word, reinterpret_cast<cudaStream_t>(stream));
  });
}
