// The dense layers for few rows (answers to single samples, small batches): every weight is read once, straight into registers.
//
// A warp takes 16 rows of the weights (of a pair: 8 of each matrix) as one operand of mma.sync and up to 8 NT rows of x, which lie in shared
// memory, as the other.  A sum of products does not mind in which order its terms come, so a lane's share of k is 16 contiguous bytes
// of a row, not what the instruction's layout spreads over it: whole sectors are read, and a lane fetches what it uses itself, into a ring of 8
// steps of its own in shared memory (cp.async), 7 of them in flight, across the ends of rows: 112 KB an SM; with the loads of 4 steps in registers
// instead, 205 MB of fp32 weights took 73 us.
// fp32 values are taken as three bf16 numbers like in the tiles, six products; those of a step (16 values of k) start in a fresh accumulator, the
// small ones first, and are added in fp32 from there on (the tensor core truncates when it adds).  Off by 1.0e-7 in norm at 1024 values of k,
// cuBLAS's fp32 products by 1.5e-7 to 2.7e-7.
// With few weights several warps of a block share 16 rows and take k in turn.
// What bounds it: the weights' bytes; the launch with few of them.  Measured, 1 row of bf16: 205 MB of weights 38 us (5.4 TB/s), 40 MB 7.5 us; 16
// rows 41 and 8.7.  1 row of fp32, 205 MB: 49 us with the loss's second kernel, 32 rows 121 (the splits of x, which every warp makes again).
#pragma once

#include "ht_dense.cuh"

namespace ht {
namespace dense {

constexpr int kFewThreads = 512, kFewWarps = kFewThreads / 32;
constexpr int kFewRing = 8;  // steps of k in flight
constexpr uint32_t kFewRingBytes = kFewWarps * kFewRing * 1024;
// of x in shared memory and of the warps' sums: what the rings and an epilogue's own 4 KB leave
constexpr int64_t kFewMostBytes = 222 * 1024 - (int64_t)kFewRingBytes;

template <typename T>
struct FewArgs {
  const T *x, *w[2];
  int64_t x_stride;
  int rows, features, outputs;
  int pitch;     // bytes of a row of x in shared memory: 64 more than a multiple of 128, so that 8 rows of 64 bytes meet in no bank
  bool x_whole;  // rows of x start on 16 bytes
  int split;     // warps that share 16 rows of the weights: a power of two
};

template <typename T>
__device__ __forceinline__ void mma_few(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four values as three bf16 numbers each, two to a word.
struct Planes {
  uint32_t p[3][2];
};
__device__ __forceinline__ Planes split_four(const uint4 &q) {
  Planes r;
  split_pair(__uint_as_float(q.x), __uint_as_float(q.y), r.p[0][0], r.p[1][0], r.p[2][0]);
  split_pair(__uint_as_float(q.z), __uint_as_float(q.w), r.p[0][1], r.p[1][1], r.p[2][1]);
  return r;
}
// sum += the products of 16 values of k of the rows a and b of the weights with those of x.
__device__ __forceinline__ void mma_planes(float (&sum)[4], const Planes &a, const Planes &b, const Planes &x) {
  float fresh[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  auto product = [&](int w, int of_x) {
    const uint32_t rows[4] = {a.p[w][0], b.p[w][0], a.p[w][1], b.p[w][1]};
    mma_few<__nv_bfloat16>(fresh, rows, x.p[of_x][0], x.p[of_x][1]);
  };
  product(2, 0), product(0, 2), product(1, 1), product(1, 0), product(0, 1), product(0, 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) sum[i] += fresh[i];
}

// A lane's 16 bytes of a row from place `k` on, zeros behind its end, value by value.
template <typename T>
__device__ __forceinline__ uint4 load_values(const T *row, int k, int features) {
  constexpr int kValues = 16 / (int)sizeof(T);
  T t[kValues];
#pragma unroll
  for (int j = 0; j < kValues; ++j) t[j] = k + j < features ? row[k + j] : from_float<T>(0.0f);
  return *reinterpret_cast<uint4 *>(t);
}
// The same into shared memory, without waiting where the row starts on 16 bytes (FULL).
template <typename T, bool FULL>
__device__ __forceinline__ void fetch_values(uint32_t to, const T *row, int k, int features) {
  if constexpr (FULL) {
    const int bytes = k < features ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(row + (k < features ? k : 0)), "r"(bytes) : "memory");
  } else {
    const uint4 q = load_values(row, k, features);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(q.x), "r"(q.y), "r"(q.z), "r"(q.w) : "memory");
  }
}

template <typename T, int NT, bool FULL, class Epilogue>
__global__ void __launch_bounds__(kFewThreads, 1) few_rows_kernel(const FewArgs<T> a, const Epilogue epilogue) {
  constexpr bool kPair = Epilogue::kPair;
  constexpr bool kFloat = std::is_same<T, float>::value;
  constexpr int kValues = 16 / (int)sizeof(T), kStep = 4 * kValues;  // of k: a lane's, a warp's
  constexpr int kOutputs = kPair ? 8 : 16;
  extern __shared__ __align__(128) unsigned char few_smem[];  // the rings, x, then (split) the warps' sums
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, j = lane & 3;
  const int row0 = (int)blockIdx.y * (8 * NT), held = min(8 * NT, a.rows - row0);
  const int steps = (a.features + kStep - 1) / kStep;
  const int groups = (a.outputs + kOutputs - 1) / kOutputs;
  const int part = warp % a.split;
  // this warp's groups: neighbours go to different blocks, so that every SM reads as much
  const int first = (warp / a.split) * (int)gridDim.x + (int)blockIdx.x, stride = kFewWarps / a.split * (int)gridDim.x;
  const int own = part < steps ? (steps - part + a.split - 1) / a.split : 0;  // steps of this warp in a group
  const uint32_t ring = smem_addr(few_smem) + (uint32_t)(warp * kFewRing) * 1024u + (uint32_t)lane * 16u;

  // What is fetched next: step `fetch_i` of this warp's in the group `fetch_group`.
  int fetch_group = first, fetch_i = 0;
  uint32_t fetch_slot = 0;
  const T *fetch_a = nullptr, *fetch_b = nullptr;
  auto rows_of = [&](int group) {
    const int o = group * kOutputs + g;
    fetch_a = a.w[0] + (int64_t)min(o, a.outputs - 1) * a.features;
    fetch_b = kPair ? a.w[1] + (int64_t)min(o, a.outputs - 1) * a.features : a.w[0] + (int64_t)min(o + 8, a.outputs - 1) * a.features;
  };
  rows_of(fetch_group);
  after_previous_kernel();
  auto fetch = [&]() {
    if (fetch_group < groups && own > 0) {
      const int k = (part + fetch_i * a.split) * kStep + j * kValues;
      fetch_values<T, FULL>(ring + fetch_slot * 1024u, fetch_a, k, a.features);
      fetch_values<T, FULL>(ring + fetch_slot * 1024u + 512u, fetch_b, k, a.features);
      if (++fetch_i == own) {
        fetch_i = 0;
        fetch_group += stride;
        rows_of(fetch_group);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    fetch_slot = (fetch_slot + 1) % kFewRing;
  };
#pragma unroll 1
  for (int i = 0; i < kFewRing - 1; ++i) fetch();

  unsigned char *const xs = few_smem + kFewRingBytes;
  for (int r = warp; r < held; r += kFewWarps) {
    const T *from = a.x + (int64_t)(row0 + r) * a.x_stride;
    for (int i = lane; i < steps * 4; i += 32)
      *reinterpret_cast<uint4 *>(xs + (size_t)r * (size_t)a.pitch + 16 * i) =
          a.x_whole && (i + 1) * kValues <= a.features ? load_plain(reinterpret_cast<const uint4 *>(from) + i) : load_values(from, i * kValues, a.features);
  }
  __syncthreads();
  const uint32_t x_lane = smem_addr(xs) + (uint32_t)(g * a.pitch + 16 * j);
  float4 *sums = reinterpret_cast<float4 *>(xs + (size_t)min(8 * NT, a.rows) * (size_t)a.pitch);  // [warps][NT][32]
  typename Epilogue::template State<NT> state;
  epilogue.begin(state);
  uint32_t slot = 0;
  for (int base = 0; base < groups; base += stride) {  // (as often in every warp)
    const int group = base + first;
    float c[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[n][i] = 0.0f;
    for (int i = 0; i < (group < groups ? own : 0); ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kFewRing - 2) : "memory");
      const uint4 qa = lds_b128(ring + slot * 1024u), qb = lds_b128(ring + slot * 1024u + 512u);
      slot = (slot + 1) % kFewRing;
      const uint32_t wa[4] = {qa.x, qa.y, qa.z, qa.w}, wb[4] = {qb.x, qb.y, qb.z, qb.w};
      Planes pa, pb;
      if constexpr (kFloat) pa = split_four(qa), pb = split_four(qb);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint4 q = make_uint4(0u, 0u, 0u, 0u);
        if (8 * n + g < held) q = lds_b128(x_lane + (uint32_t)(8 * n * a.pitch + 64 * (part + i * a.split)));
        if constexpr (kFloat) {
          mma_planes(c[n], pa, pb, split_four(q));
        } else {
          const uint32_t x[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int h = 0; h < 4; h += 2) {
            const uint32_t w[4] = {wa[h], wb[h], wa[h + 1], wb[h + 1]};
            mma_few<T>(c[n], w, x[h], x[h + 1]);
          }
        }
      }
      fetch();
    }
    if (a.split > 1) {
      __syncthreads();  // the sums of the groups before have been read
#pragma unroll
      for (int n = 0; n < NT; ++n) sums[(warp * NT + n) * 32 + lane] = make_float4(c[n][0], c[n][1], c[n][2], c[n][3]);
      __syncthreads();
      if (part != 0) continue;
#pragma unroll
      for (int n = 0; n < NT; ++n)
        for (int i = 1; i < a.split; ++i) {
          const float4 q = sums[((warp + i) * NT + n) * 32 + lane];
          c[n][0] += q.x, c[n][1] += q.y, c[n][2] += q.z, c[n][3] += q.w;
        }
    }
    // this lane: rows row0 + 8 n + 2 j and the next; outputs o and o + 8, or the gate and the value of o
    const int o = group * kOutputs + g;
#pragma unroll
    for (int n = 0; n < NT; ++n) epilogue.template values<NT>(state, n, row0 + 8 * n + 2 * j, o, a.outputs, c[n]);
  }
  epilogue.template end<NT>(state, row0, lane);
}

// How few rows are computed: tiles of 8 rows (0: by some_rows_kernel), blocks, bytes of a row of x, warps that share weights.
struct FewPlan {
  int tiles, blocks, pitch, split;
};

// Whether the rows are few enough, and how: 32 rows at the most, in groups whose x fits beside the rings.
template <typename T>
bool few_rows(int64_t rows, int64_t features, int64_t outputs, bool pair, FewPlan *plan) {
  if (rows < 1 || rows > 32 || features > (1 << 20)) return false;
  const int64_t pitch = round_up(features * (int64_t)sizeof(T), 128) + 64;
  int tiles = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
  auto bytes = [&]() { return std::min<int64_t>(rows, 8 * tiles) * pitch + (int64_t)sizeof(float4) * 32 * kFewWarps * tiles; };
  while (tiles > 1 && bytes() > kFewMostBytes) tiles /= 2;
  if (bytes() > kFewMostBytes) return false;
  const int64_t groups = (outputs + (pair ? 7 : 15)) / (pair ? 8 : 16), most = 148;
  plan->tiles = tiles;
  plan->pitch = (int)pitch;
  plan->split = 1;
  while (plan->split < kFewWarps && groups * plan->split * 2 <= most * kFewWarps) plan->split *= 2;
  plan->blocks = (int)std::min<int64_t>(groups, most);  // (every SM has its share of the groups, even if some of its warps have none)
  return true;
}

template <typename T, class Epilogue>
int launch_few(FewArgs<T> a, const Epilogue &e, const FewPlan &plan, cudaStream_t stream) {
  a.pitch = plan.pitch;
  a.x_whole = a.x_stride * (int64_t)sizeof(T) % 16 == 0 || a.rows == 1;
  a.split = plan.split;
  const size_t x_bytes = (size_t)std::min(a.rows, 8 * plan.tiles) * (size_t)plan.pitch;
  const size_t bytes = kFewRingBytes + x_bytes + (plan.split > 1 ? sizeof(float4) * 32 * kFewWarps * (size_t)plan.tiles : 0);
  const dim3 grid((unsigned)plan.blocks, (unsigned)((a.rows + 8 * plan.tiles - 1) / (8 * plan.tiles)));
  constexpr size_t kMost = (size_t)kFewRingBytes + (size_t)kFewMostBytes;
  auto by_tiles = [&](auto full) -> int {
    constexpr bool kFull = decltype(full)::value;
    return plan.tiles == 1   ? launch_next<few_rows_kernel<T, 1, kFull, Epilogue>>(grid, kFewThreads, bytes, kMost, stream, 1, a, e)
           : plan.tiles == 2 ? launch_next<few_rows_kernel<T, 2, kFull, Epilogue>>(grid, kFewThreads, bytes, kMost, stream, 1, a, e)
                             : launch_next<few_rows_kernel<T, 4, kFull, Epilogue>>(grid, kFewThreads, bytes, kMost, stream, 1, a, e);
  };
  return a.features * (int64_t)sizeof(T) % 16 == 0 ? by_tiles(std::true_type()) : by_tiles(std::false_type());
}

// ---- some more rows, few weights --------------------------------------------------------------------------------------
// fp32, up to 128 rows: a tile of 128 rows would have a handful of SMs walk k through three planes (100 rows, 1000 to 2 x 700: 35 us).  Here a
// block takes 16 rows of the weights (of a pair: 8 of each), its 16 warps take 64 rows of x each and share k, and x comes straight
// from L2 in the instruction's layout, since no warp uses what another does.  Every step's sum starts afresh and is added in fp32 (chains of 48
// additions in the tensor core lost 1.5e-6 of the sums); the warps' sums are added last, 8 rows a warp.
// What bounds it: rows x k from L2 for every 16 rows of the weights, and the latency of a few loads in a row (100 rows, 1000 to 2 x 700: 17 us;
// 14.5 with two TF32 numbers a value, which the largest finite numbers did not survive).
constexpr int kSomeTiles = 8;  // of 8 rows a warp

template <typename T, class Epilogue>
__global__ void __launch_bounds__(kFewThreads, 1) some_rows_kernel(const FewArgs<T> a, const Epilogue epilogue) {
  constexpr bool kPair = Epilogue::kPair;
  constexpr int kOutputs = kPair ? 8 : 16, kStep = 16;
  static_assert(std::is_same<T, float>::value, "16-bit rows take the tiles");
  extern __shared__ __align__(128) unsigned char few_smem[];
  float4 *const sums = reinterpret_cast<float4 *>(few_smem);  // [warps][tiles][32]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, j = lane & 3;
  const int part = warp % a.split, row0 = warp / a.split * (8 * kSomeTiles);
  const int steps = (a.features + kStep - 1) / kStep, groups = (a.outputs + kOutputs - 1) / kOutputs;
  after_previous_kernel();
  typename Epilogue::template State<1> state;
  epilogue.begin(state);
  for (int group = (int)blockIdx.x; group < groups; group += (int)gridDim.x) {
    const int o = group * kOutputs + g;
    const T *row_a = a.w[0] + (int64_t)min(o, a.outputs - 1) * a.features;
    const T *row_b = kPair ? a.w[1] + (int64_t)min(o, a.outputs - 1) * a.features : a.w[0] + (int64_t)min(o + 8, a.outputs - 1) * a.features;
    float c[kSomeTiles][4];
#pragma unroll
    for (int n = 0; n < kSomeTiles; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[n][i] = 0.0f;
    for (int s = part; s < steps; s += a.split) {
      const int k = s * kStep + j * 4;
      const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
      const bool there = k < a.features;
      const uint4 qa = there ? load_plain(reinterpret_cast<const uint4 *>(row_a + k)) : zero, qb = there ? load_plain(reinterpret_cast<const uint4 *>(row_b + k)) : zero;
      uint4 q[kSomeTiles];
#pragma unroll
      for (int n = 0; n < kSomeTiles; ++n) {
        const int r = row0 + 8 * n + g;
        q[n] = there && r < a.rows ? load_plain(reinterpret_cast<const uint4 *>(a.x + (int64_t)r * a.x_stride + k)) : zero;
      }
      const Planes pa = split_four(qa), pb = split_four(qb);
#pragma unroll
      for (int n = 0; n < kSomeTiles; ++n) mma_planes(c[n], pa, pb, split_four(q[n]));
    }
    __syncthreads();  // the sums of the group before have been read
#pragma unroll
    for (int n = 0; n < kSomeTiles; ++n) sums[(warp * kSomeTiles + n) * 32 + lane] = make_float4(c[n][0], c[n][1], c[n][2], c[n][3]);
    __syncthreads();
    if (part < kSomeTiles) {  // this warp: the tile `part` of its rows
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int i = 0; i < a.split; ++i) {
        const float4 t = sums[((warp - part + i) * kSomeTiles + part) * 32 + lane];
        v[0] += t.x, v[1] += t.y, v[2] += t.z, v[3] += t.w;
      }
      epilogue.template values<1>(state, 0, row0 + 8 * part + 2 * j, o, a.outputs, v);
    }
  }
  if (part < kSomeTiles) epilogue.end_alone(state, row0 + 8 * part, lane);
}

// Whether that is the way: more rows than the kernel above takes, and few enough groups of weights that every block has one or two.
template <typename T>
bool some_rows(int64_t rows, int64_t features, int64_t outputs, int64_t x_stride, bool pair, FewPlan *plan) {
  const int64_t groups = (outputs + (pair ? 7 : 15)) / (pair ? 8 : 16);
  if (sizeof(T) != 4 || rows < 1 || rows > 128 || features > 2048 || features % 4 != 0 || x_stride % 4 != 0 || groups > 2 * 148) return false;
  plan->tiles = 0;
  plan->split = rows > 64 ? 8 : 16;
  plan->blocks = (int)std::min<int64_t>(groups, 148);
  return true;
}

template <class Epilogue>
int launch_some(FewArgs<float> a, const Epilogue &e, const FewPlan &plan, cudaStream_t stream) {
  a.split = plan.split;
  constexpr size_t kBytes = sizeof(float4) * 32 * kSomeTiles * kFewWarps;
  return launch_next<some_rows_kernel<float, Epilogue>>(dim3((unsigned)plan.blocks), kFewThreads, kBytes, kBytes, stream, 1, a, e);
}

template <typename T, class Epilogue>
int launch_rows(const FewArgs<T> &a, const Epilogue &e, const FewPlan &plan, cudaStream_t stream) {
  if constexpr (std::is_same<T, float>::value)
    if (plan.tiles == 0) return launch_some(a, e, plan, stream);
  return launch_few(a, e, plan, stream);
}

}  // namespace dense
}  // namespace ht
