// Softmax cross entropy of a linear layer's class scores, with its gradient, without the scores in memory:
//
//     s[n, v] = sum_k x[n, k] w[v, k] + bias[v]        loss[n] = log sum_v exp s[n, v] - s[n, target[n]]
//     g[n, v] = r_n (exp(s[n, v]) / sum_v exp s[n, v] - [v = target[n]])     dx = g w     dw = g^T x     dbias = sum_n g
//
// r_n is the upstream gradient of row n (of a mean: divided by the rows that count); rows whose target is the ignored one
// have loss 0 and no gradient, whatever they hold.
//
// Forward: one tile product whose epilogue keeps, per row and half a tile's columns, the largest score m and
// l = sum exp(s - m) in fp32, and the target's score; a second kernel joins the pieces in a fixed order.  The row's (m, l) are
// what the backward needs besides the inputs.
// Backward: a piece of the classes at a time (so that g of a piece, in the operands' type, stays within a bound), the scores are
// formed again, turned into g in the epilogue, and g enters the two products of ht_dense_products.cu.  That is 8 N V K
// operations for a training step where 6 N V K are needed; keeping the scores would cost 4 N V bytes and their traffic.
// g is rounded to bf16 for bf16: 2^-9 of a term that enters sums, below what rounding the sums themselves costs.  For fp16 it is held as two
// bf16 numbers and for fp32 as three, like x and w beside it (GradKind).
// Measured, 16384 x 1024, 50000 classes in bf16: forward 1092 us (1537 TFLOP/s; tensor pipe 77 %), per piece of 12544 classes the gradient of the
// scores 304 us (1384), dx 289 and dw 285 us; a step takes 5.5 ms where those add up to 4.75, power bounds it.
#include "ht_dense_rows.cuh"

namespace ht {
namespace dense {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Joins two pieces of a softmax: largest score m and l = sum exp(s - m); an empty piece has m = -inf, l = 0.
__device__ __forceinline__ void join(float &m, float &l, float m2, float l2) {
  const float top = fmaxf(m, m2), at = top == -INFINITY ? 0.0f : top;
  l = l * exp2_fast((m - at) * kLog2e) + l2 * exp2_fast((m2 - at) * kLog2e);
  m = top;
}

template <typename T>
struct LossEpilogue {
  static constexpr bool kPair = false;
  struct State {
    float m, l;
    int target;
  };
  int rows, cols;
  const T *bias;
  const int64_t *target;
  float2 *partial;      // [rows][slots], slots = 2 n_blocks
  int slots;
  float *target_score;  // [rows]
  unsigned *ended;      // set to 0 for the kernel that joins the pieces
  __device__ __forceinline__ void begin(State &s, const Where &w, bool) const {
    if (w.m_block == 0 && w.n_block == 0 && w.half == 0 && w.quarter == 0 && w.lane == 0) *ended = 0u;
    s.m = -INFINITY, s.l = 0.0f, s.target = -1;
    if (w.inside) {
      const int64_t t = load_plain(target + w.row);
      if (t >= 0 && t < cols) s.target = (int)t;
    }
  }
  __device__ __forceinline__ void unit(State &s, const Where &w, int col, float (&v)[32]) const {
    const int n = cols - col;
    if (n <= 0) return;
    if (bias != nullptr) {
      float b[32];
      load_columns(bias + col, b, n);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] += b[i];
    }
    if (n < 32) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i >= n) v[i] = -INFINITY;
    }
    const int at = s.target - col;
    if (at >= 0 && at < 32) {
      float score = 0.0f;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i == at) score = v[i];
      target_score[w.row] = score;
    }
    float top = v[0];
#pragma unroll
    for (int i = 1; i < 32; ++i) top = fmaxf(top, v[i]);
    top = fmaxf(top, s.m);
    const float m = top == -INFINITY ? 0.0f : top;  // (every score so far is -inf: their exponentials are 0)
    float sum = 0.0f, sum2 = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      sum += exp2_fast((v[i] - m) * kLog2e);
      sum2 += exp2_fast((v[i + 1] - m) * kLog2e);
    }
    s.l = s.l * exp2_fast((s.m - m) * kLog2e) + (sum + sum2);
    s.m = top;
  }
  __device__ __forceinline__ void end(State &s, const Where &w) const {
    if (w.inside) partial[(size_t)w.row * (size_t)slots + (size_t)(w.n_block * 2 + w.half)] = make_float2(s.m, s.l);
  }
};

// g of one piece of the classes as an operand, and its sums over 32 rows for the bias's gradient.
template <typename T>
struct LossGradEpilogue {
  static constexpr bool kPair = false;
  struct State {
    float m, scale, factor;  // g = exp(s - m) scale - [v = target] factor
    int target;
  };
  int rows, cols, first;  // the piece: classes first .. first + cols - 1
  const T *bias;
  const float2 *stats;
  const int64_t *target;
  int64_t ignore, classes;
  const float *grad;      // of single rows, or null: one for all, which leaves with the sums
  typename GradKind<T>::Operand *g;  // [planes][rows][pitch]
  int pitch;
  size_t plane;
  float *row_sums;  // [row_sum_count][pitch] or null
  __device__ __forceinline__ void begin(State &s, const Where &w, bool) const {
    s.m = s.scale = s.factor = 0.0f, s.target = -1;
    if (!w.inside) return;
    const float2 q = load_plain(stats + w.row);
    const int64_t t = load_plain(target + w.row);
    const bool valid = t >= 0 && t < classes;
    if (t != ignore) s.factor = !valid ? NAN : grad != nullptr ? load_plain(grad + w.row) : 1.0f;
    if (t != ignore && valid) s.target = (int)t;
    s.m = q.x;
    s.scale = s.factor / q.y;
  }
  __device__ __forceinline__ void unit(State &s, const Where &w, int col, float (&v)[32]) const {
    const int n = cols - col;
    if (n <= 0) return;
    if (bias != nullptr) {
      float b[32];
      load_columns(bias + first + col, b, n);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] += b[i];
    }
    const int at = s.target - first - col;
    const bool none = s.factor == 0.0f;  // a row that does not count, or is not there
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float p = exp2_fast((v[i] - s.m) * kLog2e) * s.scale;
      v[i] = none || i >= n ? 0.0f : i == at ? p - s.factor : p;
    }
    if (w.inside) store_operand<T>(g + (size_t)w.row * (size_t)pitch + col, plane, v);
    if (row_sums != nullptr) row_sums[(size_t)(w.m_block * 4 + w.quarter) * (size_t)pitch + col + w.lane] = sum_rows(v, w.lane);
  }
  __device__ __forceinline__ void end(State &, const Where &) const {}
};

// The same for few rows: a lane's scores are those of two rows a tile of 8.
template <typename T>
struct FewLossEpilogue {
  static constexpr bool kPair = false;
  template <int NT>
  struct State {
    float m[NT][2], l[NT][2];
  };
  int rows, slots;
  const T *bias;
  const int64_t *target;
  float2 *partial;
  float *target_score;
  unsigned *ended;
  template <typename S>
  __device__ __forceinline__ void begin(S &s) const {
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *ended = 0u;
    for (auto &m : s.m) m[0] = m[1] = -INFINITY;
    for (auto &l : s.l) l[0] = l[1] = 0.0f;
  }
  template <int NT>
  __device__ __forceinline__ void values(State<NT> &s, int n, int row, int o, int outputs, const float (&c)[4]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (row + i >= rows) continue;
      const int64_t t = load_plain(target + row + i);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = o + 8 * h;
        if (at >= outputs) continue;
        const float v = c[2 * h + i] + (bias != nullptr ? to_float(bias[at]) : 0.0f);
        if (t == at) target_score[row + i] = v;
        const float top = fmaxf(s.m[n][i], v), m = top == -INFINITY ? 0.0f : top;
        s.l[n][i] = s.l[n][i] * exp2_fast((s.m[n][i] - m) * kLog2e) + exp2_fast((v - m) * kLog2e);
        s.m[n][i] = top;
      }
    }
  }
  // rows that no other warp has
  __device__ __forceinline__ void end_alone(State<1> &s, int row0, int lane) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        const float m = __shfl_xor_sync(0xffffffffu, s.m[0][i], d), l = __shfl_xor_sync(0xffffffffu, s.l[0][i], d);
        join(s.m[0][i], s.l[0][i], m, l);
      }
      const int row = row0 + 2 * lane + i;
      if (lane < 4 && row < rows) partial[(size_t)row * (size_t)slots + blockIdx.x] = make_float2(s.m[0][i], s.l[0][i]);
    }
  }
  template <int NT>
  __device__ __forceinline__ void end(State<NT> &s, int row0, int lane) const {
    // the lanes with the same rows, then (each warp has its own outputs) the warps: a block's scores are one piece
    __shared__ float2 pieces[kFewWarps][8 * NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          const float m = __shfl_xor_sync(0xffffffffu, s.m[n][i], d), l = __shfl_xor_sync(0xffffffffu, s.l[n][i], d);
          join(s.m[n][i], s.l[n][i], m, l);
        }
        if (lane < 4) pieces[threadIdx.x >> 5][8 * n + 2 * lane + i] = make_float2(s.m[n][i], s.l[n][i]);
      }
    __syncthreads();
    if (threadIdx.x >= 8 * NT || row0 + (int)threadIdx.x >= rows) return;
    float2 all = pieces[0][threadIdx.x];
    for (int i = 1; i < kFewWarps; ++i) join(all.x, all.y, pieces[i][threadIdx.x].x, pieces[i][threadIdx.x].y);
    partial[(size_t)(row0 + (int)threadIdx.x) * (size_t)slots + blockIdx.x] = all;
  }
};

// Joins the pieces of every row, a warp each, in a fixed order: stats[row] = (m, l), the row's loss to `loss`.  A row whose target is
// no class: loss NaN and a flag.  For a sum or mean every block adds its rows' losses in fp64, and the last one to end the blocks' sums,
// in an order that depends on the number of rows alone; it leaves the number of rows that count behind the statistics.  Reads 8 bytes a
// row and piece: 8192 rows of 172 pieces 8 us, latency of a few loads in a row.
struct JoinArgs {
  const float2 *partial;
  int slots;
  const float *target_score;
  const int64_t *target;
  int64_t ignore, rows, classes;
  float2 *stats;
  float *row_loss, *total;  // one of them, the other null: single rows, or their sum or mean
  bool mean;
  double2 *block_sums;  // [blocks]: sum of losses, rows that count
  unsigned *ended;      // blocks that have, 0 at the start
  uint32_t *status_word;
};
__global__ void __launch_bounds__(256) join_rows_kernel(const JoinArgs a) {
  after_previous_kernel();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  float result = 0.0f;
  bool counts = false;
  if (row < a.rows) {
    float m = -INFINITY, l = 0.0f;
    const float2 *pieces = a.partial + (size_t)row * (size_t)a.slots;
    const int64_t t = load_plain(a.target + row);
    const float score = load_plain(a.target_score + row);  // (nothing of use where the row has no target)
#pragma unroll 4
    for (int s = lane; s < a.slots; s += 32) {
      const float2 q = load_plain(pieces + s);
      join(m, l, q.x, q.y);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, d), l2 = __shfl_xor_sync(0xffffffffu, l, d);
      join(m, l, m2, l2);
    }
    counts = t != a.ignore;
    const bool valid = t >= 0 && t < a.classes;
    if (counts) result = valid ? (float)((double)logf(l) + ((double)m - (double)score)) : NAN;
    if (lane == 0) {
      if (a.stats != nullptr) a.stats[row] = make_float2(m, l);
      if (a.row_loss != nullptr) a.row_loss[row] = result;
      if (counts && !valid && a.status_word != nullptr) atomicOr(a.status_word, HT_FLAG_TARGET_RANGE);
    }
  }
  if (a.total == nullptr) return;
  __shared__ double2 sums[8];
  __shared__ bool last;
  if (lane == 0) sums[threadIdx.x >> 5] = make_double2((double)result, counts ? 1.0 : 0.0);
  __syncthreads();
  if (threadIdx.x == 0) {
    double2 sum = sums[0];
    for (int i = 1; i < 8; ++i) sum.x += sums[i].x, sum.y += sums[i].y;
    a.block_sums[blockIdx.x] = sum;
    __threadfence();  // the block's sum, before it counts as ended
    last = atomicAdd(a.ended, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double2 sum = make_double2(0.0, 0.0);
#pragma unroll 4
  for (unsigned i = threadIdx.x; i < gridDim.x; i += 256) {
    const double2 q = __ldcg(a.block_sums + i);
    sum.x += q.x, sum.y += q.y;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    sum.x += __shfl_xor_sync(0xffffffffu, sum.x, d);
    sum.y += __shfl_xor_sync(0xffffffffu, sum.y, d);
  }
  if (lane == 0) sums[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) sum.x += sums[i].x, sum.y += sums[i].y;
    a.total[0] = (float)(a.mean ? sum.x / sum.y : sum.x);
    if (a.stats != nullptr) a.stats[a.rows].x = (float)sum.y;
  }
}

constexpr int64_t kPieceBytes = (int64_t)1 << 29;  // g of one piece, unless the caller sets less

int screen(const ht_dense_problem *p) {
  if (p == nullptr || p->rows < 0 || p->features < 1 || p->outputs < 1 || p->x_stride < p->features) return HT_ERR_INVALID_ARGUMENT;
  if (p->dtype != HT_DTYPE_F32 && p->dtype != HT_DTYPE_BF16 && p->dtype != HT_DTYPE_F16) return HT_ERR_INVALID_ARGUMENT;
  if (p->rows > 0x7fffff00 || p->features > 0x3fffff00 || p->outputs > 0x3fffff00) return HT_ERR_UNSUPPORTED;
  return HT_OK;
}

// The copies that a forward leaves for its backward: of what cannot be read as it is, with the rows that do not count as zeros.
template <typename T>
size_t keep(const ht_dense_problem &p, const T *xp, const T *wp, const int64_t *target, int64_t ignore, void *kept, Operand<T> &x, Operand<T> &w) {
  Arena arena(kept);
  const bool copied = !Operand<T>::direct(p.x_stride);
  x.set(arena, xp, p.rows, p.features, p.x_stride, copied, copied ? target : nullptr, ignore);
  w.set(arena, wp, p.outputs, p.features, p.features);
  return arena.used;
}

template <typename T>
struct ForwardPlan {
  bool few;
  FewPlan few_plan;
  Operand<T> x, w;
  TileShape shape;
  int slots;
  float2 *partial;
  float *target_score;
  double2 *block_sums;
  unsigned *ended;
  size_t bytes;
  ForwardPlan(const ht_dense_problem &p, const T *xp, const T *wp, const int64_t *target, int64_t ignore, void *kept, void *ws) {
    Arena arena(ws);
    few = few_rows<T>(p.rows, p.features, p.outputs, false, &few_plan) ||
          some_rows<T>(p.rows, p.features, p.outputs, p.x_stride, false, &few_plan);
    if (kept != nullptr) {
      keep(p, xp, wp, target, ignore, kept, x, w);
    } else if (!few) {
      x.set(arena, xp, p.rows, p.features, p.x_stride);
      w.set(arena, wp, p.outputs, p.features, p.features);
    }
    shape = tile_shape(p.rows, p.outputs, p.features, Kind<T>::kPlanes, false);
    slots = few ? few_plan.blocks : (int)(2 * ((p.outputs + shape.bn - 1) / shape.bn));
    partial = arena.take<float2>((int64_t)slots * p.rows);
    target_score = arena.take<float>(p.rows);
    block_sums = arena.take<double2>(p.rows / 8 + 1);
    ended = arena.take<unsigned>(1);
    bytes = arena.used;
  }
};

template <typename T>
int forward(const ht_dense_problem &p, const void *x, const void *w, const void *bias, const int64_t *target, int64_t ignore, int reduction,
            float *loss, float *stats, void *kept, void *ws, size_t ws_bytes, uint32_t *status_word, cudaStream_t stream) {
  ForwardPlan<T> plan(p, static_cast<const T *>(x), static_cast<const T *>(w), target, ignore, kept, ws);
  if (plan.bytes > ws_bytes || (plan.bytes > 0 && ws == nullptr)) return HT_ERR_WORKSPACE;
  int sms = 0, rc;
  if (p.rows > 0) {
    // (copies that are left for the backward are made whichever kernel runs)
    if (kept != nullptr || !plan.few) HT_TRY(lay_out<T>(stream, plan.x, plan.w));
    if (plan.few) {
      const FewArgs<T> a = {static_cast<const T *>(x), {static_cast<const T *>(w), nullptr}, p.x_stride, (int)p.rows, (int)p.features, (int)p.outputs};
      const FewLossEpilogue<T> e = {(int)p.rows, plan.slots, static_cast<const T *>(bias), target, plan.partial, plan.target_score, plan.ended};
      HT_TRY(launch_rows(a, e, plan.few_plan, stream));
    } else {
      if ((rc = sm_count(&sms)) != HT_OK) return rc;
      TileProblem t;
      t.a[0] = plan.x.m;
      t.b[0] = plan.w.m;
      t.rows = p.rows, t.cols = p.outputs, t.k = p.features;
      t.f16 = p.dtype == HT_DTYPE_F16;
      t.status_word = status_word;
      const LossEpilogue<T> e = {(int)p.rows, (int)p.outputs, static_cast<const T *>(bias), target, plan.partial, plan.slots, plan.target_score, plan.ended};
      if ((rc = launch_tiles<Kind<T>::kPlanes, false, false>(t, e, plan.shape, sms, stream)) != HT_OK) return rc;
    }
  }
  // (no rows: a sum of nothing)
  JoinArgs j = {plan.partial, plan.slots, plan.target_score, target, ignore, p.rows, p.outputs, reinterpret_cast<float2 *>(stats), nullptr, nullptr,
                reduction == HT_REDUCTION_MEAN, plan.block_sums, plan.ended, status_word};
  (reduction == HT_REDUCTION_NONE ? j.row_loss : j.total) = loss;
  if (p.rows == 0) HT_CUDA_TRY(cudaMemsetAsync(plan.ended, 0, sizeof(unsigned), stream));
  return launch_next<join_rows_kernel>(dim3((unsigned)std::max<int64_t>((p.rows + 7) / 8, 1)), 256, 0, 0, stream, 1, j);
}

template <typename T>
struct BackwardPlan {
  Operand<T> x, w;         // of the scores
  GradOperand<T> gx, gw;   // of the products that g enters; fp16: copies of their own, of w a piece at a time
  int64_t piece, pitch;  // classes of a piece, elements of a row of g
  typename GradKind<T>::Operand *g;
  float *sum, *parts, *row_sums;
  size_t bytes;
  BackwardPlan(const ht_dense_problem &p, const T *xp, const T *wp, const int64_t *target, int64_t ignore, bool has_dx, bool has_db, const void *kept,
               void *ws) {
    Arena arena(ws);
    if (kept != nullptr) {
      keep(p, xp, wp, target, ignore, const_cast<void *>(kept), x, w);
      x.ready = w.ready = true;
    }
    // (rows that do not count are zeros in the products' copy of x)
    if (kept == nullptr || (kSameOperands<T> && x.copy == nullptr))
      x.set(arena, xp, p.rows, p.features, p.x_stride, kSameOperands<T>, kSameOperands<T> ? target : nullptr, ignore), x.ready = false;
    if (kept == nullptr) w.set(arena, wp, p.outputs, p.features, p.features);
    constexpr int kPlanes = GradKind<T>::kPlanes;
    const int64_t limit = p.scratch_limit > 0 ? std::min(p.scratch_limit, kPieceBytes) : kPieceBytes;
    const int64_t per_class = std::max<int64_t>(p.rows, 1) * kPlanes * 2;
    piece = piece_of(p.outputs, limit / per_class);
    pitch = round_up(piece, 64);
    if constexpr (!kSameOperands<T>) {
      gx.set(arena, xp, p.rows, p.features, p.x_stride, true, target, ignore);
      if (has_dx) gw.set(arena, wp, piece, p.features, p.features);
    }
    g = arena.take<typename GradKind<T>::Operand>(p.rows * pitch * kPlanes);
    sum = has_dx && piece < p.outputs ? arena.take<float>(p.rows * p.features) : nullptr;
    parts = nullptr;
    int64_t most = piece < p.outputs ? 0 : product_parts(p.rows, p.features, p.outputs, kPlanes);
    for (const int64_t count : {piece, (p.outputs - 1) % piece + 1})
      most = std::max(most, product_parts(count, p.features, std::max<int64_t>(p.rows, 1), kPlanes));
    if (most > 0) parts = arena.take<float>(most);
    row_sums = has_db ? arena.take<float>(row_sum_count(p.rows, {2, 0}) * pitch) : nullptr;
    bytes = arena.used;
  }
};

template <typename T>
int backward(const ht_dense_problem &p, const void *x, const void *w, const void *bias, const int64_t *target, int64_t ignore, int reduction,
             const float *grad, const float *stats, const void *kept, void *dx_, void *dw_, void *db_, void *ws, size_t ws_bytes, uint32_t *status_word,
             cudaStream_t stream) {
  T *dx = static_cast<T *>(dx_), *dw = static_cast<T *>(dw_), *db = static_cast<T *>(db_);
  BackwardPlan<T> plan(p, static_cast<const T *>(x), static_cast<const T *>(w), target, ignore, dx != nullptr, db != nullptr, kept, ws);
  if (plan.bytes > ws_bytes || (plan.bytes > 0 && ws == nullptr)) return HT_ERR_WORKSPACE;
  if (p.rows == 0) {
    if (dw != nullptr) HT_CUDA_TRY(cudaMemsetAsync(dw, 0, sizeof(T) * (size_t)(p.outputs * p.features), stream));
    if (db != nullptr) HT_CUDA_TRY(cudaMemsetAsync(db, 0, sizeof(T) * (size_t)p.outputs, stream));
    return HT_OK;
  }
  int sms = 0, rc;
  if ((rc = sm_count(&sms)) != HT_OK) return rc;
  Scale scale;
  if (reduction != HT_REDUCTION_NONE) scale.number = grad;
  if (reduction == HT_REDUCTION_MEAN) scale.count = stats + 2 * p.rows;
  constexpr int kPlanes = GradKind<T>::kPlanes;
  for (int64_t first = 0; first < p.outputs; first += plan.piece) {
    const int64_t count = std::min(plan.piece, p.outputs - first);
    LayOut<T> copies = {};
    if constexpr (!kSameOperands<T>) plan.gx.from(plan.x, 0, p.rows), plan.gw.from(plan.w, first, count);
    if (first == 0) copies.add(plan.x), copies.add(plan.w), copies.add(plan.gx);
    copies.add(plan.gw);
    HT_TRY(lay_out<T>(copies, stream));
    TileProblem t;
    t.f16 = p.dtype == HT_DTYPE_F16;
    t.status_word = status_word;
    t.a[0] = plan.x.m;
    t.b[0] = plan.w.m;
    t.rows = p.rows, t.cols = count, t.k = p.features, t.b_n0 = first;
    LossGradEpilogue<T> e = {};
    e.rows = (int)p.rows, e.cols = (int)count, e.first = (int)first;
    e.bias = static_cast<const T *>(bias);
    e.stats = reinterpret_cast<const float2 *>(stats);
    e.target = target, e.ignore = ignore, e.classes = p.outputs;
    e.grad = reduction == HT_REDUCTION_NONE ? grad : nullptr;
    e.g = plan.g, e.pitch = (int)plan.pitch, e.plane = (size_t)(p.rows * plan.pitch);
    e.row_sums = plan.row_sums;
    const TileShape shape = tile_shape(p.rows, count, p.features, Kind<T>::kPlanes, false);
    if ((rc = launch_tiles<Kind<T>::kPlanes, false, false>(t, e, shape, sms, stream)) != HT_OK) return rc;
    Matrix g;
    g.data = plan.g, g.rows = p.rows, g.cols = count, g.pitch = plan.pitch, g.planes = kPlanes, g.plane = p.rows * plan.pitch;
    StoreEpilogue<T> store = {};
    store.scale = scale;
    store.cols = (int)p.features;
    store.split = 0x7fffffff;
    store.sum_align = row_alignment(plan.sum, p.features * (int64_t)sizeof(float));
    if (dx != nullptr) {
      TileProblem q = t;
      q.f16 = false;
      q.a[0] = g;
      q.rows = p.rows, q.cols = p.features, q.k = count, q.b_n0 = 0, q.b_k0 = kSameOperands<T> ? first : 0;
      if (!kSameOperands<T>) q.b[0] = plan.gw.m;
      store.rows = store.part = (int)p.rows;
      store.out = dx, store.align = row_alignment(dx, p.features * (int64_t)sizeof(T));
      store.sum = plan.sum, store.begins = first == 0, store.keep = first + count < p.outputs;
      if ((rc = product_dx<T>(q, store, plan.piece < p.outputs ? nullptr : plan.parts, sms, stream)) != HT_OK) return rc;
    }
    if (dw != nullptr) {
      TileProblem q = t;
      q.f16 = false;
      q.a[0] = g;
      q.b[0] = kSameOperands<T> ? plan.x.m : plan.gx.m;
      q.rows = count, q.cols = p.features, q.k = p.rows, q.b_n0 = 0;
      store.rows = store.part = (int)count;
      store.out = dw + (size_t)first * (size_t)p.features, store.align = row_alignment(store.out, p.features * (int64_t)sizeof(T));
      store.sum = nullptr, store.keep = false;
      if ((rc = product_dw<T>(q, store, plan.parts, sms, stream)) != HT_OK) return rc;
    }
    if (db != nullptr)
      HT_TRY(column_sums<T>(plan.row_sums, row_sum_count(p.rows, shape), plan.pitch, count, store.scale, db + first, nullptr, plan.pitch, stream));
  }
  return HT_OK;
}

template <typename F>
auto by_type(int dtype, F &&f) {
  return dtype == HT_DTYPE_F32 ? f(float()) : dtype == HT_DTYPE_BF16 ? f(__nv_bfloat16()) : f(__half());
}

}  // namespace
}  // namespace dense
}  // namespace ht

using namespace ht;
using namespace ht::dense;

extern "C" size_t ht_linear_class_loss_workspace_bytes(const ht_dense_problem *p, int backward) {
  if (screen(p) != HT_OK) return 0;
  return by_type(p->dtype, [&](auto zero) -> size_t {
    typedef decltype(zero) T;
    return backward != 0 ? BackwardPlan<T>(*p, nullptr, nullptr, nullptr, 0, true, true, nullptr, nullptr).bytes
                         : ForwardPlan<T>(*p, nullptr, nullptr, nullptr, 0, nullptr, nullptr).bytes;
  });
}

extern "C" size_t ht_linear_class_loss_kept_bytes(const ht_dense_problem *p) {
  if (screen(p) != HT_OK || p->rows == 0) return 0;
  return by_type(p->dtype, [&](auto zero) -> size_t {
    typedef decltype(zero) T;
    Operand<T> x, w;
    return keep<T>(*p, nullptr, nullptr, nullptr, 0, nullptr, x, w);
  });
}

extern "C" int ht_linear_class_loss_forward(const ht_dense_problem *p, const void *x, const void *w, const void *bias, const int64_t *target,
                                            int64_t ignore_index, int reduction, float *loss, float *stats, void *kept, void *workspace,
                                            size_t workspace_bytes, uint32_t *status_word, ht_stream_t stream) {
  int rc = screen(p);
  if (rc != HT_OK) return rc;
  if (reduction != HT_REDUCTION_NONE && reduction != HT_REDUCTION_MEAN && reduction != HT_REDUCTION_SUM) return HT_ERR_INVALID_ARGUMENT;
  if (p->rows == 0 && reduction == HT_REDUCTION_NONE) return HT_OK;
  if (loss == nullptr || (p->rows > 0 && (x == nullptr || w == nullptr || target == nullptr))) return HT_ERR_INVALID_ARGUMENT;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(stats) |
        reinterpret_cast<uintptr_t>(kept)) & 15u) != 0)
    return HT_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return HT_ERR_WORKSPACE;
  return by_type(p->dtype, [&](auto zero) -> int {
    return forward<decltype(zero)>(*p, x, w, bias, target, ignore_index, reduction, loss, stats, kept, workspace, workspace_bytes, status_word,
                                   reinterpret_cast<cudaStream_t>(stream));
  });
}

extern "C" int ht_linear_class_loss_backward(const ht_dense_problem *p, const void *x, const void *w, const void *bias, const int64_t *target,
                                             int64_t ignore_index, int reduction, const float *grad, const float *stats, const void *kept, void *dx, void *dw,
                                             void *dbias, void *workspace, size_t workspace_bytes, uint32_t *status_word, ht_stream_t stream) {
  int rc = screen(p);
  if (rc != HT_OK) return rc;
  if (reduction != HT_REDUCTION_NONE && reduction != HT_REDUCTION_MEAN && reduction != HT_REDUCTION_SUM) return HT_ERR_INVALID_ARGUMENT;
  if (p->rows > 0 && (x == nullptr || w == nullptr || target == nullptr || grad == nullptr || stats == nullptr)) return HT_ERR_INVALID_ARGUMENT;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(stats) |
        reinterpret_cast<uintptr_t>(kept) | reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(dw)) & 15u) != 0)
    return HT_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return HT_ERR_WORKSPACE;
  return by_type(p->dtype, [&](auto zero) -> int {
    return backward<decltype(zero)>(*p, x, w, bias, target, ignore_index, reduction, grad, stats, kept, dx, dw, dbias, workspace, workspace_bytes,
                                    status_word, reinterpret_cast<cudaStream_t>(stream));
  });
}
