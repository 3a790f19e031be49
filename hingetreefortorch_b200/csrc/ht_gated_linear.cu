// A gated projection in front of a forest: both projections, the activation and the product in one kernel, and its gradient.
//
//     a = x wg^T + bg      u = x wv^T + bv      h = act(a) u
//     da = dh u act'(a)    du = dh act(a)       dx = da wg + du wv     dwg = da^T x     dwv = du^T x     dbg, dbv: column sums
//
// Forward: one tile product over the rows of both weights side by side, 64 or 128 columns of each; the epilogue has the two products
// of an element in one thread and writes h alone.
// Backward: of the forward nothing is kept but copies of operands that cannot be read as they are.  The projections are formed again, the
// epilogue reads dh and writes da and du in the operands' type, and those enter the products of ht_dense_products.cu: dx as one sum over
// both, dwg and dwv as one product.  16 N K H operations for a training step where 12 N K H are needed; keeping a and u in fp32, which
// the gradient's accuracy asks for, would cost 8 N H bytes and 16 N H of traffic.  da and du are rounded to bf16 for bf16 (2^-9 of a term that
// enters sums); for fp16 they are held as two bf16 numbers and for fp32 as three, like x and the weights beside them (GradKind).
// Measured, 8192 x 784 to 12700 in bf16: forward 262 us (1245 TFLOP/s, tensor pipe 66 %: power and clock), projections again with da and du
// 318 us (1027, 54 %: 208 MB of dh in and 416 MB out beside the products), dx 274 and both weights 282 us; 4096 x 784 to 2048 in fp32: 120,
// 174, 129 and 129 us.
#include "ht_dense_rows.cuh"

namespace ht {
namespace dense {
namespace {

// The activation g and its derivative d at a.  EXACT: fp32 results; otherwise what is rounded to 16 bits afterwards.
template <bool EXACT>
__device__ __forceinline__ float sigmoid(float a) {
  return __fdividef(1.0f, 1.0f + (EXACT ? expf(-a) : __expf(-a)));  // (a quotient of 2 ulp)
}
template <bool EXACT, bool SLOPE>
__device__ __forceinline__ float activate_one(int act, float a, float &slope) {
  if (act == HT_ACTIVATION_SILU) {
    const float s = sigmoid<EXACT>(a);
    if (SLOPE) slope = s * (1.0f + a * (1.0f - s));
    return a * s;
  }
  if (act == HT_ACTIVATION_SIGMOID) {
    const float s = sigmoid<EXACT>(a);
    if (SLOPE) slope = s * (1.0f - s);
    return s;
  }
  if (act == HT_ACTIVATION_GELU) {  // with the normal distribution function
    float phi, e;
    if (EXACT) {
      phi = 0.5f * erfcf(a * -0.70710678118654752f);
      e = SLOPE ? expf(-0.5f * a * a) : 0.0f;
    } else {
      // erfc(z) = exp(-z^2) t P(t), t = 1 / (1 + 0.425 z), the form of 7.1.26 in Abramowitz and Stegun, Handbook of Mathematical Functions; here P is
      // fitted to the least relative error over z in [0, 10], 8e-6, so that the tail is as exact as the rest (7.1.26 itself is off by 1.5e-7 of 1,
      // 0.16 % of the tail at -5).  The exponential is the slope's too.
      const float z = fabsf(a) * 0.70710678118654752f, t = __fdividef(1.0f, fmaf(0.425f, z, 1.0f));
      e = __expf(-0.5f * a * a);
      const float tail =
          0.5f * e * t *
          fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.153831834f, 0.427965646f), -0.0298281749f), 0.286887415f), 0.228281937f), 0.240533059f);
      phi = a < 0.0f ? tail : 1.0f - tail;
    }
    if (SLOPE) slope = fmaf(a * 0.39894228040143268f, e, phi);
    return a * phi;
  }
  if (SLOPE) slope = a > 0.0f ? 1.0f : 0.0f;
  return a < 0.0f ? 0.0f : a;  // (no number stays none)
}
template <bool EXACT, bool SLOPE>
__device__ __forceinline__ void activate(int act, const float (&a)[32], float (&g)[32], float (&d)[32]) {
  auto all = [&](int which) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      float slope = 0.0f;
      g[i] = activate_one<EXACT, SLOPE>(which, a[i], slope);
      if (SLOPE) d[i] = slope;
    }
  };
  if (act == HT_ACTIVATION_SILU)
    all(HT_ACTIVATION_SILU);
  else if (act == HT_ACTIVATION_GELU)
    all(HT_ACTIVATION_GELU);
  else if (act == HT_ACTIVATION_RELU)
    all(HT_ACTIVATION_RELU);
  else
    all(HT_ACTIVATION_SIGMOID);
}

template <typename T>
__device__ __forceinline__ void add_bias(const T *bias, int col, int n, float (&v)[32]) {
  if (bias == nullptr) return;
  float b[32];
  load_columns(bias + col, b, n);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] += b[i];
}

template <typename T>
struct GatedEpilogue {
  static constexpr bool kPair = true;
  static constexpr bool kExact = sizeof(T) == 4;
  struct State {};
  int rows, cols, act;
  const T *bg, *bv;
  T *h;  // [rows, cols]
  int align;
  __device__ __forceinline__ void begin(State &, const Where &, bool) const {}
  __device__ __forceinline__ void unit(State &, const Where &w, int col, float (&a)[32], float (&u)[32]) const {
    const int n = cols - col;
    if (n <= 0) return;
    add_bias(bg, col, n, a);
    add_bias(bv, col, n, u);
    float g[32];
    activate<kExact, false>(act, a, g, g);
#pragma unroll
    for (int i = 0; i < 32; ++i) g[i] *= u[i];
    const int top = w.row - w.lane;
    if (top < rows) store_box(w, h + (size_t)top * (size_t)cols + col, (size_t)cols, min(32, rows - top), min(32, n), align, g);
  }
  __device__ __forceinline__ void end(State &, const Where &) const {}
};

template <typename T>
struct FewGatedEpilogue {
  static constexpr bool kPair = true;
  template <int NT>
  struct State {};
  int rows, cols, act;
  const T *bg, *bv;
  T *h;
  template <typename S>
  __device__ __forceinline__ void begin(S &) const {}
  template <int NT>
  __device__ __forceinline__ void values(State<NT> &, int, int row, int o, int outputs, const float (&c)[4]) const {
    if (o >= outputs) return;
    const float ba = bg != nullptr ? to_float(bg[o]) : 0.0f, bu = bv != nullptr ? to_float(bv[o]) : 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float slope;
      if (row + i < rows) h[(size_t)(row + i) * (size_t)cols + o] = from_float<T>(activate_one<sizeof(T) == 4, false>(act, c[i] + ba, slope) * (c[2 + i] + bu));
    }
  }
  __device__ __forceinline__ void end_alone(State<1> &, int, int) const {}
  template <int NT>
  __device__ __forceinline__ void end(State<NT> &, int, int) const {}
};

// da and du of a piece of the outputs, side by side in one operand, and their sums over 32 rows for the biases' gradients.
template <typename T>
struct GatedGradEpilogue {
  static constexpr bool kPair = true;
  static constexpr bool kExact = sizeof(T) == 4;
  static constexpr int kBoxes = (int)kBoxBytes / (1024 * (int)sizeof(T));  // of dh that a warp's shared memory holds
  struct State {
    int unit;
  };
  int rows, cols, act, first, outputs;  // the piece: outputs first .. first + cols - 1
  const T *bg, *bv;
  const T *dh;          // [rows, outputs]
  int align;
  typename GradKind<T>::Operand *g;  // [planes][rows][2 pitch]: da, then du
  int pitch;
  size_t plane;
  float *row_sums;  // [row_sum_count][2 pitch] or null
  __device__ __forceinline__ void fetch(const Where &w, int slot, int row, int col) const {
    const int r = row - w.lane;
    const bool some = r < rows && col < cols;
    begin_box(w.box + (uint32_t)slot * 1024u * (uint32_t)sizeof(T), dh + (some ? (size_t)r * (size_t)outputs + first + col : 0), (size_t)outputs,
              some ? min(32, rows - r) : 0, min(32, cols - col), align, w.lane);
  }
  __device__ __forceinline__ void begin(State &s, const Where &w, bool first_tile) const {
    s.unit = 0;
    if (first_tile)  // later ones have been fetched under the tile before
      for (int i = 0; i < min(kBoxes, w.units); ++i) fetch(w, i, w.row, w.col + 32 * i);
  }
  __device__ __forceinline__ void unit(State &s, const Where &w, int col, float (&a)[32], float (&u)[32]) const {
    const int n = cols - col;
    float dh_[32];
    const int r = w.row - w.lane, boxes = min(kBoxes, w.units), slot = s.unit % kBoxes;
    finish_box(w.box + (uint32_t)slot * 1024u * (uint32_t)sizeof(T), dh + (r < rows ? (size_t)r * (size_t)outputs + first + col : 0), (size_t)outputs,
               r < rows ? min(32, rows - r) : 0, min(32, n), align, w.lane, boxes == 1, dh_);
    // its place is free for the unit `boxes` further on, of this tile or the next
    const int then = s.unit + boxes;
    if (then < w.units)
      fetch(w, slot, w.row, w.col + 32 * then);
    else
      fetch(w, slot, w.next_row, w.next_col + 32 * (then - w.units));
    ++s.unit;
    if (n <= 0) return;
    add_bias(bg, first + col, n, a);
    add_bias(bv, first + col, n, u);
    float act_a[32], slope[32];
    activate<kExact, true>(act, a, act_a, slope);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float d = dh_[i];
      a[i] = w.inside && i < n ? d * u[i] * slope[i] : 0.0f;
      u[i] = w.inside && i < n ? d * act_a[i] : 0.0f;
    }
    typename GradKind<T>::Operand *to = g + (size_t)w.row * (size_t)(2 * pitch) + col;
    if (w.inside) {
      store_operand<T>(to, plane, a);
      store_operand<T>(to + pitch, plane, u);
    }
    if (row_sums != nullptr) {
      float *sums = row_sums + (size_t)(w.m_block * 4 + w.quarter) * (size_t)(2 * pitch) + col + w.lane;
      sums[0] = sum_rows(a, w.lane);
      sums[pitch] = sum_rows(u, w.lane);
    }
  }
  __device__ __forceinline__ void end(State &, const Where &) const {}
};

constexpr int64_t kPieceBytes = (int64_t)1 << 29;  // da and du of one piece, unless the caller sets less

int screen(const ht_dense_problem *p) {
  if (p == nullptr || p->rows < 0 || p->features < 1 || p->outputs < 1 || p->x_stride < p->features) return HT_ERR_INVALID_ARGUMENT;
  if (p->dtype != HT_DTYPE_F32 && p->dtype != HT_DTYPE_BF16 && p->dtype != HT_DTYPE_F16) return HT_ERR_INVALID_ARGUMENT;
  if (p->activation < HT_ACTIVATION_SILU || p->activation > HT_ACTIVATION_SIGMOID) return HT_ERR_INVALID_ARGUMENT;
  if (p->rows > 0x7fffff00 || p->features > 0x3fffff00 || p->outputs > 0x3fffff00) return HT_ERR_UNSUPPORTED;
  return HT_OK;
}

template <typename T>
struct Plan {
  bool few = false;  // the forward
  FewPlan few_plan;
  Operand<T> x, wg, wv;         // of the projections
  GradOperand<T> gx, gwg, gwv;  // of the products that da and du enter; fp16: copies of their own, of the weights a piece at a time
  int64_t piece = 0, pitch = 0;
  typename GradKind<T>::Operand *g = nullptr;
  float *sum = nullptr, *parts = nullptr, *row_sums = nullptr;
  size_t bytes = 0, kept_bytes = 0;
  Plan(const ht_dense_problem &p, const void *xp, const void *wgp, const void *wvp, bool backward, bool has_dx, bool has_bias, bool keeps, void *kept,
       void *ws) {
    Arena arena(ws);
    few = !backward && (few_rows<T>(p.rows, p.features, p.outputs, true, &few_plan) ||
                        some_rows<T>(p.rows, p.features, p.outputs, p.x_stride, true, &few_plan));
    // the copies of what cannot be read as it is: made by the forward for both where they are kept
    Arena keeping(kept);
    Arena &copies = keeps ? keeping : arena;
    if (!few || keeps) {
      x.set(copies, static_cast<const T *>(xp), p.rows, p.features, p.x_stride);
      wg.set(copies, static_cast<const T *>(wgp), p.outputs, p.features, p.features);
      wv.set(copies, static_cast<const T *>(wvp), p.outputs, p.features, p.features);
      x.ready = wg.ready = wv.ready = backward && keeps;
    }
    kept_bytes = keeping.used;
    bytes = arena.used;
    if (few) return;
    if (backward) {
      const int64_t limit = p.scratch_limit > 0 ? std::min(p.scratch_limit, kPieceBytes) : kPieceBytes;
      constexpr int kPlanes = GradKind<T>::kPlanes;
      const int64_t per_output = std::max<int64_t>(p.rows, 1) * kPlanes * 4;
      piece = piece_of(p.outputs, limit / per_output);
      pitch = round_up(piece, 64);
      if constexpr (!kSameOperands<T>) {
        gx.set(arena, static_cast<const T *>(xp), p.rows, p.features, p.x_stride);
        if (has_dx) gwg.set(arena, static_cast<const T *>(wgp), piece, p.features, p.features);
        if (has_dx) gwv.set(arena, static_cast<const T *>(wvp), piece, p.features, p.features);
      }
      g = arena.template take<typename GradKind<T>::Operand>(p.rows * 2 * pitch * kPlanes);
      sum = has_dx && piece < p.outputs ? arena.take<float>(p.rows * p.features) : nullptr;
      int64_t most = piece < p.outputs ? 0 : product_parts(p.rows, p.features, 2 * p.outputs, kPlanes);
      for (const int64_t count : {piece, (p.outputs - 1) % piece + 1})
        for (const int64_t height : {count, pitch + count})  // one weight's gradient, both
          most = std::max(most, product_parts(height, p.features, std::max<int64_t>(p.rows, 1), kPlanes));
      if (most > 0) parts = arena.take<float>(most);
      row_sums = has_bias ? arena.take<float>(row_sum_count(p.rows, {2, 0}) * 2 * pitch) : nullptr;
    }
    bytes = arena.used;
  }
};

template <typename T>
int forward(const ht_dense_problem &p, const void *x, const void *wg, const void *wv, const void *bg, const void *bv, void *h, void *kept, void *ws,
            size_t ws_bytes, uint32_t *status_word, cudaStream_t stream) {
  Plan<T> plan(p, x, wg, wv, false, false, false, kept != nullptr, kept, ws);
  if (plan.bytes > ws_bytes || (plan.bytes > 0 && ws == nullptr)) return HT_ERR_WORKSPACE;
  int sms = 0, rc;
  HT_TRY(lay_out<T>(stream, plan.x, plan.wg, plan.wv));
  if (plan.few) {
    const FewArgs<T> a = {static_cast<const T *>(x), {static_cast<const T *>(wg), static_cast<const T *>(wv)}, p.x_stride, (int)p.rows, (int)p.features,
                          (int)p.outputs};
    const FewGatedEpilogue<T> e = {(int)p.rows, (int)p.outputs, p.activation, static_cast<const T *>(bg), static_cast<const T *>(bv), static_cast<T *>(h)};
    return launch_rows(a, e, plan.few_plan, stream);
  }
  if ((rc = sm_count(&sms)) != HT_OK) return rc;
  TileProblem t;
  t.a[0] = plan.x.m;
  t.b[0] = plan.wg.m;
  t.b[1] = plan.wv.m;
  t.rows = p.rows, t.cols = p.outputs, t.k = p.features;
  t.f16 = p.dtype == HT_DTYPE_F16;
  t.status_word = status_word;
  GatedEpilogue<T> e = {(int)p.rows, (int)p.outputs, p.activation, static_cast<const T *>(bg), static_cast<const T *>(bv), static_cast<T *>(h),
                        row_alignment(h, p.outputs * (int64_t)sizeof(T))};
  return launch_tiles<Kind<T>::kPlanes, false, false>(t, e, tile_shape(p.rows, p.outputs, p.features, Kind<T>::kPlanes, true), sms, stream);
}

struct Gradients {
  void *dx, *dwg, *dwv, *dbg, *dbv;
};

template <typename T>
int backward(const ht_dense_problem &p, const void *x, const void *wg, const void *wv, const void *bg, const void *bv, const void *dh,
             const void *kept, const Gradients &out, void *ws, size_t ws_bytes, uint32_t *status_word, cudaStream_t stream) {
  const bool has_bias = out.dbg != nullptr || out.dbv != nullptr;
  Plan<T> plan(p, x, wg, wv, true, out.dx != nullptr, has_bias, kept != nullptr, const_cast<void *>(kept), ws);
  if (plan.bytes > ws_bytes || (plan.bytes > 0 && ws == nullptr)) return HT_ERR_WORKSPACE;
  T *dwg = static_cast<T *>(out.dwg), *dwv = static_cast<T *>(out.dwv), *dbg = static_cast<T *>(out.dbg), *dbv = static_cast<T *>(out.dbv);
  if (p.rows == 0) {
    for (T *q : {dwg, dwv})
      if (q != nullptr) HT_CUDA_TRY(cudaMemsetAsync(q, 0, sizeof(T) * (size_t)(p.outputs * p.features), stream));
    for (T *q : {dbg, dbv})
      if (q != nullptr) HT_CUDA_TRY(cudaMemsetAsync(q, 0, sizeof(T) * (size_t)p.outputs, stream));
    return HT_OK;
  }
  int sms = 0, rc;
  if ((rc = sm_count(&sms)) != HT_OK) return rc;
  constexpr int kPlanes = GradKind<T>::kPlanes;
  const size_t plane = (size_t)(p.rows * 2 * plan.pitch);
  for (int64_t first = 0; first < p.outputs; first += plan.piece) {
    const int64_t count = std::min(plan.piece, p.outputs - first);
    LayOut<T> copies = {};
    if constexpr (!kSameOperands<T>) plan.gx.from(plan.x, 0, p.rows), plan.gwg.from(plan.wg, first, count), plan.gwv.from(plan.wv, first, count);
    if (first == 0) copies.add(plan.x), copies.add(plan.wg), copies.add(plan.wv), copies.add(plan.gx);
    copies.add(plan.gwg), copies.add(plan.gwv);
    HT_TRY(lay_out<T>(copies, stream));
    TileProblem t;
    t.f16 = p.dtype == HT_DTYPE_F16;
    t.status_word = status_word;
    t.a[0] = plan.x.m;
    t.b[0] = plan.wg.m;
    t.b[1] = plan.wv.m;
    t.rows = p.rows, t.cols = count, t.k = p.features, t.b_n0 = first;
    GatedGradEpilogue<T> e = {};
    e.rows = (int)p.rows, e.cols = (int)count, e.act = p.activation, e.first = (int)first, e.outputs = (int)p.outputs;
    e.bg = static_cast<const T *>(bg), e.bv = static_cast<const T *>(bv), e.dh = static_cast<const T *>(dh);
    e.align = row_alignment(e.dh, p.outputs * (int64_t)sizeof(T));
    e.g = plan.g, e.pitch = (int)plan.pitch, e.plane = plane, e.row_sums = plan.row_sums;
    const TileShape shape = tile_shape(p.rows, count, p.features, Kind<T>::kPlanes, true);
    if ((rc = launch_tiles<Kind<T>::kPlanes, false, false>(t, e, shape, sms, stream)) != HT_OK) return rc;
    StoreEpilogue<T> store = {};
    store.cols = (int)p.features;
    store.split = 0x7fffffff;
    store.sum_align = row_alignment(plan.sum, p.features * (int64_t)sizeof(float));
    Matrix g;
    g.rows = p.rows, g.pitch = 2 * plan.pitch, g.planes = kPlanes, g.plane = (int64_t)plane;
    if (out.dx != nullptr) {
      TileProblem q = t;
      q.f16 = false;
      if (!kSameOperands<T>) q.b[0] = plan.gwg.m, q.b[1] = plan.gwv.m;
      g.cols = count;
      g.data = plan.g, q.a[0] = g;
      g.data = plan.g + plan.pitch, q.a[1] = g;
      q.segments = 2;
      q.rows = p.rows, q.cols = p.features, q.k = count, q.b_n0 = 0, q.b_k0 = kSameOperands<T> ? first : 0;
      store.rows = store.part = (int)p.rows;
      store.out = static_cast<T *>(out.dx), store.align = row_alignment(store.out, p.features * (int64_t)sizeof(T));
      store.sum = plan.sum, store.begins = first == 0, store.keep = first + count < p.outputs;
      if ((rc = product_dx<T>(q, store, plan.piece < p.outputs ? nullptr : plan.parts, sms, stream)) != HT_OK) return rc;
    }
    if (dwg != nullptr || dwv != nullptr) {
      // rows of the product: da's columns, then du's; one of the two weights alone takes its half
      TileProblem q = t;
      q.f16 = false;
      const bool both = dwg != nullptr && dwv != nullptr;
      g.data = dwg != nullptr ? plan.g : plan.g + plan.pitch;
      g.cols = both ? plan.pitch + count : count;
      q.a[0] = g;
      q.b[0] = kSameOperands<T> ? plan.x.m : plan.gx.m;
      q.rows = g.cols, q.cols = p.features, q.k = p.rows, q.b_n0 = 0;
      store.rows = (int)g.cols;
      store.part = (int)count;
      store.split = both ? (int)plan.pitch : 0x7fffffff;
      store.out = (dwg != nullptr ? dwg : dwv) + (size_t)first * (size_t)p.features;
      store.out2 = both ? dwv + (size_t)first * (size_t)p.features : nullptr;
      store.align = std::min(row_alignment(dwg, p.features * (int64_t)sizeof(T)), row_alignment(dwv, p.features * (int64_t)sizeof(T)));
      store.sum = nullptr, store.keep = false;
      if ((rc = product_dw<T>(q, store, plan.parts, sms, stream)) != HT_OK) return rc;
    }
    const int64_t blocks = row_sum_count(p.rows, shape);
    if (has_bias)
      HT_TRY(column_sums<T>(plan.row_sums, blocks, 2 * plan.pitch, count, Scale(), dbg == nullptr ? nullptr : dbg + first, dbv == nullptr ? nullptr : dbv + first,
                            plan.pitch, stream));
  }
  return HT_OK;
}

template <typename F>
auto by_type(int dtype, F &&f) {
  return dtype == HT_DTYPE_F32 ? f(float()) : dtype == HT_DTYPE_BF16 ? f(__nv_bfloat16()) : f(__half());
}

bool aligned(std::initializer_list<const void *> pointers) {
  uintptr_t all = 0;
  for (const void *p : pointers) all |= reinterpret_cast<uintptr_t>(p);
  return (all & 15u) == 0;
}

}  // namespace
}  // namespace dense
}  // namespace ht

using namespace ht;
using namespace ht::dense;

extern "C" size_t ht_gated_linear_workspace_bytes(const ht_dense_problem *p, int backward) {
  if (screen(p) != HT_OK) return 0;
  return by_type(p->dtype, [&](auto zero) -> size_t {
    return Plan<decltype(zero)>(*p, nullptr, nullptr, nullptr, backward != 0, true, true, false, nullptr, nullptr).bytes;
  });
}

extern "C" size_t ht_gated_linear_kept_bytes(const ht_dense_problem *p) {
  if (screen(p) != HT_OK || p->rows == 0) return 0;
  return by_type(p->dtype, [&](auto zero) -> size_t {
    return Plan<decltype(zero)>(*p, nullptr, nullptr, nullptr, false, false, false, true, nullptr, nullptr).kept_bytes;
  });
}

extern "C" int ht_gated_linear_forward(const ht_dense_problem *p, const void *x, const void *gate_weight, const void *value_weight,
                                       const void *gate_bias, const void *value_bias, void *h, void *kept, void *workspace, size_t workspace_bytes,
                                       uint32_t *status_word, ht_stream_t stream) {
  const int rc = screen(p);
  if (rc != HT_OK) return rc;
  if (p->rows == 0) return HT_OK;
  if (x == nullptr || gate_weight == nullptr || value_weight == nullptr || h == nullptr) return HT_ERR_INVALID_ARGUMENT;
  if (!aligned({x, gate_weight, value_weight, gate_bias, value_bias, h, kept})) return HT_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return HT_ERR_WORKSPACE;
  return by_type(p->dtype, [&](auto zero) -> int {
    return forward<decltype(zero)>(*p, x, gate_weight, value_weight, gate_bias, value_bias, h, kept, workspace, workspace_bytes, status_word,
                                   reinterpret_cast<cudaStream_t>(stream));
  });
}

extern "C" int ht_gated_linear_backward(const ht_dense_problem *p, const void *x, const void *gate_weight, const void *value_weight,
                                        const void *gate_bias, const void *value_bias, const void *dh, const void *kept, void *dx, void *dgate_weight,
                                        void *dvalue_weight, void *dgate_bias, void *dvalue_bias, void *workspace, size_t workspace_bytes,
                                        uint32_t *status_word, ht_stream_t stream) {
  const int rc = screen(p);
  if (rc != HT_OK) return rc;
  if (p->rows > 0 && (x == nullptr || gate_weight == nullptr || value_weight == nullptr || dh == nullptr)) return HT_ERR_INVALID_ARGUMENT;
  if (!aligned({x, gate_weight, value_weight, gate_bias, value_bias, dh, kept, dx, dgate_weight, dvalue_weight})) return HT_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return HT_ERR_WORKSPACE;
  const Gradients out = {dx, dgate_weight, dvalue_weight, dgate_bias, dvalue_bias};
  return by_type(p->dtype, [&](auto zero) -> int {
    return backward<decltype(zero)>(*p, x, gate_weight, value_weight, gate_bias, value_bias, dh, kept, out, workspace, workspace_bytes, status_word,
                                    reinterpret_cast<cudaStream_t>(stream));
  });
}
