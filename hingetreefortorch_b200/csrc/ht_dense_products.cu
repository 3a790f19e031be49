// The two products of a dense layer's backward pass: with the gradient g [rows, outputs] of its results as an operand,
//   dx = g w        g with the contracted outputs contiguous, w [outputs, features] with the features contiguous
//   dw = g^T x      both with what is kept contiguous; contracted over the rows
// Both are the tile product with the scaled store as its epilogue.
#include "ht_dense.cuh"

namespace ht {
namespace dense {

namespace {
template <typename T, bool A_MN>
int product(const TileProblem &p, StoreEpilogue<T> &e, float *parts, int sms, cudaStream_t stream) {
  constexpr int kPlanes = GradKind<T>::kPlanes;
  const TileShape shape = product_shape(p.rows, p.cols, p.k * p.segments, kPlanes, parts != nullptr);
  if (shape.split == 1) return launch_tiles<kPlanes, A_MN, true>(p, e, shape, sms, stream);
  e.parts = parts;
  e.parts_pitch = (int)round_up(p.cols, 8);
  HT_TRY((launch_tiles<kPlanes, A_MN, true>(p, e, shape, sms, stream)));
  return launch_next<add_parts_kernel<T>>(dim3(blocks_for(p.rows * (e.parts_pitch / 4), 256, 148 * 8)), 256, 0, 0, stream, 1, e, parts_of(p, shape));
}
}  // namespace

template <typename T>
int product_dx(const TileProblem &p, StoreEpilogue<T> e, float *parts, int sms, cudaStream_t stream) {
  return product<T, false>(p, e, parts, sms, stream);
}
template <typename T>
int product_dw(const TileProblem &p, StoreEpilogue<T> e, float *parts, int sms, cudaStream_t stream) {
  return product<T, true>(p, e, parts, sms, stream);
}

#define HT_DENSE_PRODUCTS(T)                                                                            \
  template int product_dx<T>(const TileProblem &, StoreEpilogue<T>, float *, int, cudaStream_t);    \
  template int product_dw<T>(const TileProblem &, StoreEpilogue<T>, float *, int, cudaStream_t);
HT_DENSE_PRODUCTS(float)
HT_DENSE_PRODUCTS(__nv_bfloat16)
HT_DENSE_PRODUCTS(__half)

}  // namespace dense
}  // namespace ht
