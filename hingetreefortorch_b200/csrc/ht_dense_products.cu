// The two products of a dense layer's backward pass: with the gradient g [rows, outputs] of its results as an operand,
//   dx = g w        g with the contracted outputs contiguous, w [outputs, features] with the features contiguous
//   dw = g^T x      both with what is kept contiguous; contracted over the rows
// Both are the tile product with the scaled store as its epilogue.
#include "ht_dense.cuh"

namespace ht {
namespace dense {

template <typename T>
int product_dx(const TileProblem &p, const StoreEpilogue<T> &e, int sms, cudaStream_t stream) {
  constexpr int kPlanes = Kind<T>::kPlanes;
  return launch_tiles<kPlanes, false, true>(p, e, tile_shape(p.rows, p.cols, p.k * p.segments, kPlanes, false), sms, stream);
}
template <typename T>
int product_dw(const TileProblem &p, const StoreEpilogue<T> &e, int sms, cudaStream_t stream) {
  constexpr int kPlanes = Kind<T>::kPlanes;
  return launch_tiles<kPlanes, true, true>(p, e, tile_shape(p.rows, p.cols, p.k, kPlanes, false), sms, stream);
}

#define HT_DENSE_PRODUCTS(T)                                                                       \
  template int product_dx<T>(const TileProblem &, const StoreEpilogue<T> &, int, cudaStream_t);    \
  template int product_dw<T>(const TileProblem &, const StoreEpilogue<T> &, int, cudaStream_t);
HT_DENSE_PRODUCTS(float)
HT_DENSE_PRODUCTS(__nv_bfloat16)
HT_DENSE_PRODUCTS(__half)

}  // namespace dense
}  // namespace ht
