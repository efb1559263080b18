// Instances of the dense layer's backward pass as one launch for f32 operands.
#include "dense_product.h"

namespace petdense_k {

hipError_t pair_f32(const Pair& p, int lx, int lk, int tile, int q8, hipStream_t s) {
  return pair<float>(p, lx, lk, tile, q8, s);
}

hipError_t fused_f32(const Pair& p, int tile, int q8, hipStream_t s) { return fused<float>(p, tile, q8, s); }

}  // namespace petdense_k
