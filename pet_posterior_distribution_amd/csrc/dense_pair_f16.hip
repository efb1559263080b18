// Instances of the dense layer's backward pass as one launch for f16 operands.
#include "dense_product.h"

namespace petdense_k {

hipError_t pair_f16(const Pair& p, int lx, int lk, int tile, int q8, hipStream_t s) {
  return pair<_Float16>(p, lx, lk, tile, q8, s);
}

hipError_t fused_f16(const Pair& p, int tile, int q8, hipStream_t s) { return fused<_Float16>(p, tile, q8, s); }

}  // namespace petdense_k
