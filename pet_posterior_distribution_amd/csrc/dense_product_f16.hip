// Instances of the dense layer's tiled products for f16 operands.
#include "dense_product.h"

namespace petdense_k {

hipError_t product_f16(const Product& p, int layout, int loader, int tile, int q8, hipStream_t s) {
  return product<_Float16>(p, layout, loader, tile, q8, s);
}

}  // namespace petdense_k
