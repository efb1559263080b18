// Instances of the dense layer's tiled products for f32 operands.
#include "dense_product.h"

namespace petdense_k {

hipError_t product_f32(const Product& p, int layout, int loader, int tile, int q8, hipStream_t s) {
  return product<float>(p, layout, loader, tile, q8, s);
}

}  // namespace petdense_k
