// The products of vq_linear* for f32 elements (device code in vq_linear.h).
#include "vq_linear.h"

VQL_KERNELS(float)

int vql_product_f32(const VqLinearArgs& a, int layout, int config, bool dma, hipStream_t s) {
  return vql_product<float>(a, layout, config, dma, s);
}
