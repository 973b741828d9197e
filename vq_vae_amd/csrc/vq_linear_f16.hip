// The products of vq_linear* for f16 elements (device code in vq_linear.h).
#include "vq_linear.h"

VQL_KERNELS(_Float16)

int vql_product_f16(const VqLinearArgs& a, int layout, int config, bool dma, hipStream_t s) {
  return vql_product<_Float16>(a, layout, config, dma, s);
}
