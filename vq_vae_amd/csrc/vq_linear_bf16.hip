// The products of vq_linear* for bf16 elements (device code in vq_linear.h).
#include "vq_linear.h"

VQL_KERNELS(VqBf16)

int vql_product_bf16(const VqLinearArgs& a, int layout, int config, bool dma, hipStream_t s) {
  return vql_product<VqBf16>(a, layout, config, dma, s);
}
