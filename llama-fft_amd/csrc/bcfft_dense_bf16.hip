// bcfft_dense_bf16.hip — the dense products of bf16 operands (kernels: bcfft_dense_tile.h, bcfft_dense_launch.h).
#include "bcfft_dense_launch.h"

namespace bcfft {
void launch_product_bf16(const DenseArgs& a, DenseLayout layout, Shape sh, hipStream_t s) {
  launch_product_dt<BCFFT_BF16>(a, layout, sh, s);
}
}  // namespace bcfft
