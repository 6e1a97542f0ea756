// bcfft_dense_f32.hip — the dense products of fp32 operands (kernels: bcfft_dense_tile.h, bcfft_dense_launch.h).
#include "bcfft_dense_launch.h"

namespace bcfft {
void launch_product_f32(const DenseArgs& a, DenseLayout layout, Shape sh, hipStream_t s) {
  launch_product_dt<BCFFT_F32>(a, layout, sh, s);
}
}  // namespace bcfft
