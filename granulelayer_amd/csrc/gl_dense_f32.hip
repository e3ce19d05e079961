// fp32 instances of the dense tile kernel (gl_dense.h): fp32 MFMA, 1/16 of the bf16 rate, so a stage's LDS reads
// and copies are a small part of its products and no tile past 128 x 128 is needed.  2048 x 4096 over 1024: 133 us,
// 129 TFLOP/s; 4096 x 4096 over 4096: 994 us, 138 TFLOP/s (a large library product reaches 154).  The deep tile has
// eight waves: one workgroup a CU then keeps as many waves as two of the plain one.
#include "gl_dense.h"

namespace gl {

int launch_dense_tile_f32(int form, int tile, const DenseK& a, int splits, hipStream_t s) {
  if (tile == DENSE_128) return launch_dense_tile_of<4, 16, 128, 128, 2, 2, 2, 2>(form, a, splits, s);
  if (tile == DENSE_128_DEEP) return launch_dense_tile_of<4, 16, 128, 128, 4, 2, 3, 3>(form, a, splits, s);
  return launch_dense_tile_of<4, 16, 64, 128, 2, 2, 3, 3>(form, a, splits, s);
}

}  // namespace gl
