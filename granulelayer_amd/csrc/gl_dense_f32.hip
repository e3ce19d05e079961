// fp32 instances of the dense tile kernel (gl_dense.h): fp32 MFMA, 1/16 of the bf16 rate, so a stage's
// LDS reads are a small part of its products and no tile past 128 x 128 is needed.
#include "gl_dense.h"

namespace gl {

int launch_dense_tile_f32(int form, int tile, const DenseK& a, int splits, hipStream_t s) {
  if (tile == DENSE_128) return launch_dense_tile_of<4, 128, 128, 2, 2>(form, a, splits, s);
  return launch_dense_tile_of<4, 64, 128, 2, 2>(form, a, splits, s);
}

}  // namespace gl
