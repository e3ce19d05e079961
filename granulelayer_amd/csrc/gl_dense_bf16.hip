// bf16 instances of the dense tile kernel (gl_dense.h).
#include "gl_dense.h"

namespace gl {

int launch_dense_tile_bf16(int form, int tile, const DenseK& a, int splits, hipStream_t s) {
  if (tile == DENSE_256) return launch_dense_tile_of<2, 256, 256, 2, 4>(form, a, splits, s);
  if (tile == DENSE_128) return launch_dense_tile_of<2, 128, 128, 2, 2>(form, a, splits, s);
  return launch_dense_tile_of<2, 64, 128, 2, 2>(form, a, splits, s);
}

}  // namespace gl
