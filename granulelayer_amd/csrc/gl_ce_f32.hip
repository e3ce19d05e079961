// fp32 instances of the dense tile kernel (gl_dense.h) for the cross entropy (gl_ce.hip), with the tiles of
// gl_dense_f32.hip.
#include "gl_dense.h"

namespace gl {

int launch_rows_tile_f32(int kind, int form, int tile, const DenseRowsK& a, int splits, hipStream_t s) {
  if (tile == DENSE_128) return launch_rows_tile_of<4, 16, 128, 128, 2, 2, 2, 2>(kind, form, a, splits, s);
  if (tile == DENSE_128_DEEP) return launch_rows_tile_of<4, 16, 128, 128, 4, 2, 3, 3>(kind, form, a, splits, s);
  return launch_rows_tile_of<4, 16, 64, 128, 2, 2, 3, 3>(kind, form, a, splits, s);
}

}  // namespace gl
