// bf16 instances of the dense tile kernel (gl_dense.h) for the cross entropy (gl_ce.hip), with the tiles of
// gl_dense_bf16.hip.
#include "gl_dense.h"

namespace gl {

int launch_rows_tile_bf16(int kind, int form, int tile, const DenseRowsK& a, int splits, hipStream_t s) {
  switch (tile) {
    case DENSE_256: return launch_rows_tile_of<2, 16, 256, 256, 2, 4, 3, 2>(kind, form, a, splits, s);
    case DENSE_256X128: return launch_rows_tile_of<2, 32, 256, 128, 4, 2, 3, 3>(kind, form, a, splits, s);
    case DENSE_128: return launch_rows_tile_of<2, 32, 128, 128, 2, 2, 2, 2>(kind, form, a, splits, s);
    case DENSE_128_DEEP: return launch_rows_tile_of<2, 32, 128, 128, 2, 2, 3, 3>(kind, form, a, splits, s);
    default: return launch_rows_tile_of<2, 32, 64, 128, 2, 2, 3, 3>(kind, form, a, splits, s);
  }
}

}  // namespace gl
