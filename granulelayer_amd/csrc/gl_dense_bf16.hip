// bf16 instances of the dense tile kernel (gl_dense.h).
//
// 4096 x 4096 over 16384 (TN), 16384 x 4096 over 4096 (NT, NN), one MI355X: 397, 411 and 412 us, 1.33 to 1.38 PFLOP/s,
// at a clock that the card's power sets (1.6 GHz).  A stage of the 256 x 256 tile takes 2320 clocks (NT) to 2470 (TN)
// against 2048 of matrix instructions.  P has three stages of LDS and Q two, all 160 KB: with two each a
// stage's copies come late and it takes 2720 to 2830; five stages of 64 bytes (2600) fetch RC lines twice.
#include "gl_dense.h"

namespace gl {

int launch_dense_tile_bf16(int form, int tile, const DenseK& a, int splits, hipStream_t s) {
  switch (tile) {
    case DENSE_256: return launch_dense_tile_of<2, 256, 256, 2, 4, 3, 2>(form, a, splits, s);
    case DENSE_256X128: return launch_dense_tile_of<2, 256, 128, 4, 2, 3, 3>(form, a, splits, s);
    case DENSE_128: return launch_dense_tile_of<2, 128, 128, 2, 2, 2, 2>(form, a, splits, s);
    case DENSE_128_DEEP: return launch_dense_tile_of<2, 128, 128, 2, 2, 3, 3>(form, a, splits, s);
    default: return launch_dense_tile_of<2, 64, 128, 2, 2, 3, 3>(form, a, splits, s);
  }
}

}  // namespace gl
