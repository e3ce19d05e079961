// bf16 instances of the dense tile kernel (gl_dense.h).
//
// 16384 x 4096 over 4096 (NT, NN), 4096 x 4096 over 16384 (TN), one MI355X: 395, 399 and 373 us, 1.38 to 1.47 PFLOP/s
// (library products 347, 402 and 457), at a clock that the card's power sets (1.75 GHz).  A stage of the 256 x 256 tile takes 2500 (TN) to 2600 clocks, of which
// 2048 are matrix instructions and about 350 the copies' (2216 without any).  P has three stages of LDS and Q
// two, all 160 KB; with two each copies come late (416, 420 and 402 us), and five stages of 64 bytes fetch RC lines twice.
// Instructions of 16 x 16 where two waves of a SIMD share its power, of 32 x 32 in the smaller tiles (gl_dense.h).
#include "gl_dense.h"

namespace gl {

int launch_dense_tile_bf16(int form, int tile, const DenseK& a, int splits, hipStream_t s) {
  switch (tile) {
    case DENSE_256: return launch_dense_tile_of<2, 16, 256, 256, 2, 4, 3, 2>(form, a, splits, s);
    case DENSE_256X128: return launch_dense_tile_of<2, 32, 256, 128, 4, 2, 3, 3>(form, a, splits, s);
    case DENSE_128: return launch_dense_tile_of<2, 32, 128, 128, 2, 2, 2, 2>(form, a, splits, s);
    case DENSE_128_DEEP: return launch_dense_tile_of<2, 32, 128, 128, 2, 2, 3, 3>(form, a, splits, s);
    default: return launch_dense_tile_of<2, 32, 64, 128, 2, 2, 3, 3>(form, a, splits, s);
  }
}

}  // namespace gl
