// Activations put into 8 bits and read back (gl_pack8, gl_unpack8); the format is in gl_pack8.h.
//
// Both kernels move each byte once and are bound by memory.  A lane holds 8 values of one 32-value
// block, so four neighbouring lanes share a block and its maximum is two lane swaps; a wave's
// accesses are contiguous along the row.  131072 x 2048 bf16: 160 us into 8 bits (5.1 TB/s), 156 us back (5.2 TB/s).
#include "gl_internal.h"
#include "gl_pack8.h"

namespace gl {

namespace {

constexpr int THREADS = 256;
constexpr int SEGS = 4;  // accesses a lane has in flight

// Lanes along a row: a power of two from 4 (one block) to 64; a workgroup holds THREADS / tpr rows.
inline int lanes_per_row(int slots) {
  int t = 4;
  while (t < 64 && t < slots) t *= 2;
  return t;
}

// grid: x = groups of THREADS / tpr rows, y = segments of SEGS * tpr slots of 8 values
template <bool BF>
__global__ __launch_bounds__(THREADS) void pack8_kernel(const void* __restrict__ x, long long sx, long long rows, int cols,
                                                        int tpr_log2, uint8_t* __restrict__ q, uint8_t* __restrict__ e) {
  const int nb = (cols + P8_BLOCK - 1) / P8_BLOCK;
  const long long r = (long long)blockIdx.x * (THREADS >> tpr_log2) + (threadIdx.x >> tpr_log2);
  const int c0 = (blockIdx.y * SEGS << tpr_log2) + (threadIdx.x & ((1 << tpr_log2) - 1));
  if (r >= rows) return;  // whole blocks leave together: tpr is a multiple of 4
  float v[SEGS][8];
#pragma unroll
  for (int s = 0; s < SEGS; ++s) {
    const int c = (c0 + (s << tpr_log2)) * 8;
    load8<BF>(x, r * sx + c, cols - c, v[s]);
  }
#pragma unroll
  for (int s = 0; s < SEGS; ++s) {
    const int slot = c0 + (s << tpr_log2);
    unsigned a = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) a = umax(a, abs_bits(v[s][j]));
    a = umax(a, (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, 0xB1, 0xf, 0xf, false));  // lane ^ 1
    a = umax(a, (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, 0x4E, 0xf, 0xf, false));  // lane ^ 2
    if (slot >= nb * 4) continue;
    const int ex = p8_exp(a);
    const float is = p8_inv_step(ex);
    uv2 w;
    w[0] = p8_codes4(v[s][0], v[s][1], v[s][2], v[s][3], is);
    w[1] = p8_codes4(v[s][4], v[s][5], v[s][6], v[s][7], is);
    *reinterpret_cast<uv2*>(q + (r * nb * P8_BLOCK + slot * 8)) = w;
    if ((slot & 3) == 0) e[r * nb + (slot >> 2)] = (uint8_t)ex;
  }
}

template <bool BF>
__global__ __launch_bounds__(THREADS) void unpack8_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ e,
                                                          long long rows, int cols, int tpr_log2, void* __restrict__ x,
                                                          long long sx) {
  const int nb = (cols + P8_BLOCK - 1) / P8_BLOCK;
  const long long r = (long long)blockIdx.x * (THREADS >> tpr_log2) + (threadIdx.x >> tpr_log2);
  const int c0 = (blockIdx.y * SEGS << tpr_log2) + (threadIdx.x & ((1 << tpr_log2) - 1));
  if (r >= rows) return;
  uv2 w[SEGS];
  int ex[SEGS];
#pragma unroll
  for (int s = 0; s < SEGS; ++s) {
    const int slot = c0 + (s << tpr_log2);
    if (slot < nb * 4) {
      w[s] = *reinterpret_cast<const uv2*>(q + (r * nb * P8_BLOCK + slot * 8));
      ex[s] = e[r * nb + (slot >> 2)];
    }
  }
#pragma unroll
  for (int s = 0; s < SEGS; ++s) {
    const int c = (c0 + (s << tpr_log2)) * 8;
    if (c >= cols) continue;
    const float st = p8_step(ex[s]);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p8_value(w[s][j >> 2], j & 3, st);
    store8<BF>(x, r * sx + c, cols - c, v);
  }
}

struct Grid {
  dim3 grid;
  int tpr_log2;
};
inline Grid grid_of(long long rows, int cols) {
  const int slots = ceil_div(cols, P8_BLOCK) * 4, tpr = lanes_per_row(slots);
  Grid g;
  g.tpr_log2 = __builtin_ctz((unsigned)tpr);
  g.grid = dim3((unsigned)((rows + THREADS / tpr - 1) / (THREADS / tpr)), (unsigned)ceil_div(slots, SEGS * tpr));
  return g;
}

int check(const GlPack8Args* a) {
  if (!a || a->rows < 0 || a->cols < 1 || a->cols > GL_DENSE_MAX_FEATURES) return GL_ERR_ARG;
  if (a->x_dtype != GL_DTYPE_F32 && a->x_dtype != GL_DTYPE_BF16) return GL_ERR_UNSUPPORTED;
  if (a->rows >= GL_DENSE_MAX_ROWS) return GL_ERR_UNSUPPORTED;
  if (a->rows == 0) return 0;
  if (!a->x || !a->q || !a->e || a->sx < 0 || (a->rows > 1 && a->sx < a->cols)) return GL_ERR_ARG;
  const uintptr_t es = a->x_dtype == GL_DTYPE_F32 ? 4 : 2;
  if (((uintptr_t)a->x & (es - 1)) || ((uintptr_t)a->q & 7)) return GL_ERR_ARG;
  return 0;
}

}  // namespace

int launch_unpack8(const uint8_t* q, const uint8_t* e, long long rows, int cols, void* x, long long sx, int x_dtype,
                   hipStream_t s) {
  const Grid g = grid_of(rows, cols);
  if (x_dtype == GL_DTYPE_BF16)
    GL_LAUNCH(GL_KERNEL_UNPACK8, unpack8_kernel<true>, g.grid, dim3(THREADS), 0, s, q, e, rows, cols, g.tpr_log2, x, sx);
  else
    GL_LAUNCH(GL_KERNEL_UNPACK8, unpack8_kernel<false>, g.grid, dim3(THREADS), 0, s, q, e, rows, cols, g.tpr_log2, x, sx);
  GL_CHECK_LAUNCH();
  return 0;
}

}  // namespace gl

using namespace gl;

extern "C" int gl_pack8(const GlPack8Args* a, void* stream) {
  GL_TRY(check(a));
  if (a->rows == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
  const Grid g = grid_of(a->rows, a->cols);
  if (a->x_dtype == GL_DTYPE_BF16)
    GL_LAUNCH(GL_KERNEL_PACK8, pack8_kernel<true>, g.grid, dim3(THREADS), 0, s, a->x, a->sx, a->rows, a->cols, g.tpr_log2,
              a->q, a->e);
  else
    GL_LAUNCH(GL_KERNEL_PACK8, pack8_kernel<false>, g.grid, dim3(THREADS), 0, s, a->x, a->sx, a->rows, a->cols, g.tpr_log2,
              a->q, a->e);
  GL_CHECK_LAUNCH();
  return 0;
}

extern "C" int gl_unpack8(const GlPack8Args* a, void* stream) {
  GL_TRY(check(a));
  if (a->rows == 0) return 0;
  return launch_unpack8(a->q, a->e, a->rows, a->cols, a->x, a->sx, a->x_dtype, (hipStream_t)stream);
}
