// Layer norm over the features of a row, and its backward.
//
//     mu = mean x    r = 1 / sqrt(mean (x - mu)^2 + eps)    xh = (x - mu) r    y = xh w + b
//     dx = r (g - mean g - xh mean(g xh)),  g = w dy        dw = sum over the rows of dy xh    db = of dy
//
// Bound by bytes: x read and y written forward; x and dy read and dx written backward.  A row stays in the registers of
// its threads between its sums and its results, 8 neighbouring features a vector, so everything moves once; the mean is
// subtracted before squares are summed (two reductions a row).  Workgroups take rows in turn and keep what belongs to
// the features in registers meanwhile: w and b, and of the backward the sums of dw and db, which a second kernel adds
// over the workgroups in a fixed order.  Sums are fp32; results are rounded once.
#include "gl_internal.h"
#include "gl_pack8.h"

namespace gl {

namespace {

// the sum over a wave's lanes, the same bits in all of them
__device__ __forceinline__ float wave_total(float v) {
  v += dpp<0xB1>(v);   // lane ^ 1
  v += dpp<0x4E>(v);   // lane ^ 2
  v += dpp<0x141>(v);  // the other quad of eight
  v += dpp<0x140>(v);  // the other eight of a row
  const auto p16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(p16[0]) + __uint_as_float(p16[1]);
  const auto p32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(p32[0]) + __uint_as_float(p32[1]);
}

struct NormK {
  const void* X;
  const void* dY;  // backward
  const void* w;   // or null: ones
  const void* b;   // or null: zeros
  void* Y;         // forward; backward: dX, or null
  float* stats;    // [M][2] mean and r; forward: or null
  float* part;     // backward: [workgroups][2][D] sums of dw and db, or null
  long long sx, sy, sdy, M;
  int D, w_bf;
  float eps;
};

// eight parameters from feature c, of which n are there
__device__ __forceinline__ void norm_params(const void* p, bool bf, int c, int n, float otherwise, float (&v)[8]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = otherwise;
  } else if (bf) {
    load8<true>(p, c, n, v);
  } else {
    load8<false>(p, c, n, v);
  }
}

// T threads a row (a wave, or the workgroup), V vectors a thread: rows of up to 8 T V features.
template <int T, int V, bool XBF, bool YBF>
__global__ __launch_bounds__(T < 256 ? 256 : T) void norm_fwd_kernel(NormK a) {
  constexpr int ROWS = T < 256 ? 256 / T : 1, NW = T / 64;  // rows of a workgroup at a time, waves of a row
  __shared__ float red[2][NW];
  const int t = threadIdx.x % T;
  float w[V][8], b[V][8];
#pragma unroll
  for (int y = 0; y < V; ++y) {
    const int c = (y * T + t) * 8;
    norm_params(a.w, a.w_bf, c, a.D - c, 1.f, w[y]);
    norm_params(a.b, a.w_bf, c, a.D - c, 0.f, b[y]);
  }
  auto total = [&](float v, int which) {
    v = wave_total(v);
    if constexpr (NW > 1) {
      if ((threadIdx.x & 63) == 0) red[which][threadIdx.x >> 6] = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) v += red[which][k];
    }
    return v;
  };
  // (a row's threads leave together: rows of a workgroup share no barrier)
  for (long long m = (long long)blockIdx.x * ROWS + threadIdx.x / T; m < a.M; m += (long long)gridDim.x * ROWS) {
    float x[V][8], s = 0.f;
#pragma unroll
    for (int y = 0; y < V; ++y) {
      const int c = (y * T + t) * 8;
      load8<XBF>(a.X, m * a.sx + c, a.D - c, x[y]);
    }
#pragma unroll
    for (int y = 0; y < V; ++y)
#pragma unroll
      for (int j = 0; j < 8; ++j) s += x[y][j];
    const float mean = total(s, 0) / (float)a.D;  // (by 1 / D a constant row's would be off its value)
    s = 0.f;
#pragma unroll
    for (int y = 0; y < V; ++y) {
      const int left = a.D - (y * T + t) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[y][j] -= mean;
        if (left >= 8 || j < left) s = __builtin_fmaf(x[y][j], x[y][j], s);
      }
    }
    const float r = 1.f / __builtin_sqrtf(total(s, 1) / (float)a.D + a.eps);
#pragma unroll
    for (int y = 0; y < V; ++y) {
      const int c = (y * T + t) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[y][j] = __builtin_fmaf(x[y][j] * r, w[y][j], b[y][j]);
      store8<YBF>(a.Y, m * a.sy + c, a.D - c, x[y]);
    }
    if (a.stats && t == 0) {
      a.stats[2 * m] = mean;
      a.stats[2 * m + 1] = r;
    }
  }
}

template <int T, int V, bool XBF, bool YBF>
__global__ __launch_bounds__(T < 256 ? 256 : T) void norm_bwd_kernel(NormK a) {
  constexpr int ROWS = T < 256 ? 256 / T : 1, NW = T / 64;
  __shared__ float red[2][NW][2];
  extern __shared__ __align__(16) float sums[];  // [ROWS][8 T V] of rows that share a workgroup
  const int t = threadIdx.x % T;
  float w[V][8], dw[V][8], db[V][8];
#pragma unroll
  for (int y = 0; y < V; ++y) {
    const int c = (y * T + t) * 8;
    norm_params(a.w, a.w_bf, c, a.D - c, 1.f, w[y]);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[y][j] = db[y][j] = 0.f;
  }
  const float inv = 1.f / (float)a.D;
  int turn = 0;
  for (long long m = (long long)blockIdx.x * ROWS + threadIdx.x / T; m < a.M; m += (long long)gridDim.x * ROWS) {
    float x[V][8], g[V][8];
    const float mean = a.stats[2 * m], r = a.stats[2 * m + 1];
#pragma unroll
    for (int y = 0; y < V; ++y) {
      const int c = (y * T + t) * 8;
      load8<XBF>(a.X, m * a.sx + c, a.D - c, x[y]);
      load8<YBF>(a.dY, m * a.sdy + c, a.D - c, g[y]);
    }
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int y = 0; y < V; ++y)
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // (behind the row g is 0)
        x[y][j] = (x[y][j] - mean) * r;
        dw[y][j] = __builtin_fmaf(g[y][j], x[y][j], dw[y][j]);
        db[y][j] += g[y][j];
        g[y][j] *= w[y][j];
        s0 += g[y][j];
        s1 = __builtin_fmaf(g[y][j], x[y][j], s1);
      }
    if (!a.Y) continue;
    s0 = wave_total(s0);
    s1 = wave_total(s1);
    if constexpr (NW > 1) {  // the other half is written when every thread has passed a barrier after it read this one
      if ((threadIdx.x & 63) == 0) {
        red[turn][threadIdx.x >> 6][0] = s0;
        red[turn][threadIdx.x >> 6][1] = s1;
      }
      __syncthreads();
      s0 = s1 = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        s0 += red[turn][k][0];
        s1 += red[turn][k][1];
      }
      turn ^= 1;
    }
    s0 *= inv;
    s1 *= inv;
#pragma unroll
    for (int y = 0; y < V; ++y) {
      const int c = (y * T + t) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[y][j] = r * (g[y][j] - s0 - x[y][j] * s1);
      store8<XBF>(a.Y, m * a.D + c, a.D - c, x[y]);
    }
  }
  if (!a.part) return;
  float* part = a.part + (long long)blockIdx.x * 2 * a.D;
  auto write = [&](float (&v)[V][8], float* to) {
    if constexpr (ROWS > 1) {
      float* own = sums + (threadIdx.x / T) * (8 * T * V);
      __syncthreads();
#pragma unroll
      for (int y = 0; y < V; ++y)
#pragma unroll
        for (int j = 0; j < 8; ++j) own[(y * T + t) * 8 + j] = v[y][j];
      __syncthreads();
      for (int c = threadIdx.x; c < a.D; c += 256) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < ROWS; ++k) s += sums[k * (8 * T * V) + c];
        to[c] = s;
      }
    } else {
#pragma unroll
      for (int y = 0; y < V; ++y) {
        const int c = (y * T + t) * 8;
        store8<false>(to, c, a.D - c, v[y]);
      }
    }
  };
  write(dw, part);
  write(db, part + a.D);
}

// ---- rows that do not fit the registers of a workgroup -------------------------------------------------------
// Forward: a workgroup reads its row three times (the caches hold it).  Backward: g's two means a row first, then
// workgroups of 2048 features by a share of the rows.
constexpr int WIDE_T = 1024;
template <bool XBF, bool YBF, bool BWD>
__global__ __launch_bounds__(WIDE_T) void norm_wide_kernel(NormK a, float* means) {
  __shared__ float red[2][WIDE_T / 64];
  const float inv = 1.f / (float)a.D;
  auto total = [&](float v, int which) {
    v = wave_total(v);
    if ((threadIdx.x & 63) == 0) red[which][threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int k = 0; k < WIDE_T / 64; ++k) v += red[which][k];
    return v;
  };
  for (long long m = blockIdx.x; m < a.M; m += gridDim.x) {
    if constexpr (BWD) {
      const float mean = a.stats[2 * m], r = a.stats[2 * m + 1];
      float s0 = 0.f, s1 = 0.f;
      for (int c = threadIdx.x * 8; c < a.D; c += WIDE_T * 8) {
        float x[8], g[8], w[8];
        load8<XBF>(a.X, m * a.sx + c, a.D - c, x);
        load8<YBF>(a.dY, m * a.sdy + c, a.D - c, g);
        norm_params(a.w, a.w_bf, c, a.D - c, 1.f, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          g[j] *= w[j];
          s0 += g[j];
          s1 = __builtin_fmaf(g[j], (x[j] - mean) * r, s1);
        }
      }
      s0 = total(s0, 0);
      s1 = total(s1, 1);
      if (threadIdx.x == 0) {
        means[2 * m] = s0 * inv;
        means[2 * m + 1] = s1 * inv;
      }
      __syncthreads();
    } else {
      float s = 0.f, x[8];
      for (int c = threadIdx.x * 8; c < a.D; c += WIDE_T * 8) {
        load8<XBF>(a.X, m * a.sx + c, a.D - c, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) s += x[j];
      }
      const float mean = total(s, 0) / (float)a.D;  // (by 1 / D a constant row's would be off its value)
      s = 0.f;
      for (int c = threadIdx.x * 8; c < a.D; c += WIDE_T * 8) {
        load8<XBF>(a.X, m * a.sx + c, a.D - c, x);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j < a.D) s = __builtin_fmaf(x[j] - mean, x[j] - mean, s);
      }
      const float r = 1.f / __builtin_sqrtf(total(s, 1) / (float)a.D + a.eps);
      for (int c = threadIdx.x * 8; c < a.D; c += WIDE_T * 8) {
        float w[8], b[8];
        load8<XBF>(a.X, m * a.sx + c, a.D - c, x);
        norm_params(a.w, a.w_bf, c, a.D - c, 1.f, w);
        norm_params(a.b, a.w_bf, c, a.D - c, 0.f, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __builtin_fmaf((x[j] - mean) * r, w[j], b[j]);
        store8<YBF>(a.Y, m * a.sy + c, a.D - c, x);
      }
      if (a.stats && threadIdx.x == 0) {
        a.stats[2 * m] = mean;
        a.stats[2 * m + 1] = r;
      }
    }
  }
}
template <bool XBF, bool YBF>
__global__ __launch_bounds__(256) void norm_wide_dx_kernel(NormK a, const float* means) {
  const int c = (blockIdx.y * 256 + threadIdx.x) * 8, left = a.D - c;
  if (left <= 0) return;
  float w[8], dw[8], db[8];
  norm_params(a.w, a.w_bf, c, left, 1.f, w);
#pragma unroll
  for (int j = 0; j < 8; ++j) dw[j] = db[j] = 0.f;
  for (long long m = blockIdx.x; m < a.M; m += gridDim.x) {
    const float mean = a.stats[2 * m], r = a.stats[2 * m + 1];
    float x[8], g[8];
    load8<XBF>(a.X, m * a.sx + c, left, x);
    load8<YBF>(a.dY, m * a.sdy + c, left, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = (x[j] - mean) * r;
      dw[j] = __builtin_fmaf(g[j], x[j], dw[j]);
      db[j] += g[j];
    }
    if (!a.Y) continue;
    const float s0 = means[2 * m], s1 = means[2 * m + 1];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = r * (g[j] * w[j] - s0 - x[j] * s1);
    store8<XBF>(a.Y, m * a.D + c, left, x);
  }
  if (!a.part) return;
  float* part = a.part + (long long)blockIdx.x * 2 * a.D;
  store8<false>(part, c, left, dw);
  store8<false>(part + a.D, c, left, db);
}

// dw and db from the workgroups' sums: 64 columns by 16 waves, each a share of the workgroups, added in a fixed order
__global__ __launch_bounds__(1024) void norm_dw_kernel(const float* __restrict__ part, int groups, int D, void* dw, void* db,
                                                       int g_bf, int accumulate) {
  __shared__ float sums[16][64];
  const int l = threadIdx.x & 63, k = threadIdx.x >> 6;
  const long long c = (long long)blockIdx.x * 64 + l;
  float s = 0.f;
  if (c < 2LL * D) {
#pragma unroll 8
    for (int i = k; i < groups; i += 16) s += part[(long long)i * 2 * D + c];
  }
  sums[k][l] = s;
  __syncthreads();
  if (k != 0 || c >= 2LL * D) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += sums[i][l];
  void* to = c < D ? dw : db;
  const long long at = c < D ? c : c - D;
  if (!to) return;
  if (g_bf) ((unsigned short*)to)[at] = to_bf16(s);
  else ((float*)to)[at] = accumulate ? ((float*)to)[at] + s : s;
}

// ---- plans -----------------------------------------------------------------------------------------------------
// Widest row of T threads with V vectors each.  T and V are the least that hold the row.
enum { NORM_512 = 0, NORM_1K, NORM_2K, NORM_4K, NORM_8K, NORM_16K, NORM_WIDE };
inline int norm_form(int D) {
  int f = NORM_512;
  while (f < NORM_WIDE && D > (512 << f)) ++f;
  return f;
}
inline int norm_rows(int form) { return form <= NORM_1K ? 4 : 1; }  // of a workgroup at a time
constexpr int CUS = 256;
inline long long least(long long a, long long b) { return a < b ? a : b; }
inline int fwd_groups(long long M, int D) {
  const int f = norm_form(D);
  return (int)least((M + norm_rows(f) - 1) / norm_rows(f), f == NORM_WIDE ? 2 * CUS : (f == NORM_16K ? 2 : f == NORM_8K ? 4 : 8) * CUS);
}
// workgroups of the backward that keep sums (each leaves 8 D bytes of them)
inline int bwd_groups(long long M, int D) {
  const int f = norm_form(D);
  if (f == NORM_WIDE) return (int)least(M, 64);
  return (int)least((M + norm_rows(f) - 1) / norm_rows(f), 2 * CUS);
}

template <bool BWD, int T, int V, bool XBF, bool YBF>
int launch_norm_as(const NormK& k, int groups, hipStream_t s) {
  constexpr int threads = T < 256 ? 256 : T;
  if constexpr (BWD) {
    constexpr size_t lds = T < 256 ? 256 * 8 * V * 4 : 0;
    GL_LAUNCH(GL_KERNEL_NORM_BWD, (norm_bwd_kernel<T, V, XBF, YBF>), dim3((unsigned)groups), dim3(threads), lds, s, k);
  } else {
    GL_LAUNCH(GL_KERNEL_NORM, (norm_fwd_kernel<T, V, XBF, YBF>), dim3((unsigned)groups), dim3(threads), 0, s, k);
  }
  GL_CHECK_LAUNCH();
  return 0;
}
template <bool BWD, bool XBF, bool YBF>
int launch_norm_of(const NormK& k, int groups, float* means, hipStream_t s) {
  switch (norm_form(k.D)) {
    case NORM_512: return launch_norm_as<BWD, 64, 1, XBF, YBF>(k, groups, s);
    case NORM_1K: return launch_norm_as<BWD, 64, 2, XBF, YBF>(k, groups, s);
    case NORM_2K: return launch_norm_as<BWD, 256, 1, XBF, YBF>(k, groups, s);
    case NORM_4K: return launch_norm_as<BWD, 256, 2, XBF, YBF>(k, groups, s);
    case NORM_8K: return launch_norm_as<BWD, 512, 2, XBF, YBF>(k, groups, s);
    case NORM_16K: return launch_norm_as<BWD, 1024, 2, XBF, YBF>(k, groups, s);
    default: break;
  }
  if constexpr (BWD) {
    if (k.Y) {
      GL_LAUNCH(GL_KERNEL_NORM_BWD, (norm_wide_kernel<XBF, YBF, true>), dim3((unsigned)least(k.M, 2 * CUS)), dim3(WIDE_T), 0, s,
                k, means);
      GL_CHECK_LAUNCH();
    }
    GL_LAUNCH(GL_KERNEL_NORM_BWD, (norm_wide_dx_kernel<XBF, YBF>), dim3((unsigned)groups, (unsigned)ceil_div(k.D, 2048)),
              dim3(256), 0, s, k, (const float*)means);
  } else {
    GL_LAUNCH(GL_KERNEL_NORM, (norm_wide_kernel<XBF, YBF, false>), dim3((unsigned)groups), dim3(WIDE_T), 0, s, k, means);
  }
  GL_CHECK_LAUNCH();
  return 0;
}
template <bool BWD>
int launch_norm(const NormK& k, int x_dtype, int y_dtype, int groups, float* means, hipStream_t s) {
  const bool y = y_dtype == GL_DTYPE_BF16;
  if (x_dtype == GL_DTYPE_BF16)
    return y ? launch_norm_of<BWD, true, true>(k, groups, means, s) : launch_norm_of<BWD, true, false>(k, groups, means, s);
  return y ? launch_norm_of<BWD, false, true>(k, groups, means, s) : launch_norm_of<BWD, false, false>(k, groups, means, s);
}

bool dtype_ok(int d) { return d == GL_DTYPE_F32 || d == GL_DTYPE_BF16; }
bool on_element(const void* p, int dtype) { return ((uintptr_t)p & (dtype == GL_DTYPE_BF16 ? 1 : 3)) == 0; }
bool row_ok(long long stride, long long rows, long long cols) { return rows <= 1 || stride >= cols; }

int check_norm(const GlNormArgs* a) {
  if (!a || a->M < 0 || a->D < 1 || !(a->eps >= 0.f)) return GL_ERR_ARG;
  if (a->D > GL_DENSE_MAX_FEATURES || a->M > GL_NORM_MAX_ROWS) return GL_ERR_UNSUPPORTED;
  if (!dtype_ok(a->x_dtype) || !dtype_ok(a->y_dtype) || !dtype_ok(a->w_dtype)) return GL_ERR_UNSUPPORTED;
  if (a->M == 0) return 0;
  if (!a->X || !a->Y || !row_ok(a->sx, a->M, a->D) || !row_ok(a->sy, a->M, a->D)) return GL_ERR_ARG;
  if (!on_element(a->X, a->x_dtype) || !on_element(a->Y, a->y_dtype) || !on_element(a->weight, a->w_dtype) ||
      !on_element(a->bias, a->w_dtype) || !on_element(a->stats, GL_DTYPE_F32))
    return GL_ERR_ARG;
  return 0;
}
int check_norm_bwd(const GlNormBwdArgs* a) {
  if (!a || a->M < 0 || a->D < 1) return GL_ERR_ARG;
  if (a->D > GL_DENSE_MAX_FEATURES || a->M > GL_NORM_MAX_ROWS) return GL_ERR_UNSUPPORTED;
  if (!dtype_ok(a->x_dtype) || !dtype_ok(a->dy_dtype) || !dtype_ok(a->w_dtype) || !dtype_ok(a->g_dtype)) return GL_ERR_UNSUPPORTED;
  if (a->accumulate && a->g_dtype != GL_DTYPE_F32) return GL_ERR_ARG;
  if (a->M == 0) return 0;
  if (!a->X || !a->dY || !a->stats || !row_ok(a->sx, a->M, a->D) || !row_ok(a->sdy, a->M, a->D)) return GL_ERR_ARG;
  if (!on_element(a->X, a->x_dtype) || !on_element(a->dY, a->dy_dtype) || !on_element(a->weight, a->w_dtype) ||
      !on_element(a->dX, a->x_dtype) || !on_element(a->dweight, a->g_dtype) || !on_element(a->dbias, a->g_dtype) ||
      !on_element(a->stats, GL_DTYPE_F32))
    return GL_ERR_ARG;
  return 0;
}
// bytes of the workgroups' sums, then of the rows' means
size_t part_bytes(const GlNormBwdArgs* a) {
  return a->dweight || a->dbias ? (size_t)round_up((long long)bwd_groups(a->M, a->D) * 8 * a->D, 256) : 0;
}
size_t bwd_bytes(const GlNormBwdArgs* a) {
  return part_bytes(a) + (norm_form(a->D) == NORM_WIDE && a->dX ? (size_t)round_up(a->M * 8, 256) : 0);
}

}  // namespace

}  // namespace gl

using namespace gl;

extern "C" int gl_norm_fwd(const GlNormArgs* a, void* stream) {
  GL_TRY(check_norm(a));
  if (a->M == 0) return 0;
  NormK k{};
  k.X = a->X;
  k.w = a->weight;
  k.b = a->bias;
  k.Y = a->Y;
  k.stats = a->stats;
  k.sx = a->sx;
  k.sy = a->sy;
  k.M = a->M;
  k.D = a->D;
  k.w_bf = a->w_dtype == GL_DTYPE_BF16;
  k.eps = a->eps;
  return launch_norm<false>(k, a->x_dtype, a->y_dtype, fwd_groups(a->M, a->D), nullptr, (hipStream_t)stream);
}

extern "C" int gl_norm_bwd_workspace(const GlNormBwdArgs* a, size_t* bytes) {
  GL_TRY(check_norm_bwd(a));
  if (!bytes) return GL_ERR_ARG;
  *bytes = a->M == 0 ? 0 : bwd_bytes(a);
  return 0;
}

extern "C" int gl_norm_bwd(const GlNormBwdArgs* a, void* stream) {
  GL_TRY(check_norm_bwd(a));
  if (a->M == 0 || (!a->dX && !a->dweight && !a->dbias)) return 0;
  const size_t need = bwd_bytes(a);
  if (a->ws_bytes < need) return GL_ERR_WORKSPACE;
  if (need && (!a->ws || ((uintptr_t)a->ws & 255))) return GL_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  const int groups = bwd_groups(a->M, a->D);
  const size_t part = part_bytes(a);
  NormK k{};
  k.X = a->X;
  k.dY = a->dY;
  k.w = a->weight;
  k.Y = a->dX;
  k.stats = const_cast<float*>(a->stats);
  k.part = part ? (float*)a->ws : nullptr;
  k.sx = a->sx;
  k.sdy = a->sdy;
  k.M = a->M;
  k.D = a->D;
  k.w_bf = a->w_dtype == GL_DTYPE_BF16;
  GL_TRY(launch_norm<true>(k, a->x_dtype, a->dy_dtype, groups, (float*)((char*)a->ws + part), s));
  if (part) {
    GL_LAUNCH(GL_KERNEL_NORM_DW, norm_dw_kernel, dim3((unsigned)ceil_div(2LL * a->D, 64)), dim3(1024), 0, s,
              (const float*)k.part, groups, a->D, a->dweight, a->dbias, (int)(a->g_dtype == GL_DTYPE_BF16), a->accumulate);
    GL_CHECK_LAUNCH();
  }
  return 0;
}
