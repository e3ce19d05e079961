// Dense projection of a few rows (serving): the weights are read once and set the time.
//
// A workgroup owns 16 features n and all of K: its waves take 256-byte pieces of the 16 weight rows in
// turn, load them straight into MFMA fragments (lane l: row l % 16, 16 bytes at 16 (l / 16) of every 64),
// and add their sums over LDS in a fixed order.  A fragment's rows past M or N repeat the last row and are
// not stored.  Loads are at the elements' alignment, so odd strides and widths need no copy.
// 4096 x 4096 bf16 weights, in a graph: 1 row 6.9 us (4.9 TB/s), 16 rows 9.6 us (8.0 the one under a kernel trace).
#include "gl_dense.h"

namespace gl {

namespace {

template <int ES>
__device__ __forceinline__ uv4 load16(const char* row, int k, int kbytes, bool whole) {
  if (whole || k + 16 <= kbytes) return reinterpret_cast<const bytes16*>(row + k)->v;
  uv4 v = {0u, 0u, 0u, 0u};
  if constexpr (ES == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (k + 4 * j < kbytes) v[j] = *reinterpret_cast<const unsigned*>(row + k + 4 * j);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + 2 * j < kbytes) v[j >> 1] |= (unsigned)*reinterpret_cast<const unsigned short*>(row + k + 2 * j) << (16 * (j & 1));
  }
  return v;
}

template <int ES>
__device__ __forceinline__ f32x4 mma16(uv4 w, uv4 x, f32x4 c) {
  if constexpr (ES == 2) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w[j]), __uint_as_float(x[j]), c, 0, 0, 0);
    return c;
  }
}

// MT: groups of 16 rows; PIECES: 256-byte pieces of a row that a wave has in flight
template <int ES, int MT, int PIECES>
__global__ __launch_bounds__(1024) void dense_few_kernel(const char* __restrict__ X, long long sxb, const char* __restrict__ W,
                                                         long long swb, int M, int K, DenseEpi e) {
  extern __shared__ __align__(16) float sums[];  // [waves][MT][16 m][16 n]
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
  const int n0 = blockIdx.x * 16;
  const char* wr = W + (long long)min(n0 + (l & 15), e.N - 1) * swb;
  const char* xr[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) xr[t] = X + (long long)min(16 * t + (l & 15), M - 1) * sxb;
  const int kb = K * ES;  // below 2^23
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto pieces = [&](int p, bool whole) {
    uv4 wf[PIECES][4], xf[PIECES][MT][4];
#pragma unroll
    for (int q = 0; q < PIECES; ++q)
#pragma unroll
      for (int u = 0; u < 4; ++u) wf[q][u] = load16<ES>(wr, p + q * nw * 256 + (l >> 4) * 16 + 64 * u, kb, whole);
#pragma unroll
    for (int q = 0; q < PIECES; ++q)
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < 4; ++u) xf[q][t][u] = load16<ES>(xr[t], p + q * nw * 256 + (l >> 4) * 16 + 64 * u, kb, whole);
#pragma unroll
    for (int q = 0; q < PIECES; ++q)
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t] = mma16<ES>(wf[q][u], xf[q][t][u], acc[t]);
  };
  int p = wave * 256;
  for (; p + ((PIECES - 1) * nw + 1) * 256 <= kb; p += PIECES * nw * 256) pieces(p, true);
  if (p < kb) pieces(p, false);  // what is past the end is zero
#pragma unroll
  for (int t = 0; t < MT; ++t)
    *reinterpret_cast<f32x4*>(sums + ((wave * MT + t) * 16 + (l & 15)) * 16 + 4 * (l >> 4)) = acc[t];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 256; i += blockDim.x) {
    float s = 0.f;
    for (int w = 0; w < nw; ++w) s += sums[w * MT * 256 + i];
    const int m = i >> 4, n = n0 + (i & 15);
    if (m >= M || n >= e.N) continue;
    if (e.bias) s += ld_param((const float*)e.bias, e.op_bf, n);
    s = act_rt(e.act, s);
    if (e.res) s += ld_param((const float*)e.res, e.res_bf, m * e.sr + n);
    if (e.c_bf) ((unsigned short*)e.C)[m * e.sc + n] = to_bf16(s);
    else ((float*)e.C)[m * e.sc + n] = s;
  }
}

template <int ES, int MT, int PIECES>
int launch_few(const GlDenseArgs* a, const DenseEpi& e, hipStream_t s) {
  // one 256-byte piece of every weight row per wave, up to the 16 waves of a workgroup
  int nw = ceil_div((long long)a->K * ES, 256);
  nw = nw < 4 ? 4 : (nw > 16 ? 16 : nw);
  const size_t lds = (size_t)nw * MT * 1024;
  GL_LAUNCH(GL_KERNEL_DENSE_FEW, (dense_few_kernel<ES, MT, PIECES>), dim3((unsigned)ceil_div(a->N, 16)), dim3(nw * 64), lds, s,
            (const char*)a->X, a->sx * ES, (const char*)a->W, a->sw * ES, (int)a->M, a->K, e);
  GL_CHECK_LAUNCH();
  return 0;
}
template <int ES>
int launch_few_of(const GlDenseArgs* a, const DenseEpi& e, hipStream_t s) {
  if (a->M <= 16) return (long long)a->K * ES > 16 * 256 ? launch_few<ES, 1, 2>(a, e, s) : launch_few<ES, 1, 1>(a, e, s);
  if (a->M <= 32) return launch_few<ES, 2, 1>(a, e, s);
  return launch_few<ES, 4, 1>(a, e, s);
}

}  // namespace

int launch_dense_few(const GlDenseArgs* a, const DenseEpi& e, hipStream_t s) {
  return a->dtype == GL_DTYPE_BF16 ? launch_few_of<2>(a, e, s) : launch_few_of<4>(a, e, s);
}

}  // namespace gl
