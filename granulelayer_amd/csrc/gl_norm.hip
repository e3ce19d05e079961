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
//
// 32768 x 8192 bf16: forward 191 us (5.6 TB/s), backward 269 (6.0) + 5; 8192 x 4096 fp32 with bf16 results: 39 (5.2),
// 69 (4.8) + 4; 16384 x 1024 bf16: 13.4 (5.0), 26 (3.9); a copy of 4 GB reaches 4.97.  Rows that do not begin on 16 bytes:
// 32768 x 2101 bf16 69 (4.0), 107 (3.9), where 2096 takes 63 and 93.
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

// Eight features as they are stored: a row that is on its way to the next turn, and one that is read twice.
template <bool BF>
struct Eight {
  uv4 w[BF ? 1 : 2];
};
typedef unsigned uv4_at __attribute__((ext_vector_type(4), aligned(2)));
// STREAM: the caches need not keep it
template <bool BF, bool STREAM>
__device__ __forceinline__ Eight<BF> load_eight(const void* p, long long i, int n) {
  Eight<BF> e;
  if (n >= 8) {
#pragma unroll
    for (int h = 0; h < (BF ? 1 : 2); ++h) {
      const uv4_at* q = reinterpret_cast<const uv4_at*>((const char*)p + (BF ? 2 : 4) * i + 16 * h);
      if constexpr (STREAM) e.w[h] = __builtin_nontemporal_load(q);
      else e.w[h] = *q;
    }
  } else {
    float v[8];
    load8<BF>(p, i, n, v);
    if constexpr (BF) {
#pragma unroll
      for (int j = 0; j < 4; ++j) e.w[0][j] = __float_as_uint(v[2 * j]) >> 16 | __float_as_uint(v[2 * j + 1]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) e.w[j >> 2][j & 3] = __float_as_uint(v[j]);
    }
  }
  return e;
}
template <bool BF>
__device__ __forceinline__ float value(const Eight<BF>& e, int j) {
  if constexpr (BF) return __uint_as_float(j & 1 ? e.w[0][j >> 1] & 0xffff0000u : e.w[0][j >> 1] << 16);
  else return __uint_as_float(e.w[j >> 2][j & 3]);
}
template <bool BF, bool STREAM>
__device__ __forceinline__ void store_eight(void* p, long long i, int n, const float (&v)[8]) {
  if (!STREAM || n < 8) {
    store8<BF>(p, i, n, v);
  } else if constexpr (BF) {
    uv4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = to_bf16x2(v[2 * j], v[2 * j + 1]);
    __builtin_nontemporal_store(w, reinterpret_cast<uv4_at*>((char*)p + 2 * i));
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uv4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(v[4 * h + j]);
      __builtin_nontemporal_store(w, reinterpret_cast<uv4_at*>((char*)p + 4 * i + 16 * h));
    }
  }
}

// A thread's eight features from the c-th on: the row's last eight where it would end before them, of which those from `lo`
// on are its own (rows of fewer: `hi` of them; threads behind the row: none).  So every load is a vector: a wave that
// gathered a row's end by elements would wait for them at once, and with them for the row that is on its way.
struct Place {
  int c, lo, hi;
};
__device__ __forceinline__ Place place_of(int c, int D) {
  const int last = D > 8 ? D - 8 : 0;
  return Place{c < last ? c : last, c <= last ? 0 : c - last < 8 ? c - last : 8, D < 8 ? D : 8};
}
__device__ __forceinline__ bool own(const Place& p, int j) { return j >= p.lo && j < p.hi; }
// stores a place's own features
template <bool BF, bool STREAM>
__device__ __forceinline__ void store_own(void* to, long long row, const Place& p, const float (&v)[8]) {
  if (p.lo == 0) {
    store_eight<BF, STREAM>(to, row + p.c, p.hi, v);
  } else {
#pragma unroll
    for (int j = 1; j < 8; ++j)
      if (own(p, j)) {
        if constexpr (BF) ((unsigned short*)to)[row + p.c + j] = to_bf16(v[j]);
        else ((float*)to)[row + p.c + j] = v[j];
      }
  }
}

// Totals over the threads of a row, the same bits in all of them: a wave's, or (WAVE false) those of up to 16 waves, of
// which this is number `wave`, through `red`, 16 pairs that are 0 where there is no wave.
template <bool WAVE>
__device__ __forceinline__ void row_totals(float& a, float& b, float (*red)[2], int wave) {
  a = wave_total(a);
  b = wave_total(b);
  if constexpr (!WAVE) {
    const int l = threadIdx.x & 63;
    if (l == 0) {
      red[wave][0] = a;
      red[wave][1] = b;
    }
    __syncthreads();
    a = red[l & 15][0];
    b = red[l & 15][1];
    a += dpp<0xB1>(a);
    b += dpp<0xB1>(b);
    a += dpp<0x4E>(a);
    b += dpp<0x4E>(b);
    a += dpp<0x141>(a);
    b += dpp<0x141>(b);
    a += dpp<0x140>(a);
    b += dpp<0x140>(b);
  }
}

// A row is a wave's (WAVE: four rows a workgroup) or a workgroup's, with V vectors a thread.  The next turn's row is
// loaded before this one's sums, so a workgroup always has a row on its way.
template <bool WAVE, int V, bool XBF, bool YBF, bool STREAM>
__global__ __launch_bounds__(WAVE || V == 1 ? 256 : 512) void norm_fwd_kernel(NormK a) {
  __shared__ float red[2][16][2];
  constexpr int ROWS = WAVE ? 4 : 1;
  const int T = WAVE ? 64 : blockDim.x, t = WAVE ? threadIdx.x & 63 : threadIdx.x;
  if constexpr (!WAVE) {
    if (threadIdx.x < 64) (&red[0][0][0])[threadIdx.x] = 0.f;
    __syncthreads();
  }
  Place at[V];
  float w[V][8], b[V][8];
#pragma unroll
  for (int y = 0; y < V; ++y) {
    at[y] = place_of((y * T + t) * 8, a.D);
    norm_params(a.w, a.w_bf, at[y].c, at[y].hi, 1.f, w[y]);
    norm_params(a.b, a.w_bf, at[y].c, at[y].hi, 0.f, b[y]);
  }
  const long long step = (long long)gridDim.x * ROWS;
  long long m = (long long)blockIdx.x * ROWS + (WAVE ? threadIdx.x >> 6 : 0);
  Eight<XBF> next[V];
  auto fetch = [&](long long row) {
#pragma unroll
    for (int y = 0; y < V; ++y) next[y] = load_eight<XBF, STREAM>(a.X, row * a.sx + at[y].c, at[y].hi);
  };
  if (m < a.M) fetch(m);
  for (; m < a.M; m += step) {
    float x[V][8], s = 0.f, none = 0.f;
#pragma unroll
    for (int y = 0; y < V; ++y)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[y][j] = value<XBF>(next[y], j);
        if (own(at[y], j)) s += x[y][j];
      }
    if (m + step < a.M) fetch(m + step);
    row_totals<WAVE>(s, none, red[0], t >> 6);
    const float mean = s / (float)a.D;  // (by 1 / D a constant row's would be off its value)
    s = 0.f;
#pragma unroll
    for (int y = 0; y < V; ++y)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[y][j] -= mean;
        if (own(at[y], j)) s = __builtin_fmaf(x[y][j], x[y][j], s);
      }
    row_totals<WAVE>(s, none, red[1], t >> 6);
    const float r = 1.f / __builtin_sqrtf(s / (float)a.D + a.eps);
#pragma unroll
    for (int y = 0; y < V; ++y) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[y][j] = __builtin_fmaf(x[y][j] * r, w[y][j], b[y][j]);
      store_own<YBF, STREAM>(a.Y, m * a.sy, at[y], x[y]);
    }
    if (a.stats && t == 0) {
      a.stats[2 * m] = mean;
      a.stats[2 * m + 1] = r;
    }
  }
}

// The backward's workgroups have `teams` rows at a time, T threads each (WAVE: one), that add their sums of dw and db
// up in LDS at the end: a workgroup leaves 8 D bytes of them however many rows it has at a time.
// AHEAD: the next turn's row is loaded before this one's sums; with two vectors a thread there are no registers for it.
template <bool WAVE, int V, bool XBF, bool YBF, bool STREAM>
__global__ __launch_bounds__(1024) void norm_bwd_kernel(NormK a, int T, int teams) {
  constexpr bool AHEAD = V == 1;
  constexpr int MOST = WAVE ? 16 : V == 1 ? 8 : 1;  // teams (of 128 threads and more, or 1024)
  __shared__ float red[2][WAVE ? 1 : MOST][16][2];
  __shared__ float sums[V == 1 ? 8192 : 1];
  const int team = WAVE ? wave_uniform(threadIdx.x >> 6) : wave_uniform(threadIdx.x / (unsigned)T), t = threadIdx.x - team * T;
  if constexpr (!WAVE) {
    for (int i = threadIdx.x; i < MOST * 64; i += blockDim.x) (&red[0][0][0][0])[i] = 0.f;
    __syncthreads();
  }
  Place at[V];
  float w[V][8], dw[V][8], db[V][8];
#pragma unroll
  for (int y = 0; y < V; ++y) {
    at[y] = place_of((y * T + t) * 8, a.D);
    norm_params(a.w, a.w_bf, at[y].c, at[y].hi, 1.f, w[y]);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[y][j] = db[y][j] = 0.f;
  }
  const float inv = 1.f / (float)a.D;
  const long long step = (long long)gridDim.x * teams;
  Eight<XBF> nx[V], x[V];
  Eight<YBF> ng[V], g[V];
  float next_mean = 0.f, next_r = 0.f;
  auto fetch = [&](long long row) {
    if (row >= a.M) return;
#pragma unroll
    for (int y = 0; y < V; ++y) {
      nx[y] = load_eight<XBF, STREAM>(a.X, row * a.sx + at[y].c, at[y].hi);
      ng[y] = load_eight<YBF, STREAM>(a.dY, row * a.sdy + at[y].c, at[y].hi);
    }
    next_mean = a.stats[2 * row];
    next_r = a.stats[2 * row + 1];
  };
  if constexpr (AHEAD) fetch((long long)blockIdx.x * teams + team);
  int turn = 0;
  for (long long first = (long long)blockIdx.x * teams; first < a.M; first += step) {  // the workgroup's turns
    const long long m = first + team;
    if constexpr (!AHEAD) fetch(m);
    const float mean = next_mean, r = next_r;
#pragma unroll
    for (int y = 0; y < V; ++y) {
      x[y] = nx[y];
      g[y] = ng[y];
    }
    if constexpr (AHEAD) fetch(m + step);
    float s0 = 0.f, s1 = 0.f;
    if (m < a.M) {
#pragma unroll
      for (int y = 0; y < V; ++y)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float h = (value<XBF>(x[y], j) - mean) * r, d = own(at[y], j) ? value<YBF>(g[y], j) : 0.f, e = d * w[y][j];
          dw[y][j] = __builtin_fmaf(d, h, dw[y][j]);
          db[y][j] += d;
          s0 += e;
          s1 = __builtin_fmaf(e, h, s1);
        }
    }
    if (!a.Y) continue;
    // (red's other half is written when every thread has passed a barrier since it read this one)
    row_totals<WAVE>(s0, s1, red[turn][WAVE ? 0 : team], t >> 6);
    turn ^= 1;
    s0 *= inv;
    s1 *= inv;
    if (m < a.M) {
#pragma unroll
      for (int y = 0; y < V; ++y) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float h = (value<XBF>(x[y], j) - mean) * r;
          v[j] = r * (value<YBF>(g[y], j) * w[y][j] - s0 - h * s1);
        }
        store_own<XBF, STREAM>(a.Y, m * a.D, at[y], v);
      }
    }
  }
  if (!a.part) return;
  float* part = a.part + (long long)blockIdx.x * 2 * a.D;
  auto write = [&](float (&v)[V][8], float* to) {
    if (V == 1 && teams > 1) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (own(at[0], j)) sums[team * 8 * T + at[0].c + j] = v[0][j];
      __syncthreads();
      for (int c = threadIdx.x; c < a.D; c += blockDim.x) {
        float s = sums[c];
        for (int k = 1; k < teams; ++k) s += sums[k * 8 * T + c];
        to[c] = s;
      }
    } else {
#pragma unroll
      for (int y = 0; y < V; ++y) store_own<false, false>(to, 0, at[y], v[y]);
    }
  };
  write(dw, part);
  write(db, part + a.D);
}

// ---- rows that do not fit the registers of a workgroup -------------------------------------------------------
// Forward: a workgroup reads its row three times, from the caches as far as they hold the rows of all workgroups.  Backward: g's two
// means a row first, then workgroups of 2048 features by a share of the rows.  Forward and backward, us, and TB/s of x and y (x, dy
// and dx) once: 4096 x 20000 bf16 101 (3.2), 204 (2.4), where 16384 features take 56 (4.8), 95 (4.2) in registers; 2048 x 32768 fp32
// 163 (3.3), 274 (2.9); 512 x 2^18 fp32, 512 MB on their way, 450 (2.4), 580 (2.8); 128 rows of 2^20 bf16 417 (1.3), 662 (1.2): one
// workgroup a row leaves half of the CUs idle there.
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
constexpr int CUS = 256;
constexpr int NORM_MOST = 16384;  // features that the registers of a workgroup hold
// Bytes of x and y past which they go around the caches: 32768 x 8192 bf16 forward 191 us, 201 through them, backward 269
// and 293.  Of fewer, what comes next finds them there, and the pass itself gains less (16384 x 4096 bf16, 268 MB, 50.0 and
// 52.9 us) or loses (16384 x 1024 14.6 and 13.4).
constexpr long long NORM_STREAM = 256LL << 20;
inline long long least(long long a, long long b) { return a < b ? a : b; }

// Forward: vectors of a thread (rows of up to 1024 features are a wave's), threads, and workgroups: as many as run at
// once, no more than rows.  bf16: 16384 x 768 a workgroup a row 14.7 us, a wave 12.1 (8192 x 640 9.2 and 8.4; 16384 x 1024 15.0
// and 13.4); one vector and two: 16384 x 1500 23.3 and 25.9, 2048 27.7 and 28.9, 32768 x 2100 73.3 and 62.5, 2560 77.3 and
// 64.7, 16384 x 4000 54.9 and 54.4.  (Four: 16384 features in 512 threads.)
inline int fwd_vectors(int D) { return D <= 512 ? 1 : D <= 1024 ? 2 : D <= 2048 ? 1 : D <= 8192 ? 2 : 4; }
inline int fwd_threads(int D) { return D <= 1024 ? 256 : 64 * ceil_div(D, 512 * fwd_vectors(D)); }
inline int fwd_groups(long long M, int D) {
  if (D > NORM_MOST) return (int)least(M, 2 * CUS);
  return (int)least(D <= 1024 ? (M + 3) / 4 : M, 2048 / fwd_threads(D) * CUS);
}
// Backward: threads of a row (up to 512 features are a wave's), its teams (fewer where rows are: every CU has some),
// and workgroups, one a CU, or two where half a CU's threads are enough for one (8192 x 5000 bf16: 56 us, 64 with one).
// Teams against workgroups of one each, as many threads a CU: 16384 x 1024 26 us and 39, 8192 x 640 15.9 and 25.8,
// 32768 x 2560 91 and 93.
inline int bwd_threads(int D) { return D > 8192 ? 1024 : 64 * ceil_div(D, 512); }
inline int bwd_teams(long long M, int D) { return (int)least(1024 / bwd_threads(D), (M + CUS - 1) / CUS); }
inline int bwd_groups(long long M, int D) {
  if (D > NORM_MOST) return (int)least(M, 64);
  const int teams = bwd_teams(M, D);
  return (int)least((M + teams - 1) / teams, bwd_threads(D) * teams <= 768 ? 2 * CUS : CUS);
}

template <bool WAVE, int V, bool XBF, bool YBF, bool STREAM>
int launch_fwd_as(const NormK& k, hipStream_t s) {
  GL_LAUNCH(GL_KERNEL_NORM, (norm_fwd_kernel<WAVE, V, XBF, YBF, STREAM>), dim3((unsigned)fwd_groups(k.M, k.D)),
            dim3((unsigned)fwd_threads(k.D)), 0, s, k);
  GL_CHECK_LAUNCH();
  return 0;
}
template <bool WAVE, int V, bool XBF, bool YBF, bool STREAM>
int launch_bwd_as(const NormK& k, hipStream_t s) {
  const int T = bwd_threads(k.D), teams = bwd_teams(k.M, k.D);
  GL_LAUNCH(GL_KERNEL_NORM_BWD, (norm_bwd_kernel<WAVE, V, XBF, YBF, STREAM>), dim3((unsigned)bwd_groups(k.M, k.D)),
            dim3((unsigned)(T * teams)), 0, s, k, T, teams);
  GL_CHECK_LAUNCH();
  return 0;
}
template <bool BWD, bool XBF, bool YBF, bool STREAM>
int launch_norm_rows(const NormK& k, hipStream_t s) {
  if constexpr (BWD) {
    if (k.D <= 512) return launch_bwd_as<true, 1, XBF, YBF, STREAM>(k, s);
    if (k.D <= 8192) return launch_bwd_as<false, 1, XBF, YBF, STREAM>(k, s);
    return launch_bwd_as<false, 2, XBF, YBF, STREAM>(k, s);
  } else {
    if (k.D <= 512) return launch_fwd_as<true, 1, XBF, YBF, STREAM>(k, s);
    if (k.D <= 1024) return launch_fwd_as<true, 2, XBF, YBF, STREAM>(k, s);
    if (k.D <= 2048) return launch_fwd_as<false, 1, XBF, YBF, STREAM>(k, s);
    if (k.D <= 8192) return launch_fwd_as<false, 2, XBF, YBF, STREAM>(k, s);
    return launch_fwd_as<false, 4, XBF, YBF, STREAM>(k, s);
  }
}
template <bool BWD, bool XBF, bool YBF>
int launch_norm_of(const NormK& k, float* means, hipStream_t s) {
  if (k.D <= NORM_MOST) {
    const bool stream = k.M * k.D * ((XBF ? 2 : 4) + (YBF ? 2 : 4)) > NORM_STREAM;
    return stream ? launch_norm_rows<BWD, XBF, YBF, true>(k, s) : launch_norm_rows<BWD, XBF, YBF, false>(k, s);
  }
  const unsigned groups = (unsigned)(BWD ? bwd_groups(k.M, k.D) : fwd_groups(k.M, k.D));
  if constexpr (BWD) {
    if (k.Y) {
      GL_LAUNCH(GL_KERNEL_NORM_BWD, (norm_wide_kernel<XBF, YBF, true>), dim3((unsigned)least(k.M, 2 * CUS)), dim3(WIDE_T), 0, s,
                k, means);
      GL_CHECK_LAUNCH();
    }
    GL_LAUNCH(GL_KERNEL_NORM_BWD, (norm_wide_dx_kernel<XBF, YBF>), dim3(groups, (unsigned)ceil_div(k.D, 2048)),
              dim3(256), 0, s, k, (const float*)means);
  } else {
    GL_LAUNCH(GL_KERNEL_NORM, (norm_wide_kernel<XBF, YBF, false>), dim3(groups), dim3(WIDE_T), 0, s, k, means);
  }
  GL_CHECK_LAUNCH();
  return 0;
}
template <bool BWD>
int launch_norm(const NormK& k, int x_dtype, int y_dtype, float* means, hipStream_t s) {
  const bool y = y_dtype == GL_DTYPE_BF16;
  if (x_dtype == GL_DTYPE_BF16)
    return y ? launch_norm_of<BWD, true, true>(k, means, s) : launch_norm_of<BWD, true, false>(k, means, s);
  return y ? launch_norm_of<BWD, false, true>(k, means, s) : launch_norm_of<BWD, false, false>(k, means, s);
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
  return part_bytes(a) + (a->D > NORM_MOST && a->dX ? (size_t)round_up(a->M * 8, 256) : 0);
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
  return launch_norm<false>(k, a->x_dtype, a->y_dtype, nullptr, (hipStream_t)stream);
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
  GL_TRY(launch_norm<true>(k, a->x_dtype, a->dy_dtype, (float*)((char*)a->ws + part), s));
  if (part) {
    GL_LAUNCH(GL_KERNEL_NORM_DW, norm_dw_kernel, dim3((unsigned)ceil_div(2LL * a->D, 64)), dim3(1024), 0, s,
              (const float*)k.part, groups, a->D, a->dweight, a->dbias, (int)(a->g_dtype == GL_DTYPE_BF16), a->accumulate);
    GL_CHECK_LAUNCH();
  }
  return 0;
}
