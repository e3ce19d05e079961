// The dense products: C[m, n] = sum_r P(m, r) Q(n, r) with an epilogue, on MFMA tiles.
//
// Three products make a projection and its backward:
//     Y  = X W^T     P = X  [M, K], Q = W  [N, K]    both with the reduction along a row ("RC")
//     dX = dz W      P = dz [M, N], Q = W  [N, K]    Q with the reduction along its rows ("RS")
//     dW = dz^T X    P = dz [M, N], Q = X  [M, K]    both RS
// and one kernel computes them: an RC operand's fragments are 16-byte LDS reads, an RS operand's go
// through the transposing LDS read (bf16) or are read value by value (fp32), so no operand is
// transposed in memory.
#pragma once

#include "gl_internal.h"
#include "gl_pack8.h"

namespace gl {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

// Bytes of the reduction a stage holds per row: 64 bf16 or 32 fp32.
constexpr int DENSE_BK = 128;

// What becomes of a product's sums.
struct DenseEpi {
  const void* bias;  // operands' type, or null
  const void* res;   // or null
  long long sr;
  void* C;
  long long sc;
  void* z;           // what is kept of z (GL_KEEP_*)
  uint8_t* ze;
  long long M;
  int N;
  int act, keep;
  int op_bf, res_bf, c_bf;  // types are bf16 (else fp32)
  int accumulate;           // C (fp32) is added to
};

struct DenseK {
  const void* P;
  const void* Q;
  long long ldp, ldq;  // bytes between rows
  long long R;         // reduction; behind it an RC operand's rows have zeros up to 16 bytes
  int tiles_m, tiles_n;
  int steps, steps_per_split;  // stages of DENSE_BK bytes
  float* part;                 // split products: sums [split][M][N], joined by dense_join_kernel
  DenseEpi e;
};

// ---- epilogue ------------------------------------------------------------------------------------
__device__ __forceinline__ float gelu_f(float z) { return 0.5f * z * (1.f + erff(z * 0.70710678118654752f)); }
__device__ __forceinline__ float act_rt(int act, float z) {
  return act == GL_ACT_RELU ? __builtin_fmaxf(z, 0.f) : (act == GL_ACT_GELU ? gelu_f(z) : z);
}

// four neighbours of a row, of which the first n are there
__device__ __forceinline__ void load4(const void* p, bool bf, long long i, int n, float (&v)[4]) {
  if (n >= 4) {
    if (bf) {
      const uv2 w = reinterpret_cast<const bytes8*>((const char*)p + 2 * i)->v;
      v[0] = __uint_as_float(w[0] << 16);
      v[1] = __uint_as_float(w[0] & 0xffff0000u);
      v[2] = __uint_as_float(w[1] << 16);
      v[3] = __uint_as_float(w[1] & 0xffff0000u);
    } else {
      const uv4 w = reinterpret_cast<const bytes16*>((const char*)p + 4 * i)->v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(w[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < n ? ld_param((const float*)p, bf, i + j) : 0.f;
  }
}
__device__ __forceinline__ void store4(void* p, bool bf, long long i, int n, const float (&v)[4]) {
  if (n >= 4) {
    if (bf) {
      uv2 w;
      w[0] = to_bf16x2(v[0], v[1]);
      w[1] = to_bf16x2(v[2], v[3]);
      reinterpret_cast<bytes8*>((char*)p + 2 * i)->v = w;
    } else {
      uv4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(v[j]);
      reinterpret_cast<bytes16*>((char*)p + 4 * i)->v = w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) {
        if (bf) ((unsigned short*)p)[i + j] = to_bf16(v[j]);
        else ((float*)p)[i + j] = v[j];
      }
  }
}

// The sums v of columns n..n + 3 of row m (n a multiple of 4).  Eight neighbouring lanes hold the 32
// columns of a block, and all of them call this, whatever m and n.
__device__ __forceinline__ void dense_epilogue(const DenseEpi& e, long long m, int n, float (&v)[4]) {
  const bool in = m < e.M && n < e.N;
  if (e.bias) {
    float b[4];
    load4(e.bias, e.op_bf, n, e.N - n, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += b[j];
  }
  if (e.keep == GL_KEEP_SIGN) {
    unsigned w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < e.N && v[j] > 0.f) w |= 1u << ((n & 31) + j);
    w |= (unsigned)__shfl_xor((int)w, 1);
    w |= (unsigned)__shfl_xor((int)w, 2);
    w |= (unsigned)__shfl_xor((int)w, 4);
    if (in && (n & 31) == 0) ((unsigned*)e.z)[m * ((e.N + 31) / 32) + n / 32] = w;
  } else if (e.keep == GL_KEEP_Z) {
    if (in) store4(e.z, e.op_bf, m * ((e.N + 7) / 8 * 8) + n, e.N - n, v);
  } else if (e.keep == GL_KEEP_Z8) {
    const int nblk = (e.N + 31) / 32;
    unsigned a = 0;
    float t[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      t[j] = n + j < e.N ? v[j] : 0.f;
      a = umax(a, abs_bits(t[j]));
    }
    a = umax(a, (unsigned)__shfl_xor((int)a, 1));
    a = umax(a, (unsigned)__shfl_xor((int)a, 2));
    a = umax(a, (unsigned)__shfl_xor((int)a, 4));
    const int ex = p8_exp(a);
    if (m < e.M && n < nblk * 32) {
      *(unsigned*)((uint8_t*)e.z + (m * nblk * 32 + n)) = p8_codes4(t[0], t[1], t[2], t[3], p8_inv_step(ex));
      if ((n & 31) == 0) e.ze[m * nblk + n / 32] = (uint8_t)ex;
    }
  }
  if (!in) return;
  if (e.act != GL_ACT_IDENTITY) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = act_rt(e.act, v[j]);
  }
  float r[4];
  if (e.res) {
    load4(e.res, e.res_bf, m * e.sr + n, e.N - n, r);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += r[j];
  }
  if (e.accumulate) {
    load4(e.C, false, m * e.sc + n, e.N - n, r);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += r[j];
  }
  store4(e.C, e.c_bf, m * e.sc + n, e.N - n, v);
}

// ---- the tile kernel -------------------------------------------------------------------------------
// Block -> tile.  The 8 XCDs take consecutive workgroups in turn and have an L2 each, so XCD x gets the
// x-th contiguous share of the tiles; inside it tiles go in columns of GROUP_M, which keeps the share's
// running workgroups on few distinct rows of either operand.
constexpr int GROUP_M = 8;
__device__ __forceinline__ void tile_of(int bid, int nblk, int tiles_m, int tiles_n, int& tm, int& tn, int& split) {
  const int x = bid & 7, q = nblk >> 3, r = nblk & 7;
  int id = x * q + (x < r ? x : r) + (bid >> 3);
  const int per = tiles_m * tiles_n;
  split = id / per;
  id -= split * per;
  const int band = GROUP_M * tiles_n, b = id / band, m0 = b * GROUP_M;
  const int h = tiles_m - m0 < GROUP_M ? tiles_m - m0 : GROUP_M;
  id -= b * band;
  tn = id / h;
  tm = m0 + id - tn * h;
}

// 16 bytes per lane straight from a buffer into LDS at (wave-uniform) lds + 16 lane; offsets at or past
// the buffer's size put zeros there.  Issued from asm so that the compiler's own waits do not count it:
// the caller waits with stage_wait() and a barrier before the data is read.
__device__ __forceinline__ void dma16(unsigned off, i32x4 rsrc, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :: "v"(off), "s"(rsrc), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ i32x4 buffer_of(const char* p, long long bytes) {
  const unsigned long long a = (unsigned long long)p;
  const unsigned n = bytes <= 0 ? 0u : (bytes > 0x7fffffffLL ? 0x7fffffffu : (unsigned)bytes);
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(unsigned)a);
  r[1] = __builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32) & 0xffff);
  r[2] = __builtin_amdgcn_readfirstlane((int)n);
  r[3] = 0x00020000;
  return r;
}
constexpr unsigned DMA_NOWHERE = 0x80000000u;  // past any buffer_of

// One operand's side of a tile: DIM rows of the output (RC) or columns (RS) by DENSE_BK bytes of
// reduction, staged by NW waves.
//
// LDS of an RC operand: rows of 128 bytes, 16-byte chunk c of row r at c ^ (r & 7), so that the 32 rows
// of a fragment's read fall on all banks.  Of an RS operand: the reduction's rows of DIM values; for
// bf16 the 32-byte unit u of row r at u ^ swz(r): a transposing read takes 32 bytes of four rows r..r + 3
// (two such groups per half wave, of neighbouring units), and the swizzle puts those on all banks.
template <int ES, int DIM, int NW, bool RC>
struct Side {
  static constexpr int BYTES = DIM * DENSE_BK;
  static constexpr int LOADS = BYTES / 1024 / NW;  // of one wave and stage
  static constexpr int RROWS = DENSE_BK / ES;      // rows of an RS stage
  static constexpr int PITCH = DIM * ES;
  static_assert(LOADS * NW * 1024 == BYTES, "whole loads");

  const char* p;
  long long ld, left;  // bytes: of a row; from p to the operand's end
  unsigned off[LOADS];
  int k_lane;  // RC: this lane's first byte of the reduction in a stage
  long long rbytes;

  static __device__ __forceinline__ int swz(int r) {
    if constexpr (ES == 2) return (((r & 3) << 1) | (((r >> 3) & 1) << 3)) & (DIM / 16 - 1);
    return 0;
  }

  // base: the operand; first: the tile's first row (RC) or column (RS); dim, R: the operand's size
  __device__ __forceinline__ void init(const void* base, long long ldb, long long first, long long dim, long long R,
                                       int step0) {
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    // Ends are taken up to 16 bytes: a buffer checks whole words, and the 16 bytes that hold an element
    // of a 16-byte-aligned row are there (zeros behind an RC row's end, columns that nobody stores
    // behind an RS row's).
    ld = ldb;
    rbytes = (R * ES + 15) & ~15LL;
    if constexpr (RC) {
      p = (const char*)base + first * ld + (long long)step0 * DENSE_BK;
      left = (dim - 1 - first) * ld + rbytes - (long long)step0 * DENSE_BK;
      rbytes -= (long long)step0 * DENSE_BK;
      k_lane = ((l & 7) ^ (l >> 3)) * 16;
#pragma unroll
      for (int t = 0; t < LOADS; ++t) off[t] = (unsigned)((t * NW + w) * 8 + (l >> 3)) * (unsigned)ld + k_lane;
    } else {
      p = (const char*)base + (long long)step0 * RROWS * ld + first * ES;
      left = (R - 1 - (long long)step0 * RROWS) * ld + (((dim - first) * ES + 15) & ~15LL);
      constexpr int SPR = PITCH / 16;
#pragma unroll
      for (int t = 0; t < LOADS; ++t) {
        const int s = (t * NW + w) * 64 + l, r = s / SPR, c = s % SPR;
        off[t] = (unsigned)r * (unsigned)ld + (((c >> 1) ^ swz(r)) * 2 + (c & 1)) * 16;
      }
    }
  }
  // issue the loads of the next stage into LDS at `lds` and step on
  __device__ __forceinline__ void issue(unsigned lds) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const i32x4 b = buffer_of(p, left);
#pragma unroll
    for (int t = 0; t < LOADS; ++t) {
      unsigned o = off[t];
      if constexpr (RC) o = k_lane < rbytes ? o : DMA_NOWHERE;
      dma16(o, b, lds + (t * NW + w) * 1024);
    }
    if constexpr (RC) {
      p += DENSE_BK;
      left -= DENSE_BK;
      rbytes -= DENSE_BK;
    } else {
      p += RROWS * ld;
      left -= RROWS * ld;
    }
  }
};

// A lane's part of a 32-row fragment: row l % 32, and of the 32 bytes of reduction at kk * 32 the half l / 32.
template <int ES> struct Frag;
template <> struct Frag<2> {
  bf16x8 v;
};
template <> struct Frag<4> {
  f32x4 v;
};

template <int ES, int DIM, bool RC>
struct Reader {
  unsigned a[4];  // RC: byte of chunk kk; RS: see at()
  unsigned col[RC ? 1 : DIM / 32];
  // base: this wave's first row / column of the tile, a multiple of 32
  __device__ __forceinline__ void init(int base) {
    const int l = threadIdx.x & 63;
    if constexpr (RC) {
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) a[kk] = (base + (l & 31)) * DENSE_BK + (((2 * kk + (l >> 5)) ^ (l & 7)) * 16);
    } else if constexpr (ES == 2) {
      const int g = l >> 4, i = l & 15, r = 8 * (g >> 1) + (i >> 2);
      const int sw = Side<ES, DIM, 1, false>::swz(r);
#pragma unroll
      for (int t = 0; t < DIM / 32; ++t)
        col[t] = r * (DIM * 2) + (((base / 16 + 2 * t + (g & 1)) ^ sw) * 32) + 8 * (i & 3);
    } else {
      col[0] = (l >> 5) * 4 * (DIM * 4) + (base + (l & 31)) * 4;
    }
  }
  __device__ __forceinline__ Frag<ES> read(const char* lds, int t, int kk) const {
    Frag<ES> f;
    if constexpr (RC) {
      f.v = *reinterpret_cast<const decltype(f.v)*>(lds + a[kk] + t * 32 * DENSE_BK);
    } else if constexpr (ES == 2) {
      typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
      union {
        i16x4 h[2];
        bf16x8 v;
      } u;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(lds + col[t] + (16 * kk + 4 * h) * (DIM * 2)));
      f.v = u.v;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f.v[e] = *reinterpret_cast<const float*>(lds + col[0] + (8 * kk + e) * (DIM * 4) + t * 128);
    }
    return f;
  }
};

// rows of the output are Q's (n), its columns P's (m): a lane then holds neighbours of a row of C
__device__ __forceinline__ f32x16 mma(const Frag<2>& q, const Frag<2>& p, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(q.v, p.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(const Frag<4>& q, const Frag<4>& p, f32x16 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(q.v[e], p.v[e], c, 0, 0, 0);
  return c;
}

template <int ES, int BM, int BN, int WM, int WN, bool PRC, bool QRC>
__global__ __launch_bounds__(64 * WM * WN) void dense_tile_kernel(DenseK a) {
  constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
  typedef Side<ES, BM, NW, PRC> SP;
  typedef Side<ES, BN, NW, QRC> SQ;
  constexpr int STAGE = SP::BYTES + SQ::BYTES;
  extern __shared__ __align__(1024) char smem[];
  int tm, tn, split;
  tile_of(blockIdx.x, gridDim.x, a.tiles_m, a.tiles_n, tm, tn, split);
  const int k0 = split * a.steps_per_split;
  const int nk = min(a.steps - k0, a.steps_per_split);
  const long long m0 = (long long)tm * BM;
  const int n0 = tn * BN;
  const int w = threadIdx.x >> 6, wm = w / WN, wn = w % WN;

  SP sp;
  SQ sq;
  sp.init(a.P, a.ldp, m0, a.e.M, a.R, k0);
  sq.init(a.Q, a.ldq, n0, a.e.N, a.R, k0);
  Reader<ES, BM, PRC> rp;
  Reader<ES, BN, QRC> rq;
  rp.init(wm * TM * 32);
  rq.init(wn * TN * 32);
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;

  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int x = 0; x < 16; ++x) acc[i][j][x] = 0.f;

  sp.issue(lds0);
  sq.issue(lds0 + SP::BYTES);
  for (int k = 0; k < nk; ++k) {
    const unsigned cur = (k & 1) * STAGE, nxt = STAGE - cur;
    stage_wait();
    __syncthreads();
    if (k + 1 < nk) {
      sp.issue(lds0 + nxt);
      sq.issue(lds0 + nxt + SP::BYTES);
    }
    const char* lp = smem + cur;
    const char* lq = lp + SP::BYTES;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      Frag<ES> fp[TM], fq[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) fp[i] = rp.read(lp, i, kk);
#pragma unroll
      for (int j = 0; j < TN; ++j) fq[j] = rq.read(lq, j, kk);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mma(fq[j], fp[i], acc[i][j]);
    }
  }

  // The sums go through LDS, 32 rows of the wave's 64 columns at a time, so that a lane gets 4 neighbours
  // of a row, 16 lanes a whole row (128 bytes of bf16), and the epilogue is a rolled loop.  Rows are 68
  // floats apart: 16 rows of a store then fall on all banks.
  static_assert(TN == 2 && NW * 32 * 68 * 4 <= 2 * STAGE, "a wave's rows of 64 columns");
  __syncthreads();
  const int l = threadIdx.x & 63;
  float* own = reinterpret_cast<float*>(smem) + w * 32 * 68;
  float* part = a.part ? a.part + (long long)split * a.e.M * a.e.N : nullptr;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 t;
#pragma unroll
        for (int x = 0; x < 4; ++x) t[x] = acc[i][j][4 * g + x];
        *reinterpret_cast<f32x4*>(own + (l & 31) * 68 + 32 * j + 8 * g + 4 * (l >> 5)) = t;
      }
    const int n = n0 + wn * 64 + (l & 15) * 4;
#pragma unroll 1
    for (int r = l >> 4; r < 32; r += 4) {
      const long long m = m0 + (wm * TM + i) * 32 + r;
      const f32x4 t = *reinterpret_cast<const f32x4*>(own + r * 68 + (l & 15) * 4);
      float v[4] = {t[0], t[1], t[2], t[3]};
      if (part) {
        if (m < a.e.M && n < a.e.N) store4(part, false, m * a.e.N + n, a.e.N - n, v);
      } else {
        dense_epilogue(a.e, m, n, v);
      }
    }
  }
}

// ---- host side ---------------------------------------------------------------------------------------
enum { DENSE_NT = 0, DENSE_NN = 1, DENSE_TN = 2 };  // P, Q: RC RC; RC RS; RS RS
enum { DENSE_256 = 0, DENSE_128 = 1, DENSE_64 = 2, DENSE_TILES = 3 };
constexpr int DENSE_BM[DENSE_TILES] = {256, 128, 64}, DENSE_BN[DENSE_TILES] = {256, 128, 128};

template <int ES, int BM, int BN, int WM, int WN, bool PRC, bool QRC>
int launch_dense_tile_as(const DenseK& a, int splits, hipStream_t s) {
  constexpr size_t lds = 2 * (BM + BN) * DENSE_BK;
  const void* f = (const void*)dense_tile_kernel<ES, BM, BN, WM, WN, PRC, QRC>;
  GL_TRY(set_lds_limit(f, lds));
  GL_LAUNCH(GL_KERNEL_DENSE, (dense_tile_kernel<ES, BM, BN, WM, WN, PRC, QRC>),
            dim3((unsigned)(a.tiles_m * a.tiles_n * splits)), dim3(64 * WM * WN), lds, s, a);
  GL_CHECK_LAUNCH();
  return 0;
}
template <int ES, int BM, int BN, int WM, int WN>
int launch_dense_tile_of(int form, const DenseK& a, int splits, hipStream_t s) {
  if (form == DENSE_NT) return launch_dense_tile_as<ES, BM, BN, WM, WN, true, true>(a, splits, s);
  if (form == DENSE_NN) return launch_dense_tile_as<ES, BM, BN, WM, WN, true, false>(a, splits, s);
  return launch_dense_tile_as<ES, BM, BN, WM, WN, false, false>(a, splits, s);
}
int launch_dense_tile_bf16(int form, int tile, const DenseK& a, int splits, hipStream_t s);
int launch_dense_tile_f32(int form, int tile, const DenseK& a, int splits, hipStream_t s);

// few rows (gl_dense_few.hip): the forward of up to DENSE_FEW_ROWS rows that keeps nothing
constexpr int DENSE_FEW_ROWS = 64;
int launch_dense_few(const GlDenseArgs* a, const DenseEpi& e, hipStream_t s);

}  // namespace gl
