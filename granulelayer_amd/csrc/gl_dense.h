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

#include <atomic>

#include "gl_internal.h"
#include "gl_pack8.h"

namespace gl {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

// Bytes of reduction of a stage: a cache line of an RC row (half lines are fetched twice), 64 bf16 or 32 fp32.
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
  int steps, steps_per_split;  // stages
  float* part;                 // split products: sums [split][M][N], joined by dense_join_kernel
  DenseEpi e;
};

// What a product's kernel does besides: nothing; take the number of its rows (of C, or where both operands
// are RS of the reduction) and a factor from device memory; and the two products of the softmax cross entropy, logits = X W^T
// of a piece of the classes, that leave a tile's softmax statistics or their gradient and no logits (gl_ce.hip).
enum { DENSE_PLAIN, DENSE_ROWS, DENSE_CE_STATS, DENSE_CE_GRAD };
struct DenseRowsK : DenseK {
  const int* rows;           // or null: as the sizes say
  const float* alpha;        // DENSE_ROWS: factor of the product, or null: 1
  // statistics
  const long long* target;
  const int* index;          // row of `target` of every row of X, or null: its own
  float* target_logit;       // [M]; like all logits behind the product in units of log 2
  float* stats;              // [M][tiles_n][2]: the tile's largest logit but the target's, and the sum of 2^(logit - it)
  void* exps;                // 2^(logit - the largest of its row's 64 columns) of the columns below exps_cols (16 bits of bf16
  float* exps_top;           // operands: exp_code; else fp32; rows of padded(exps_cols), zeros behind the last and at the target), and
  int exps_cols;             // these largest [M][ceil(exps_cols / 64)]; or null
  // gradient
  const uv4* row_info;       // [M]: the largest logit; factor of 2^(logit - it); the target; the gradient at it
  int first;                 // class of the product's first column
  float* col_sums;           // [tiles_m * waves along m][N], or null
  int pitch;                 // of C's rows; columns from N to there are zeros
};
template <int KIND> struct DenseArgs { typedef DenseRowsK type; };
template <> struct DenseArgs<DENSE_PLAIN> { typedef DenseK type; };

// ---- activations -----------------------------------------------------------------------------------
// GELU from the normal distribution's upper tail: with a = |z| and Q(a) = 1 - Phi(a),
//     gelu(z) = max(z, 0) - a Q(a)
// and Q(a) = 2^R(a): log2 of the tail is smooth, and a polynomial of degree 8, fitted on [0, 8] by least squares
// weighted with a Q(a), leaves 1.3e-8 in a Q(a) with its coefficients in fp32.  That weight evens out the absolute error:
// evaluated in fp32 gelu is within 2.5e-7 of the exact values over [-14, 14] (the last place of z near 4), and within 5e-8
// for z < 0.  Relative to gelu the tail is off by 2e-5 down to z = -4, 0.4% at -5, 5% at -6 and 84% at -8, where
// gelu is -5e-15; 1 + erf in fp32 cancels there (5e-4 at -4, 5% at -5, nothing left from about -5.5).  Below -8, at -inf
// too, the result stays at -8e-16.  15 instruction slots, against about 40 with erff.
// max(z, 0) by comparison: NaN stays NaN.
__device__ __forceinline__ float upper_tail(float a) {
  float r = -1.8003542e-06f;
  r = __builtin_fmaf(r, a, 2.66367551e-05f);
  r = __builtin_fmaf(r, a, -0.00012340954f);
  r = __builtin_fmaf(r, a, -0.000296153215f);
  r = __builtin_fmaf(r, a, 0.00728624407f);
  r = __builtin_fmaf(r, a, -0.0526671633f);
  r = __builtin_fmaf(r, a, -0.459141284f);
  r = __builtin_fmaf(r, a, -1.15111637f);
  r = __builtin_fmaf(r, a, -0.999999523f);
  return __builtin_amdgcn_exp2f(r);
}
__device__ __forceinline__ float relu_f(float z) { return z < 0.f ? 0.f : z; }
__device__ __forceinline__ float gelu_f(float z) {
  const float a = __builtin_fminf(__builtin_fabsf(z), 8.f);
  return __builtin_fmaf(-a, upper_tail(a), relu_f(z));
}
// gelu'(z) = D(a) for z < 0 and 1 - D(a) else, D(a) = Q(a) - a phi(a) = exp(-a^2 / 2) P(a): P of degree 10, by
// least squares weighted with the exponential, leaves 8e-8 on [0, 6.5], and D(6.5) is below 2e-9; within 1.7e-7 in
// fp32.  One exponential, 18 slots.
__device__ __forceinline__ float dgelu_f(float z) {
  const float m = __builtin_fabsf(z), a = m > 6.5f ? 6.5f : m;  // NaN stays
  float p = 1.63169273e-06f;
  p = __builtin_fmaf(p, a, -3.5207835e-05f);
  p = __builtin_fmaf(p, a, 0.000339738821f);
  p = __builtin_fmaf(p, a, -0.00197462901f);
  p = __builtin_fmaf(p, a, 0.00793939456f);
  p = __builtin_fmaf(p, a, -0.024313936f);
  p = __builtin_fmaf(p, a, 0.0611548908f);
  p = __builtin_fmaf(p, a, -0.132513806f);
  p = __builtin_fmaf(p, a, 0.249916792f);
  p = __builtin_fmaf(p, a, -0.797878802f);
  p = __builtin_fmaf(p, a, 0.49999994f);
  const float d = p * __builtin_amdgcn_exp2f(a * a * -0.72134752f);
  return z < 0.f ? d : 1.f - d;
}
__device__ __forceinline__ float act_rt(int act, float z) {
  return act == GL_ACT_RELU ? relu_f(z) : (act == GL_ACT_GELU ? gelu_f(z) : z);
}

// ---- epilogue ------------------------------------------------------------------------------------
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
typedef unsigned uv4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned uv2_any __attribute__((ext_vector_type(2), aligned(2)));
// STREAM: a hint that the caches need not keep it
template <bool STREAM = false>
__device__ __forceinline__ void store4(void* p, bool bf, long long i, int n, const float (&v)[4]) {
  if (n >= 4) {
    if (bf) {
      uv2 w;
      w[0] = to_bf16x2(v[0], v[1]);
      w[1] = to_bf16x2(v[2], v[3]);
      if constexpr (STREAM) __builtin_nontemporal_store(w, reinterpret_cast<uv2_any*>((char*)p + 2 * i));
      else reinterpret_cast<bytes8*>((char*)p + 2 * i)->v = w;
    } else {
      uv4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(v[j]);
      if constexpr (STREAM) __builtin_nontemporal_store(w, reinterpret_cast<uv4_any*>((char*)p + 4 * i));
      else reinterpret_cast<bytes16*>((char*)p + 4 * i)->v = w;
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

// Over the eight lanes that share 32 columns: neighbours, pairs, then the halves of the eight.
template <typename OP>
__device__ __forceinline__ unsigned over8(unsigned v, OP op) {
  v = op(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));   // lane ^ 1
  v = op(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));   // lane ^ 2
  v = op(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));  // 7 - lane: the other four
  return v;
}

// What is kept of z and the activation, for the sums v of columns n..n + 3 (n a multiple of 4) of the G rows m,
// m + dm, ..., to which the bias b is added.  Eight neighbouring lanes hold the 32 columns of a block, and all of
// them call this, whatever m and n.  Choices are made for all rows at once.
template <int G>
__device__ __forceinline__ void dense_forward(const DenseEpi& e, long long m, int dm, int n, float (&v)[G][4],
                                              const float (&b)[4]) {
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[g][j] += b[j];
  const int there = e.N - n, nblk = (e.N + 31) / 32;
  if (e.keep == GL_KEEP_SIGN) {
    unsigned* z = (unsigned*)e.z + m * nblk + n / 32;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      unsigned w = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < there && v[g][j] > 0.f) w |= 1u << j;
      w = over8(w << (n & 31), [](unsigned x, unsigned y) { return x | y; });
      if (m + g * dm < e.M && there > 0 && (n & 31) == 0) z[(long long)g * dm * nblk] = w;
    }
  } else if (e.keep == GL_KEEP_Z) {
    const long long ldz = (e.N + 7) / 8 * 8;  // rows have room to 8
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (m + g * dm < e.M && there > 0) store4(e.z, e.op_bf, (m + g * dm) * ldz + n, 4, v[g]);
  } else if (e.keep == GL_KEEP_Z8) {
    uint8_t* z = (uint8_t*)e.z + (m * nblk * 32 + n);
    uint8_t* ze = e.ze + (m * nblk + n / 32);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float t[4];
      unsigned a = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        t[j] = j < there ? v[g][j] : 0.f;
        a = umax(a, abs_bits(t[j]));
      }
      a = over8(a, [](unsigned x, unsigned y) { return umax(x, y); });
      const int ex = p8_exp(a);
      const unsigned q = p8_codes4(t[0], t[1], t[2], t[3], p8_inv_step(ex));
      if (m + g * dm < e.M && n < nblk * 32) {
        *(unsigned*)(z + (long long)g * dm * nblk * 32) = q;
        if ((n & 31) == 0) ze[(long long)g * dm * nblk] = (uint8_t)ex;
      }
    }
  }
  if (e.act == GL_ACT_GELU) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[g][j] = gelu_f(v[g][j]);
  } else if (e.act == GL_ACT_RELU) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[g][j] = relu_f(v[g][j]);
  }
}
__device__ __forceinline__ void dense_bias(const DenseEpi& e, int n, float (&b)[4]) {
  if (e.bias) load4(e.bias, e.op_bf, n, e.N - n, b);
  else b[0] = b[1] = b[2] = b[3] = 0.f;
}
// What is added last, as it is stored: the residual, or the gradient that C accumulates.
struct Added {
  const char* p;
  long long step;  // bytes of a row
  bool bf;
};
__device__ __forceinline__ Added dense_added(const DenseEpi& e) {
  if (e.res) return {(const char*)e.res, e.sr * (e.res_bf ? 2 : 4), e.res_bf != 0};
  if (e.accumulate) return {(const char*)e.C, e.sc * 4, false};
  return {nullptr, 0, false};
}
__device__ __forceinline__ uv4 load_added(const char* p, bool bf, int n) {
  uv4 v = {0u, 0u, 0u, 0u};
  if (n >= 4) {
    if (bf) {
      const uv2 w = reinterpret_cast<const bytes8*>(p)->v;
      v[0] = w[0];
      v[1] = w[1];
    } else {
      v = reinterpret_cast<const bytes16*>(p)->v;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < n) {
        if (bf) v[j >> 1] |= (unsigned)((const unsigned short*)p)[j] << (16 * (j & 1));
        else v[j] = ((const unsigned*)p)[j];
      }
  }
  return v;
}
__device__ __forceinline__ void add_added(float (&v)[4], uv4 r, bool bf) {
  v[0] += __uint_as_float(bf ? r[0] << 16 : r[0]);
  v[1] += __uint_as_float(bf ? r[0] & 0xffff0000u : r[1]);
  v[2] += __uint_as_float(bf ? r[1] << 16 : r[2]);
  v[3] += __uint_as_float(bf ? r[1] & 0xffff0000u : r[3]);
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
// the buffer's size put zeros there.  Issued from asm so that the compiler's own waits do not count it: the
// kernel waits with copies_barrier(), which is also what keeps reads of the data behind it.  (No clobber of
// memory here: nothing reads these bytes before that barrier, and fragments' reads may move past the copy.)
__device__ __forceinline__ void dma16(unsigned off, i32x4 rsrc, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :: "v"(off), "s"(rsrc), "s"(lds) : "m0");
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
constexpr unsigned DMA_NOWHERE = 0x80000000u;  // past any buffer_of; offsets are below

// One operand's side of a tile: DIM rows of the output (RC) or columns (RS) by DENSE_BK bytes of reduction,
// staged by NW waves.
//
// LDS of an RC operand: rows of 128 bytes, 16-byte chunk c of row r at c ^ key(r).  A 16-byte read of 16
// neighbouring rows takes each of the 16 chunks of a 256-byte bank row once: LDS then delivers 256 bytes a clock
// (half of it with c ^ (r & 7): rows r and r + 8 collide).  Of an RS operand: the reduction's rows of DIM values, the
// 32-byte unit u of row r at u ^ swz(r).  bf16: a transposing read takes 32 bytes of four rows r..r + 3, and in each half
// wave the same of rows 8 further on, or the next unit of these; fp32: 16 values of rows 4 apart.  The swizzle
// puts them on all banks.
template <int ES, int DIM, int NW, bool RC>
struct Side {
  static constexpr int BK = DENSE_BK;
  static constexpr int BYTES = DIM * BK;
  static constexpr int LOADS = BYTES / 1024 / NW;  // of one wave and stage
  static constexpr int RROWS = BK / ES;            // rows of an RS stage
  static constexpr int PITCH = DIM * ES;
  static constexpr int CPR = BK / 16;
  static_assert(LOADS * NW * 1024 == BYTES && NW % 2 == 0, "whole loads; key() of a lane's rows is the wave's");

  const char* p;
  long long ld, left;  // bytes: of a row; from p to the operand's end
  unsigned off[LOADS];
  int k_lane, k_left;  // RC: this lane's first byte of the reduction in a stage; the reduction's bytes from p

  static __device__ __forceinline__ int key(int r) { return (r >> 1) & 7; }
  static __device__ __forceinline__ int swz(int r) {
    if constexpr (ES == 4) return ((r >> 2) & 3) << 1;
    // (64 columns: rows r and r + 1 are in different halves of a bank row as it is)
    return DIM == 64 ? (r & 2) | ((r >> 3) & 1) : ((r & 3) << 1) | ((r >> 3) & 1);
  }

  // base: the operand; first: the tile's first row (RC) or column (RS); dim, R: the operand's size
  __device__ __forceinline__ void init(const void* base, long long ldb, long long first, long long dim, long long R,
                                       int step0) {
    const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
    // Ends are taken up to 16 bytes: a buffer checks whole words, and the 16 bytes that hold an element
    // of a 16-byte-aligned row are there (zeros behind an RC row's end, columns that nobody stores
    // behind an RS row's).
    ld = ldb;
    if constexpr (RC) {
      const long long rbytes = (R * ES + 15) & ~15LL;  // at most GL_DENSE_MAX_FEATURES values
      p = (const char*)base + first * ld + (long long)step0 * BK;
      left = (dim - 1 - first) * ld + rbytes - (long long)step0 * BK;
      k_left = (int)rbytes - step0 * BK;
      k_lane = ((l % CPR) ^ key(w * (64 / CPR) + l / CPR)) * 16;
#pragma unroll
      for (int t = 0; t < LOADS; ++t) off[t] = (unsigned)((t * NW + w) * (64 / CPR) + l / CPR) * (unsigned)ld + k_lane;
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
  // Copies of the next stage: prepare() and open() it, then copy() its parts in any order.  Stages past the
  // reduction's end are zeros.
  i32x4 rsrc, next_rsrc;
  unsigned dead, next_dead;  // RC: bit 31 where the lane's chunk is past the reduction's end
  __device__ __forceinline__ void prepare() {
    next_rsrc = buffer_of(p, left);
    const long long step = RC ? (long long)BK : RROWS * ld;
    p += step;
    left -= step;
    if constexpr (RC) {
      next_dead = k_lane < k_left ? 0u : DMA_NOWHERE;
      k_left -= BK;
    }
  }
  __device__ __forceinline__ void open() {
    rsrc = next_rsrc;
    dead = next_dead;
  }
  __device__ __forceinline__ void copy(int t, unsigned lds) const {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    dma16(RC ? off[t] | dead : off[t], rsrc, lds + (t * NW + w) * 1024);
  }
};

// A fragment: MS rows (16 or 32) of an operand by what a matrix instruction of MS x MS takes in 16 bytes a lane,
// 64 or 32 bytes of the reduction.  Lane l has row l % MS and the 16 bytes l / MS.
template <int ES> struct Frag;
template <> struct Frag<2> {
  static constexpr int STEPS = 1;  // matrix instructions
  bf16x8 v;
};
template <> struct Frag<4> {
  static constexpr int STEPS = 4;
  f32x4 v;
};

template <int ES, int MS, int DIM, bool RC>
struct Reader {
  static_assert(MS == 16 || (MS == 32 && ES == 2), "fp32 rows are read 16 at a time");
  unsigned at;  // byte of this lane's part of fragment 0, part 0
  // base: this wave's first row / column of the tile, a multiple of its rows / columns
  __device__ __forceinline__ void init(int base) {
    const int l = threadIdx.x & 63, g = l >> 4, i = l & 15;
    if constexpr (RC) {
      at = (base + l % MS) * DENSE_BK + ((l / MS ^ Side<ES, DIM, 2, true>::key(l % MS)) * 16);
    } else if constexpr (ES == 2) {
      const int r = 8 * (MS == 16 ? g : g >> 1) + (i >> 2), u = base / 16 + (MS == 16 ? 0 : g & 1);
      at = r * (DIM * 2) + (u ^ Side<ES, DIM, 2, false>::swz(r)) * 32 + 8 * (i & 3);
    } else {
      at = 4 * g * (DIM * 4) + ((base / 8 + (i >> 3)) ^ Side<ES, DIM, 2, false>::swz(4 * g)) * 32 + (i & 7) * 4;
    }
  }
  // part kk of fragment t of the wave, from the stage at LDS address lds: a step of swizzled bits is an exclusive or
  __device__ __forceinline__ Frag<ES> read(unsigned lds, int t, int kk) const {
    constexpr int PART = 1024 / MS;  // bytes of reduction
    Frag<ES> f;
    if constexpr (RC) {
      typedef const __attribute__((address_space(3))) decltype(f.v) lds_vec;
      f.v = *(lds_vec*)(((lds + at) ^ kk * PART) + t * MS * DENSE_BK);
    } else if constexpr (ES == 2) {
      typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
      union {
        i16x4 h[2];
        bf16x8 v;
      } u;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_i16x4*)(((lds + at) ^ t * MS * 2) + (PART / 2 * kk + 4 * h) * (DIM * 2)));
      f.v = u.v;
    } else {
      typedef const __attribute__((address_space(3))) float lds_float;
#pragma unroll
      for (int e = 0; e < 4; ++e) f.v[e] = *(lds_float*)(((lds + at) ^ t * 64) + (16 * kk + e) * (DIM * 4));
    }
    return f;
  }
};

// rows of the output are Q's (n), its columns P's (m): a lane then holds neighbours of a row of C.
//
// 16 x 16 or 32 x 32: an instruction of 16 x 16 reads and writes its sums for twice the products, which takes less
// power, and power sets the clock of large bf16 products: from registers alone 2,120 TFLOP/s against 1,890.  But it is
// half as long, and a wave that is alone on its SIMD has less to hide its reads behind.  16384 x 4096 over 4096 in 256 x
// 256 tiles, on the card where both were timed: 399 us against 409 (407 against 430 on one with a lower clock); 4096 x 1024
// over 4096 in 128 x 128 tiles, a wave a SIMD: 39.4 against 36.9.  fp32: 1040 against 1060 us (4096 x 4096 over 4096, NN).
__device__ __forceinline__ f32x4 mma(const Frag<2>& q, const Frag<2>& p, int, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(q.v, p.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(const Frag<2>& q, const Frag<2>& p, int, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(q.v, p.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const Frag<4>& q, const Frag<4>& p, int x, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(q.v[x], p.v[x], c, 0, 0, 0);
}
template <int MS> struct Sums { typedef f32x4 type; };  // a lane's of an instruction
template <> struct Sums<32> { typedef f32x16 type; };

// Every wave's LDS accesses and all but N of its copies done, then the workgroup's barrier.
template <int N>
__device__ __forceinline__ void copies_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Over the 64 / MS lanes that hold a row's sums.
template <int MS, typename OP>
__device__ __forceinline__ float over_row(float v, OP op) {
  if constexpr (MS == 16) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(p[0]), __uint_as_float(p[1]));
  }
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
constexpr float LOG2E = 1.44269504f;
// A bias in units of log 2.  The lowest finite one stays a number: logits of it and nothing else have a softmax.
__device__ __forceinline__ float ce_bias(float b) {
  constexpr float MOST = 3.402823466e38f;
  return __builtin_fabsf(b) <= MOST ? __builtin_amdgcn_fmed3f(b * LOG2E, -MOST, MOST) : b;
}
__device__ __forceinline__ int n_pitch(const DenseRowsK& a) { return a.pitch; }
__device__ __forceinline__ int n_pitch(const DenseK&) { return 0; }

// An exponential, between 0 and 1, in 16 bits: of an fp32 number's the lower 6 of the exponent and the upper 10 of the
// mantissa, to the nearest.  The value is off by up to 2^-11 of itself and by 2^-63 besides, which the code 0 stands for: 2^-11 relative
// down to about 2^-48, 0 from 2^-63 (fp16 is so down to 2^-14 and has nothing below 2^-25, and a class that is no target has
// its whole gradient from such), 0 from 0.  Of a NaN any code: its row's factor is NaN.
__device__ __forceinline__ unsigned exp_code(float e) {
  return __builtin_elementwise_sub_sat((__float_as_uint(e) + 0x1000u) >> 13, 0x10000u) & 0xffffu;
}
__device__ __forceinline__ float exp_value(unsigned c) { return __uint_as_float((c << 13) + 0x20000000u) - 0x1p-63f; }

// DENSE_CE_STATS: every row's largest logit of the tile and the sum of 2^(logit - it), both without the target's, and the
// target's where it is in the tile.  All from the sums' registers: a lane has MS columns of its row, the lanes of a row are joined by
// two (or one) swaps, the waves of a row through LDS (BM rows of WN pairs, free behind the caller's barrier).
// Columns behind N are -inf; a tile of nothing else has the largest logit -inf and the sum 0.  A NaN is left out of the
// largest and makes the sum NaN, as +inf does.
template <int ES, int MS, int BM, int BN, int WM, int WN, int TM, int TN>
__device__ __forceinline__ void ce_stats(const DenseRowsK& a, long long M, int tm, int tn,
                                         const typename Sums<MS>::type (&acc)[TM][TN], float (*lds)[2]) {
  constexpr int G = MS * MS / 256;  // groups of four columns in a lane's sums of an instruction
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, wm = w / WN, wn = w % WN;
  const int n0 = tn * BN + wn * 64, lane_col = 4 * (l / MS);
  const long long m0 = (long long)tm * BM;
  const bool inside = tn * BN + BN <= a.e.N;
  float bias[TN][4 * G];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float b[4];
      dense_bias(a.e, n0 + MS * j + 8 * g + lane_col, b);
#pragma unroll
      for (int x = 0; x < 4; ++x) bias[j][4 * g + x] = ce_bias(b[x]);
    }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int row = wm * TM * MS + i * MS + l % MS;
    const long long m = m0 + row;
    long long t = -1;
    if (m < M) t = a.target[a.index ? a.index[m] : m] - n0;
    const int at = t >= 0 && t < 64 ? (int)t - lane_col : -64;  // of this lane's columns
    float v[TN][4 * G], top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int x = 0; x < 4 * G; ++x) v[j][x] = __builtin_fmaf(acc[i][j][x], LOG2E, bias[j][x]);
    if (!inside) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int x = 0; x < 4 * G; ++x)
          if (n0 + lane_col + MS * j + 8 * (x / 4) + x % 4 >= a.e.N) v[j][x] = -__builtin_inff();
    }
    if (__builtin_amdgcn_ballot_w64(t >= 0 && t < 64)) {  // few waves have one of their rows' targets
      float picked = 0.f;
      bool here = false;
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int x = 0; x < 4 * G; ++x)
          if (at == MS * j + 8 * (x / 4) + x % 4) {
            picked = v[j][x];
            here = true;
            v[j][x] = -__builtin_inff();
          }
      if (here) a.target_logit[m] = picked;
    }
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int x = 0; x < 4 * G; ++x) top = __builtin_fmaxf(top, v[j][x]);
    top = over_row<MS>(top, [](float x, float y) { return __builtin_fmaxf(x, y); });
    const float ref = top == -__builtin_inff() ? 0.f : top;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int x = 0; x < 4 * G; ++x) s += v[j][x] = __builtin_amdgcn_exp2f(v[j][x] - ref);
    if (n0 < a.exps_cols && m < M) {  // a lane's four neighbours at a time
      const int pitch = (a.exps_cols + 7) & ~7;
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const int n = n0 + MS * j + 8 * g + lane_col;
          if (n >= pitch) continue;
          const float* q = &v[j][4 * g];
          if constexpr (ES == 2) {
            const uv2 c = {exp_code(q[0]) | exp_code(q[1]) << 16, exp_code(q[2]) | exp_code(q[3]) << 16};
            *reinterpret_cast<uv2*>((char*)a.exps + 2 * (m * pitch + n)) = c;
          } else {
            *reinterpret_cast<f32x4*>((char*)a.exps + 4 * (m * pitch + n)) = f32x4{q[0], q[1], q[2], q[3]};
          }
        }
      if (l < MS) a.exps_top[m * ((a.exps_cols + 63) >> 6) + (n0 >> 6)] = top;
    }
    s = over_row<MS>(s, [](float x, float y) { return x + y; });
    if (l < MS) {
      lds[wn * BM + row][0] = top;
      lds[wn * BM + row][1] = s;
    }
  }
  __syncthreads();
  for (int row = threadIdx.x; row < BM; row += 64 * WM * WN) {
    const long long m = m0 + row;
    if (m >= M) return;
    float top = lds[row][0];
#pragma unroll
    for (int k = 1; k < WN; ++k) top = __builtin_fmaxf(top, lds[k * BM + row][0]);
    const float ref = top == -__builtin_inff() ? 0.f : top;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < WN; ++k) s = __builtin_fmaf(lds[k * BM + row][1], __builtin_amdgcn_exp2f(lds[k * BM + row][0] - ref), s);
    float* to = a.stats + 2 * (m * a.tiles_n + tn);
    to[0] = top;
    to[1] = s;
  }
}

template <int ES, int MS, int BM, int BN, int WM, int WN, int NSP, int NSQ, bool PRC, bool QRC, int KIND = DENSE_PLAIN>
__global__ __launch_bounds__(64 * WM * WN, 2) void dense_tile_kernel(typename DenseArgs<KIND>::type a) {
  constexpr int NW = WM * WN, TM = BM / WM / MS, TN = BN / WN / MS;  // fragments of a wave
  typedef Side<ES, BM, NW, PRC> SP;
  typedef Side<ES, BN, NW, QRC> SQ;
  constexpr int LDS_Q = NSP * SP::BYTES, LDS = LDS_Q + NSQ * SQ::BYTES;  // P's stages, then Q's
  extern __shared__ __align__(1024) char smem[];
  int tm, tn, split, tiles_m = a.tiles_m, blocks = gridDim.x;
  long long M = a.e.M, R = a.R;
  if constexpr (KIND != DENSE_PLAIN) {
    if (a.rows) {
      const long long rows = *a.rows;
      if constexpr (PRC) {
        // The tiles that are there go to the first workgroups, as many to every XCD; the others end.
        M = rows < M ? rows : M;
        const int there = (int)((M + BM - 1) / BM);
        blocks = blocks / tiles_m * there;
        if ((int)blockIdx.x >= blocks) {
          if constexpr (KIND == DENSE_CE_GRAD) {
            const int id = blockIdx.x - blocks, n0 = id % a.tiles_n * BN;
            const long long first = (long long)(there + id / a.tiles_n) * WM;
            if (a.col_sums)
              for (int i = threadIdx.x; i < WM * BN; i += 64 * WM * WN)
                if (n0 + i % BN < a.e.N) a.col_sums[(first + i / BN) * a.e.N + n0 + i % BN] = 0.f;
          }
          return;
        }
        tiles_m = there;
      } else {
        R = rows < R ? rows : R;
      }
    }
  }
  tile_of(blockIdx.x, blocks, tiles_m, a.tiles_n, tm, tn, split);
  const int k0 = split * a.steps_per_split;
  const long long m0 = (long long)tm * BM;
  const int n0 = tn * BN;
  int nk = min(a.steps - k0, a.steps_per_split);
  if constexpr (KIND != DENSE_PLAIN && !PRC) {  // a split without rows: a stage of zeros
    const int steps = (int)((R * ES + DENSE_BK - 1) / DENSE_BK);
    nk = max(1, min(steps - k0, a.steps_per_split));
  }
  const int w = threadIdx.x >> 6, wm = w / WN, wn = w % WN;

  SP sp;
  SQ sq;
  sp.init(a.P, a.ldp, m0, M, R, k0);
  sq.init(a.Q, a.ldq, n0, a.e.N, R, k0);
  Reader<ES, MS, BM, PRC> rp;
  Reader<ES, MS, BN, QRC> rq;
  rp.init(wm * TM * MS);
  rq.init(wn * TN * MS);
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;

  typename Sums<MS>::type acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int x = 0; x < MS * MS / 64; ++x) acc[i][j][x] = 0.f;

  // A stage is KK parts of 64 (or 32) bytes of reduction.  Fragments are read a part ahead of the products that
  // take them, across stages too: the barrier that opens a stage stands before the last part of the stage
  // ahead of it, whose products cover the barrier and the first reads.  From then on nobody reads the
  // stage that ends, and copies of a stage further on go there: Q's NSQ on, with the last part, then P's NSP on,
  // a share with each part (issued at once they hold up every wave behind the CU's one address unit).
  constexpr int KK = DENSE_BK * MS / 1024, LP = SP::LOADS, LQ = SQ::LOADS, COPIES = LP + LQ;
  constexpr int SHARE = (COPIES + KK - 1) / KK, FIRST_SHARE = NSP > NSQ && LQ > SHARE ? LQ : SHARE;
  constexpr int REST_SHARE = KK > 1 ? (COPIES - FIRST_SHARE + KK - 2) / (KK - 1) : 0;
  // copies issued behind those of Q's next stage (and of P's, which is no later) when that has to be there
  constexpr int BEHIND = (NSQ - 2) * COPIES + (NSP - NSQ) * LP;
  static_assert(NSQ >= 2 && (NSP == NSQ || NSP == NSQ + 1) && BEHIND + FIRST_SHARE < 64 && KK % 2 == 0, "stages, parts");
  Frag<ES> fp[2][TM], fq[2][TN];
  auto copy = [&](int c, unsigned to_p, unsigned to_q) {
    if (c < LQ) sq.copy(c, lds0 + to_q);
    else sp.copy(c - LQ, lds0 + to_p);
  };
  unsigned cur_p = 0, cur_q = LDS_Q, to_p = (NSP - 1) * SP::BYTES, to_q = LDS_Q + (NSQ - 1) * SQ::BYTES;
  // Products of the fragments of `set`; among the first half of them reads of part kk of the current stage into
  // the other set, so that a barrier behind the part finds them done, among the second half the copies [c0, c1).
  // FENCE: products that the compiler may move them over.  (bf16: in bunches they take 2 to 5% more clocks; fp32: a
  // fence behind each of its long instructions takes 4% more.)
  auto part_of = [&](int set, bool reads, int kk, int c0, int c1, bool prepare) {
    constexpr int SLOTS = TM * TN * Frag<ES>::STEPS, HALF = SLOTS / 2, READS = TM + TN, FENCE = ES == 4 ? 16 : 32 / MS;
    const unsigned lp = lds0 + cur_p, lq = lds0 + cur_q;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int j = s % TN, x = s / TN % Frag<ES>::STEPS, i = s / TN / Frag<ES>::STEPS;
      acc[i][j] = mma(fq[set][j], fp[set][i], x, acc[i][j]);
      if (s < HALF) {
#pragma unroll
        for (int h = s * READS / HALF; reads && h < (s + 1) * READS / HALF; ++h) {
          if (h < TN) fq[set ^ 1][h] = rq.read(lq, h, kk);
          else fp[set ^ 1][h - TN] = rp.read(lp, h - TN, kk);
        }
      } else {
        const int y = s - HALF, n = c1 - c0;
#pragma unroll
        for (int c = y * n / HALF; c < (y + 1) * n / HALF; ++c)
          if (c0 + c < COPIES) copy(c0 + c, to_p, to_q);
      }
      if (prepare && s == SLOTS - 1) {
        sp.prepare();
        sq.prepare();
      }
      if (s % FENCE == FENCE - 1) __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto stage_of_p = [&](unsigned at) {
    sp.prepare();
    sp.open();
#pragma unroll
    for (int c = 0; c < LP; ++c) sp.copy(c, lds0 + at);
  };
  if constexpr (NSP > NSQ) stage_of_p(0);
#pragma unroll
  for (int s = 0; s < NSQ - 1; ++s) {
    sq.prepare();
    sq.open();
#pragma unroll
    for (int c = 0; c < LQ; ++c) sq.copy(c, lds0 + LDS_Q + s * SQ::BYTES);
    stage_of_p((s + NSP - NSQ) * SP::BYTES);
  }
  sp.prepare();
  sq.prepare();
  sp.open();
  sq.open();
#pragma unroll
  for (int c = 0; c < FIRST_SHARE; ++c) copy(c, to_p, to_q);
  copies_barrier<BEHIND + FIRST_SHARE>();
#pragma unroll
  for (int j = 0; j < TN; ++j) fq[0][j] = rq.read(lds0 + LDS_Q, j, 0);
#pragma unroll
  for (int i = 0; i < TM; ++i) fp[0][i] = rp.read(lds0, i, 0);
  for (int k = 0; k < nk - 1; ++k) {
#pragma unroll
    for (int kk = 0; kk < KK - 1; ++kk)
      part_of(kk & 1, true, kk + 1, FIRST_SHARE + kk * REST_SHARE, FIRST_SHARE + (kk + 1) * REST_SHARE, kk == KK - 2);
    to_p = cur_p;
    to_q = cur_q;
    cur_p = cur_p == (NSP - 1) * SP::BYTES ? 0 : cur_p + SP::BYTES;
    cur_q = cur_q == LDS_Q + (NSQ - 1) * SQ::BYTES ? LDS_Q : cur_q + SQ::BYTES;
    sp.open();
    sq.open();
    copies_barrier<BEHIND>();
    part_of((KK - 1) & 1, true, 0, 0, FIRST_SHARE, false);
  }
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) part_of(kk & 1, kk + 1 < KK, kk + 1, 0, 0, false);

  // The sums go through LDS, 32 rows of 64 columns of the wave at a time, so that a lane gets 4 neighbours
  // of a row and 16 lanes a whole row (128 bytes of bf16).  Rows are 68 floats apart: 16 rows of a store then
  // fall on all banks.  What is added to 16 rows is loaded before the stores of the 16 ahead of them:
  // stores and loads share a counter that runs in order, and a load behind a store waits for it.  A lane's rows
  // are in registers four together, so types, kinds and edges are decided once for all of them.  (A row at a
  // time, with its loads and branches, took 33,000 clocks a tile, as long as 12 stages of products.)
  static_assert(TN * MS == 64 && TM * MS % 32 == 0 && NW * 32 * 68 * 4 <= LDS, "a wave's rows of 64 columns");
  constexpr bool FORWARD = PRC && QRC && KIND == DENSE_PLAIN;  // bias, activation, residual and what is kept; else sums as they are
  constexpr int ROWS = 4;               // of a lane at a time, 4 apart
  // The caches need not keep the large tile's results and what is added to them, but the operands of the tiles that
  // still run.  By tile, not by the outputs' size.  With it and without, us: 8192 x 8192 over 4096 with an fp32 residual
  // 480 / 525, 4096 x 4096 over 16384 (TN) 372 / 387, forward and backward of 8192 x 4096 over 4096 with GELU 647 / 668, of 4096
  // x 4096 over 1024 no different (161 to 169), that forward alone 43.5 / 45.3.  What it loses: a next product that reads 32 MB of
  // results at once, 4096 x 1024 -> 4096 -> 1024 in a graph 80 / 75.  The smaller tiles go without: fp32 2048 x 4096
  // over 1024 takes 2% longer with it.
  constexpr bool STREAM = BM * BN == 65536 && KIND != DENSE_CE_GRAD;
  copies_barrier<0>();
  if constexpr (KIND == DENSE_CE_STATS) {
    ce_stats<ES, MS, BM, BN, WM, WN, TM, TN>(a, M, tm, tn, acc, reinterpret_cast<float(*)[2]>(smem));
    return;
  }
  const int l = threadIdx.x & 63;
  uv4* info = reinterpret_cast<uv4*>(smem + NW * 32 * 68 * 4);  // DENSE_CE_GRAD: the tile's rows
  if constexpr (KIND == DENSE_CE_GRAD) {
    static_assert(NW * 32 * 68 * 4 + BM * 16 <= LDS, "the rows' place");
    for (int r = threadIdx.x; r < BM; r += 64 * NW) info[r] = m0 + r < M ? a.row_info[m0 + r] : uv4{0u, 0u, 0u, 0u};
    __syncthreads();
  }
  float* own = reinterpret_cast<float*>(smem) + w * 32 * 68;
  const bool split_up = KIND != DENSE_CE_GRAD && a.part != nullptr;
  const Added added = split_up || KIND == DENSE_CE_GRAD ? Added{nullptr, 0, false} : dense_added(a.e);
  char* C = split_up ? (char*)(a.part + (long long)split * a.e.M * a.e.N) : (char*)a.e.C;
  const bool c_bf = !split_up && a.e.c_bf;
  const long long c_step = (split_up ? a.e.N : a.e.sc) * (c_bf ? 2 : 4);
  const bool inside = m0 + BM <= M && n0 + BN <= a.e.N;
  const int n = n0 + wn * 64 + (l & 15) * 4, there = a.e.N - n;
  const long long mw = m0 + wm * TM * MS + (l >> 4);
  float bias[4];
  if constexpr (FORWARD || KIND == DENSE_CE_GRAD) dense_bias(a.e, n, bias);
  if constexpr (KIND == DENSE_CE_GRAD) {
#pragma unroll
    for (int j = 0; j < 4; ++j) bias[j] = ce_bias(bias[j]);
  }
  float alpha = 1.f;
  if constexpr (KIND == DENSE_ROWS) alpha = a.alpha && !split_up ? *a.alpha : 1.f;
  float col[4] = {0.f, 0.f, 0.f, 0.f};  // DENSE_CE_GRAD: of this lane's columns
  uv4 r[ROWS];
  auto load_rows = [&](long long m) {
    const char* p = added.p + m * added.step + (long long)n * (added.bf ? 2 : 4);
    if (inside && added.bf) {
#pragma unroll
      for (int x = 0; x < ROWS; ++x) {
        const char* px = p + 4 * x * added.step;
        const uv2 t = STREAM ? (uv2)__builtin_nontemporal_load(reinterpret_cast<const uv2_any*>(px))
                             : reinterpret_cast<const bytes8*>(px)->v;
        r[x] = uv4{t[0], t[1], 0u, 0u};
      }
    } else if (inside) {
#pragma unroll
      for (int x = 0; x < ROWS; ++x) {
        const char* px = p + 4 * x * added.step;
        r[x] = STREAM ? (uv4)__builtin_nontemporal_load(reinterpret_cast<const uv4_any*>(px))
                      : reinterpret_cast<const bytes16*>(px)->v;
      }
    } else {
#pragma unroll
      for (int x = 0; x < ROWS; ++x) {
        r[x] = uv4{0u, 0u, 0u, 0u};
        if (m + 4 * x < M && there > 0) r[x] = load_added(p + 4 * x * added.step, added.bf, there);
      }
    }
  };
  if (added.p) load_rows(mw);
#pragma unroll 1
  for (int i = 0; i < TM * MS / 32; ++i) {
    // acc[h][j], four at a time: row l % MS, columns from 4 (l / MS)
#pragma unroll
    for (int h = 0; h < 32 / MS; ++h)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int g = 0; g < MS * MS / 256; ++g) {
          f32x4 t;
#pragma unroll
          for (int x = 0; x < 4; ++x) t[x] = acc[h][j][4 * g + x];
          *reinterpret_cast<f32x4*>(own + (MS * h + l % MS) * 68 + MS * j + 8 * g + 4 * (l / MS)) = t;
        }
    // a rolled loop (its code is loaded once): the rows of accumulators move up
#pragma unroll
    for (int y = 0; y + 32 / MS < TM; ++y)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[y][j] = acc[y + 32 / MS][j];
#pragma unroll 1
    for (int y = 0; y < 32; y += 4 * ROWS) {
      const long long mi = mw + i * 32 + y;
      float v[ROWS][4];
#pragma unroll
      for (int x = 0; x < ROWS; ++x) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(own + (y + 4 * x + (l >> 4)) * 68 + (l & 15) * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[x][j] = t[j];
      }
      if constexpr (FORWARD) {
        if (!split_up) dense_forward<ROWS>(a.e, mi, 4, n, v, bias);
      }
      if constexpr (KIND == DENSE_ROWS) {
#pragma unroll
        for (int x = 0; x < ROWS; ++x)
#pragma unroll
          for (int j = 0; j < 4; ++j) v[x][j] *= alpha;
      }
      if constexpr (KIND == DENSE_CE_GRAD) {
        int t[ROWS];
        float at_t[ROWS];
        bool any = false;
#pragma unroll
        for (int x = 0; x < ROWS; ++x) {
          const uv4 q = info[wm * TM * MS + i * 32 + y + 4 * x + (l >> 4)];
          const float top = __uint_as_float(q[0]), f = __uint_as_float(q[1]);
          t[x] = (int)q[2] - a.first - n;
          at_t[x] = __uint_as_float(q[3]);
          any |= (unsigned)t[x] < 4u || f == 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            v[x][j] = f * __builtin_amdgcn_exp2f(__builtin_fmaf(v[x][j], LOG2E, bias[j]) - top);
        }
        // few waves have a target, or a row without a gradient
        if (__builtin_amdgcn_ballot_w64(any)) {
#pragma unroll
          for (int x = 0; x < ROWS; ++x) {
            const bool none = __uint_as_float(info[wm * TM * MS + i * 32 + y + 4 * x + (l >> 4)][1]) == 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[x][j] = none ? 0.f : t[x] == j ? at_t[x] : v[x][j];
          }
        }
        if (!inside) {
#pragma unroll
          for (int x = 0; x < ROWS; ++x)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[x][j] = j < there ? v[x][j] : 0.f;
        }
        if (a.col_sums) {
#pragma unroll
          for (int x = 0; x < ROWS; ++x)
#pragma unroll
            for (int j = 0; j < 4; ++j) col[j] += v[x][j];
        }
      }
      if (added.p) {
        if (added.bf) {
#pragma unroll
          for (int x = 0; x < ROWS; ++x) add_added(v[x], r[x], true);
        } else {
#pragma unroll
          for (int x = 0; x < ROWS; ++x) add_added(v[x], r[x], false);
        }
        if (i + 1 < TM * MS / 32 || y + 4 * ROWS < 32) load_rows(mi + 4 * ROWS);
      }
      char* c = C + mi * c_step + (long long)n * (c_bf ? 2 : 4);
      if (inside && c_bf) {
#pragma unroll
        for (int x = 0; x < ROWS; ++x) store4<STREAM>(c + 4 * x * c_step, true, 0, 4, v[x]);
      } else if (inside) {
#pragma unroll
        for (int x = 0; x < ROWS; ++x) store4<STREAM>(c + 4 * x * c_step, false, 0, 4, v[x]);
      } else {
        const int width = KIND == DENSE_CE_GRAD ? n_pitch(a) - n : there;
#pragma unroll
        for (int x = 0; x < ROWS; ++x)
          if (mi + 4 * x < M && width > 0) store4(c + 4 * x * c_step, c_bf, 0, width, v[x]);
      }
    }
  }
  if constexpr (KIND == DENSE_CE_GRAD) {
    if (a.col_sums) {
#pragma unroll
      for (int j = 0; j < 4; ++j) col[j] = over_row<16>(col[j], [](float x, float y) { return x + y; });
      if (l < 16 && there > 0) store4(a.col_sums, false, ((long long)tm * WM + wm) * a.e.N + n, there, col);
    }
  }
}

// ---- host side ---------------------------------------------------------------------------------------
enum { DENSE_NT = 0, DENSE_NN = 1, DENSE_TN = 2 };  // P, Q: RC RC; RC RS; RS RS
// Tiles.  The large one keeps the matrix cores fed at the least traffic; the smaller ones fill the chip when
// there are few.  DEEP: three stages (one workgroup a CU), which hides more of a load's latency where few
// workgroups run.
enum { DENSE_256 = 0, DENSE_256X128 = 1, DENSE_128 = 2, DENSE_128_DEEP = 3, DENSE_64 = 4, DENSE_TILES = 5 };
constexpr int DENSE_BM[DENSE_TILES] = {256, 256, 128, 128, 64}, DENSE_BN[DENSE_TILES] = {256, 128, 128, 128, 128};

template <int ES, int MS, int BM, int BN, int WM, int WN, int NSP, int NSQ, bool PRC, bool QRC, int KIND = DENSE_PLAIN>
int launch_dense_tile_as(const typename DenseArgs<KIND>::type& a, int splits, hipStream_t s) {
  constexpr auto kernel = dense_tile_kernel<ES, MS, BM, BN, WM, WN, NSP, NSQ, PRC, QRC, KIND>;
  constexpr size_t lds = (NSP * BM + NSQ * BN) * DENSE_BK;
  // the kernel's LDS limit is raised once a device
  static std::atomic<unsigned long long> raised{0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return GL_ERR_DEVICE;
  if (!(raised.load(std::memory_order_relaxed) >> dev & 1)) {
    GL_TRY(set_lds_limit((const void*)kernel, lds));
    raised.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  GL_LAUNCH(KIND == DENSE_CE_STATS ? GL_KERNEL_CE_STATS : KIND == DENSE_CE_GRAD ? GL_KERNEL_CE_GRAD : GL_KERNEL_DENSE, kernel,
            dim3((unsigned)(a.tiles_m * a.tiles_n * splits)), dim3(64 * WM * WN), lds, s, a);
  GL_CHECK_LAUNCH();
  return 0;
}
template <int ES, int MS, int BM, int BN, int WM, int WN, int NSP, int NSQ>
int launch_dense_tile_of(int form, const DenseK& a, int splits, hipStream_t s) {
  if (form == DENSE_NT) return launch_dense_tile_as<ES, MS, BM, BN, WM, WN, NSP, NSQ, true, true>(a, splits, s);
  if (form == DENSE_NN) return launch_dense_tile_as<ES, MS, BM, BN, WM, WN, NSP, NSQ, true, false>(a, splits, s);
  return launch_dense_tile_as<ES, MS, BM, BN, WM, WN, NSP, NSQ, false, false>(a, splits, s);
}
int launch_dense_tile_bf16(int form, int tile, const DenseK& a, int splits, hipStream_t s);
int launch_dense_tile_f32(int form, int tile, const DenseK& a, int splits, hipStream_t s);
// the kinds but DENSE_PLAIN; form: NT for the two of the cross entropy, NN or TN with DENSE_ROWS
template <int ES, int MS, int BM, int BN, int WM, int WN, int NSP, int NSQ>
int launch_rows_tile_of(int kind, int form, const DenseRowsK& a, int splits, hipStream_t s) {
  if (kind == DENSE_CE_STATS) return launch_dense_tile_as<ES, MS, BM, BN, WM, WN, NSP, NSQ, true, true, DENSE_CE_STATS>(a, splits, s);
  if (kind == DENSE_CE_GRAD) return launch_dense_tile_as<ES, MS, BM, BN, WM, WN, NSP, NSQ, true, true, DENSE_CE_GRAD>(a, splits, s);
  if (form == DENSE_NN) return launch_dense_tile_as<ES, MS, BM, BN, WM, WN, NSP, NSQ, true, false, DENSE_ROWS>(a, splits, s);
  return launch_dense_tile_as<ES, MS, BM, BN, WM, WN, NSP, NSQ, false, false, DENSE_ROWS>(a, splits, s);
}
int launch_rows_tile_bf16(int kind, int form, int tile, const DenseRowsK& a, int splits, hipStream_t s);
int launch_rows_tile_f32(int kind, int form, int tile, const DenseRowsK& a, int splits, hipStream_t s);

// ---- plans (gl_dense.hip) ----------------------------------------------------------------------------
constexpr int es_of(int dtype) { return dtype == GL_DTYPE_BF16 ? 2 : 4; }
inline long long padded(long long n) { return round_up(n, 8); }  // row of a copied or computed operand

struct Operand {
  const void* p;
  long long ld;  // elements
  long long rows;
  int cols;
  bool rc;       // reduction along the row
  bool copied;   // through workspace
};
Operand operand(const void* p, long long ld, long long rows, int cols, bool rc, int es);
size_t copy_bytes(const Operand& o, int es);
// copies those of the operands (null or not) that need it to their places; they then are the copies
int launch_align(Operand* o0, void* dst0, Operand* o1, void* dst1, int es, hipStream_t s);
struct Product {
  double us;  // what the plan expects
  int tile, splits, steps_per_split, steps, tiles_m, tiles_n;
  size_t part_bytes;
};
Product plan_product(int dtype, long long M, int N, long long R, int most_splits = 32);
// rows, alpha: DENSE_ROWS (both null: DENSE_PLAIN)
int run_product(int dtype, int form, const Operand& p, const Operand& q, long long R, const Product& pl, void* part,
                const DenseEpi& e, hipStream_t s, const int* rows = nullptr, const float* alpha = nullptr);
DenseEpi store_epi(void* C, long long sc, int c_dtype, long long M, int N, int op_dtype, int accumulate);
int launch_db(const float* part, long long chunks, int N, void* db, int g_dtype, int accumulate, hipStream_t s,
              const float* alpha = nullptr);

// few rows (gl_dense_few.hip): the forward of up to DENSE_FEW_ROWS rows that keeps nothing
constexpr int DENSE_FEW_ROWS = 64;
int launch_dense_few(const GlDenseArgs* a, const DenseEpi& e, hipStream_t s);

}  // namespace gl
