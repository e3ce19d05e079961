// Fused AdamW over a list of tensors: one streaming pass reads p, g, m, v (and an fp32 master copy) and writes
// p, m, v and, of main_grad buffers, g = 0.  Bytes an element: 32 with fp32 parameters, gradient buffers and
// moments, 24 with bf16 moments, 20 with moments in 8 bits; 10 with parameters and gradients in bf16 and moments in 8 bits.
// Reference: _adamw_kernel, sparse_pooling/optim.py:26-64 (fp32 parameters; bf16 parameters with
// HAS_MASTER, with STOCH, or rounded to nearest even), a launch a tensor.  With fp32 and bf16 moments the
// update is evaluated unfused in the reference's operation order; every element is read and
// written by the same thread, so the in-place race fixed at optim.py:43-50 cannot occur.
//
// Moments in 8 bits (no counterpart in the reference): blocks of 256 neighbouring elements of a tensor share two
// fp32 scales,
//     m = s c |c|      c from -127 to 127    s = max |m| / 127^2
//     v = (r c^2)^2    c from 0 to 255       r = sqrt(max v) / 255^2
// Two neighbouring codes are 2 / c of m and 4 / c of v apart, 1.6% each next to the maximum, and sqrt(v) reaches down to
// 1.5e-5 of the largest.  A step takes a share 1 - b2 off v, 0.1%, so codes are not the nearest, which would stay where they
// are while the value decays: a value goes to one of its two neighbours, drawn so that it is kept on average, and the kept v
// is the unrounded one's on average after any number of steps, apart from it by about sqrt(2 / c) of itself (simulated over 7,000
// steps: sqrt(v) off by 4% at c = 200, 20% at 25; nearest codes 1.37 and 17 times too large there).  Codes of v are 1 at
// least where v > 0: a sqrt(v) rounded to nothing would leave m / eps.  The update itself takes the moments before they are
// put into 8 bits.
// Nearest codes (in their root) are there for callers that want no noise.  A value next to a border between two of them must not
// depend on how its sums are rounded, so moments are computed in 64 bits, which this chip does as fast as unpacked 32, and so
// are these codes where fp32 cannot tell.  A block with an infinity or a NaN in m or v has
// the scale NaN; one whose largest |m| is below 2^-100 (v: 2^-126) the scale 0.
#include "gl_common.h"
#include "gl_internal.h"
#include "gl_pack8.h"

namespace gl {

struct AdamK {
  float lr, b1, b2, eps, wd, bc1, bc2;
};

// The tensors of a launch travel as kernel arguments: nothing to copy to the device, nothing to keep alive.
constexpr int ADAM_TENSORS = 38;      // of a launch: in the 4 KB that arguments may take
constexpr int ADAM_BLOCK = 256;       // elements that share a scale
// the kernels' kinds of moments: GL_DTYPE_F32, GL_DTYPE_BF16, GL_MOMENTS_INT8, and that with nearest codes
constexpr int MOMENTS_INT8_NEAREST = 3;
constexpr bool in_8bit(int moments) { return moments == GL_MOMENTS_INT8 || moments == MOMENTS_INT8_NEAREST; }
// elements of a workgroup: a vector of 4 a thread, or two with 8-bit moments
constexpr int adam_chunk(int moments) { return in_8bit(moments) ? 2048 : 1024; }
struct AdamTensorK {
  void* p;
  void* g;
  void* m;
  void* v;
  float* master;
  float* m_scale;
  float* v_scale;
  long long n;
  long long first;                     // of the tensor's elements
  unsigned long long seed;
  float bc1, bc2;
};
struct AdamTable {
  float lr, b1, b2, eps, wd;
  int count, clear;
  double b1d, a1d, b2d, a2d;           // of the 8-bit moments: betas and 1 - beta
  unsigned first[ADAM_TENSORS + 1];    // first workgroup of every tensor
  AdamTensorK t[ADAM_TENSORS];
};
static_assert(sizeof(AdamTable) <= 4096, "kernel arguments");

// (1 - b1 and 1 - b2 of the fp32 betas, as the reference has them: 0.999 is off by 1.3e-8, 1 - 0.999 by 1.3e-5 of itself.  8-bit
// moments take the betas in 64 bits.)
__device__ __forceinline__ void adam_elem(const AdamK& c, float& p, float g, float& m, float& v) {
#pragma clang fp contract(off)
  m = c.b1 * m + (1.0f - c.b1) * g;
  v = c.b2 * v + (1.0f - c.b2) * g * g;
  const float upd = (m / c.bc1) / (__builtin_sqrtf(v / c.bc2) + c.eps);
  p = p * (1.0f - c.lr * c.wd) - c.lr * upd;
}

// Streams are read and written with non-temporal loads and stores (each element is touched once;
// at C2's 805M elements this ran at 6.3 TB/s against 5.4 with plain accesses in a measurement of
// this access pattern).  Vectors are at the elements' own alignment, so a tensor may begin anywhere.
typedef unsigned w4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned w2 __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned w1 __attribute__((aligned(1)));

// four neighbours from element i of a wave's part p, of which the first n are there
template <bool BF>
__device__ __forceinline__ void adam_load(const void* p, unsigned i, int n, float (&v)[4]) {
  if (n >= 4) {
    if constexpr (BF) {
      const w2 w = __builtin_nontemporal_load(reinterpret_cast<const w2*>((const char*)p + 2 * i));
      v[0] = __uint_as_float(w[0] << 16);
      v[1] = __uint_as_float(w[0] & 0xffff0000u);
      v[2] = __uint_as_float(w[1] << 16);
      v[3] = __uint_as_float(w[1] & 0xffff0000u);
    } else {
      const w4 w = __builtin_nontemporal_load(reinterpret_cast<const w4*>((const char*)p + 4 * i));
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(w[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < n ? ld_param_t<BF>((const float*)p, i + j) : 0.f;
  }
}
__device__ __forceinline__ void adam_store(float* p, unsigned i, int n, const float (&v)[4]) {
  if (n >= 4) {
    w4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(v[j]);
    __builtin_nontemporal_store(w, reinterpret_cast<w4*>(p + i));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) p[i + j] = v[j];
  }
}
// four bf16 in two words
__device__ __forceinline__ void adam_store(unsigned short* p, unsigned i, int n, unsigned lo, unsigned hi) {
  if (n >= 4) {
    __builtin_nontemporal_store((w2){lo, hi}, reinterpret_cast<w2*>(p + i));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) p[i + j] = (unsigned short)((j < 2 ? lo : hi) >> (16 * (j & 1)));
  }
}
__device__ __forceinline__ unsigned adam_load_codes(const void* p, unsigned i, int n) {
  const unsigned char* c = (const unsigned char*)p + i;
  if (n >= 4) return __builtin_nontemporal_load(reinterpret_cast<const w1*>(c));
  unsigned w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < n) w |= (unsigned)c[j] << (8 * j);
  return w;
}
__device__ __forceinline__ void adam_store_codes(void* p, unsigned i, int n, unsigned w) {
  unsigned char* c = (unsigned char*)p + i;
  if (n >= 4) {
    __builtin_nontemporal_store((w1)w, reinterpret_cast<w1*>(c));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) c[j] = (unsigned char)(w >> (8 * j));
  }
}

// Parameter storage of the update: fp32, or bf16 rounded to nearest even, bf16 with an fp32
// master copy (the update runs on the master, the parameter gets its rounding), or bf16 with
// stochastic rounding (optim.py:59-62).
enum { PM_F32 = 0, PM_BF16_RNE = 1, PM_BF16_MASTER = 2, PM_BF16_SR = 3 };

// Philox-4x32 (Salmon et al., SC'11) of the counter c under the key (k0, k1)
template <int ROUNDS>
__device__ __forceinline__ uv4 philox(uv4 c, unsigned k0, unsigned k1) {
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const unsigned h0 = __umulhi(0xD2511F53u, c[0]), l0 = 0xD2511F53u * c[0];
    const unsigned h1 = __umulhi(0xCD9E8D57u, c[2]), l1 = 0xCD9E8D57u * c[2];
    c = uv4{h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0};
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}
// Triton's tl.randint(seed, offset) (triton/language/random.py, 3.6): the first word of Philox-4x32-10 of the counter
// (offset low, offset high, 0, 0) under the key (seed low, seed high).
__device__ __forceinline__ unsigned philox_randint(unsigned long long seed, unsigned long long off) {
  return philox<10>(uv4{(unsigned)off, (unsigned)(off >> 32), 0u, 0u}, (unsigned)seed, (unsigned)(seed >> 32))[0];
}

// the bf16 parameter of element i from its fp32 update p
__device__ __forceinline__ unsigned round_stochastic(float p, unsigned long long seed, long long i) {
  return (__float_as_uint(p) + (philox_randint(seed, (unsigned long long)i) & 0xffffu)) >> 16;
}

// ---- 8-bit moments -----------------------------------------------------------------------------------
// the largest of the 32 lanes of half a wave, integer order (of values >= 0: the values' order, infinities and NaN above every number)
__device__ __forceinline__ unsigned half_umax(unsigned v) {
  auto up = [](unsigned a, unsigned b) { return umax(a, b); };
  v = up(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));   // lane ^ 1
  v = up(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));   // lane ^ 2
  v = up(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));  // row_ror:4
  v = up(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));  // row_ror:8
  const auto p16 = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return up(p16[0], p16[1]);
}
// 1 / x of a positive normal fp32 x to 2^-45, and sqrt(x) to about 2^-51: estimates of 2^-23 and one or two steps of Newton's
__device__ __forceinline__ double reciprocal(float x) {
  const double r = (double)__builtin_amdgcn_rcpf(x);
  return __builtin_fma(r, __builtin_fma(-(double)x, r, 1.0), r);
}
__device__ __forceinline__ double root(float x) {
  const float e = __builtin_amdgcn_sqrtf(x);
  const double d = (double)x, h = 0.5 * (double)__builtin_amdgcn_rcpf(e);
  double r = (double)e;
  r = __builtin_fma(h, __builtin_fma(-r, r, d), r);
  return __builtin_fma(h, __builtin_fma(-r, r, d), r);
}
// scales of a block from the bits of its largest fp32 |m| and v
__device__ __forceinline__ float scale_m(unsigned top) {
  if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return top < 0x0d800000u ? 0.f : (float)((double)__uint_as_float(top) * (1.0 / 16129.0));
}
__device__ __forceinline__ float scale_v(unsigned top) {
  if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return top < 0x00800000u ? 0.f : (float)(root(__uint_as_float(top)) * (1.0 / 65025.0));
}
// Codes.  In fp32, where a root is within 8e-5 of its own: adding 1.5 x 2^23 rounds it to a whole number, which is left in
// the low byte in two's complement, and `near` gathers how far roots are from whole numbers.  Where one is within
// CODE_NEAR of a border between two codes (a wave in nine) all of the wave's are decided in 64 bits instead: of floor(x + 1/2),
// x the root, an estimate decides all but which side of i + 1/2 x is on, and (i + 1/2)^2, exact in 64 bits, decides that.
constexpr float CODE_NEAR = 0x1p-13f;
__device__ __forceinline__ unsigned code_of(float x, float& near) {
  const float r = x + 12582912.f;
  near = __builtin_fmaxf(near, __builtin_fabsf(x - (r - 12582912.f)));
  return __float_as_uint(r);
}
__device__ __forceinline__ unsigned code_m(double y) {
  const float i = __builtin_floorf(__builtin_amdgcn_sqrtf((float)y) + 0.25f), h = i + 0.5f;
  return (unsigned)i + (y >= (double)(h * h) ? 1u : 0u);
}
// of the fourth root
__device__ __forceinline__ unsigned code_v(double y) {
  const float i = __builtin_floorf(__builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf((float)y)) + 0.25f), h = i + 0.5f;
  const double h2 = (double)(h * h);
  return (unsigned)i + (y >= h2 * h2 ? 1u : 0u);
}
// Noise of the codes of four neighbours, 14 bits for each m and 18 above them for each v, of which a step changes less: with
// b2 = 0.9999 and c = 10, 1 / 4000 of the way to the next code.  It is a hash of what the step has in
// hand: the elements' place, their parameters and new moments, and the step's corrections and seed; nothing is kept for it, and a
// replayed graph, whose arguments are those of its capture, draws anew from the moments.  (Where gradients are the same in every step,
// these stop changing in time, and then the corrections do: the seed must tell such steps apart.)  Seven rounds are the fewest
// that pass Philox's authors' tests.
__device__ __forceinline__ uv4 code_noise(unsigned long long vec, const float (&p)[4], const float (&m)[4], const float (&v)[4],
                                          float k0, float k1, unsigned long long seed) {
  auto hash = [](const float (&x)[4]) {
    unsigned h = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) h = h * 0x9E3779B1u + __float_as_uint(x[j]);
    return h;
  };
  return philox<7>(uv4{(unsigned)vec, (unsigned)(vec >> 32) ^ hash(p), hash(m), hash(v)}, __float_as_uint(k0) ^ (unsigned)seed,
                   __float_as_uint(k1) ^ (unsigned)(seed >> 32));
}
// Codes of |m| and v over the scale (over its square): the lower neighbour or, with the probability that keeps the value on
// average, the upper one; `noise` is one of 2^14 (2^18) equal shares.  (Where fp32 puts a quotient next to a code on its other side, the
// code is still the neighbour that is taken nearly always.)
__device__ __forceinline__ unsigned drawn_m(float q, unsigned noise) {
  const float i = __builtin_fminf(__builtin_floorf(__builtin_amdgcn_sqrtf(q)), 126.f);
  const float u = __builtin_fmaf((float)noise, 0x1p-14f, 0x1p-15f);
  return (unsigned)i + (__builtin_fmaf(-i, i, q) > u * (2.f * i + 1.f) ? 1u : 0u);
}
__device__ __forceinline__ unsigned drawn_v(float q, unsigned noise) {
  const float i = __builtin_fminf(__builtin_floorf(__builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(q))), 254.f), i2 = i * i;
  const float u = __builtin_fmaf((float)noise, 0x1p-18f, 0x1p-19f), t = 2.f * i + 1.f;
  return (unsigned)i + (__builtin_fmaf(-i2, i2, q) > u * (t * (2.f * i2 + t)) ? 1u : 0u);  // t (2 i^2 + t) = (i + 1)^4 - i^4
}
__device__ __forceinline__ unsigned low_bytes(const unsigned (&c)[4]) {
  return __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u) | __builtin_amdgcn_perm(c[3], c[2], 0x04000c0cu);
}
// c |c| of code j of m, c^4 of v: m and v over the scale and over its square
__device__ __forceinline__ double square_m(unsigned codes, int j) {
  const int c = (int)(codes << (24 - 8 * j)) >> 24;
  return (double)(c * __builtin_abs(c));
}
__device__ __forceinline__ double fourth_v(unsigned codes, int j) {
  const unsigned c = (codes >> (8 * j)) & 255u, s = c * c;
  return (double)(s * s);  // up to 255^4 < 2^32
}

// the tensor of this workgroup
__device__ __forceinline__ int adam_tensor(const AdamTable& a) {
  int t = 0;
  for (int step = 32; step > 0; step >>= 1)
    if (t + step < a.count && a.first[t + step] <= blockIdx.x) t += step;
  return t;
}

// MOM: the kind of moments; GBF: bf16 gradients.  A workgroup takes a chunk of one tensor, a
// thread a vector of each stream, or two with 8-bit moments: a block is half a wave's then, and what is done for a block (its
// maxima and scales) is done for two at once.  150M bf16 parameters and gradients, nearest codes: 305 us (4.9 TB/s; bound by instructions,
// 246 us at the rate of the fp32 stream), 352 with a block a wave (319 then); fp32 ones 393, drawn codes 445.  400M fp32 in all types:
// 2.2 ms (5.7 TB/s).  Parameters rounded stochastically take a Philox-4x32-10 an element: bf16 moments 529 us, 345 rounded to nearest.
// WHOLE: all of the wave's elements are there (no lane's ends are looked at).
constexpr int adam_vectors(int mom) { return in_8bit(mom) ? 2 : 1; }
template <int MOM, int PM, bool GBF, bool WHOLE>
__device__ __forceinline__ void adam_vector(const AdamTable& a, const AdamTensorK& t, long long base) {
  constexpr bool I8 = in_8bit(MOM), BM = MOM == GL_DTYPE_BF16;
  constexpr int V = adam_vectors(MOM);
  const AdamK c{a.lr, a.b1, a.b2, a.eps, a.wd, t.bc1, t.bc2};
  constexpr int PB = PM == PM_BF16_RNE || PM == PM_BF16_SR ? 2 : 4, MB = I8 ? 1 : (BM ? 2 : 4);
  const unsigned lane = threadIdx.x & 63;
  unsigned i[V];
  int n[V];
#pragma unroll
  for (int x = 0; x < V; ++x) {
    i[x] = I8 ? (lane >> 5) * ADAM_BLOCK + x * (ADAM_BLOCK / 2) + 4 * (lane & 31) : 4 * lane;
    const long long left = t.n - base - i[x];
    n[x] = WHOLE || left > 4 ? 4 : (left < 0 ? 0 : (int)left);
  }
  float p[V][4], g[V][4], m[V][4], v[V][4];
  char* P = (PM == PM_BF16_MASTER ? (char*)t.master : (char*)t.p) + base * PB;
  char* G = (char*)t.g + base * (GBF ? 2 : 4);
  char* M = (char*)t.m + base * MB;
  char* U = (char*)t.v + base * MB;
#pragma unroll
  for (int x = 0; x < V; ++x) {
    adam_load<PB == 2>(P, i[x], n[x], p[x]);
    adam_load<GBF>(G, i[x], n[x], g[x]);
  }
  if constexpr (I8) {
    unsigned cm[V], cv[V];
#pragma unroll
    for (int x = 0; x < V; ++x) {
      cm[x] = adam_load_codes(M, i[x], n[x]);
      cv[x] = adam_load_codes(U, i[x], n[x]);
    }
    const bool here = WHOLE || i[0] - 4 * (lane & 31) < t.n - base;  // this half's block
    const unsigned half = lane >> 5;
    float* scale_of_m = t.m_scale + base / ADAM_BLOCK;
    float* scale_of_v = t.v_scale + base / ADAM_BLOCK;
    const double sm = here ? (double)scale_of_m[half] : 0.0, sv = here ? (double)scale_of_v[half] : 0.0;
    const double bm = a.b1d * sm, bv = a.b2d * (sv * sv);
    // (behind the end: 0, and NaN in a block that is NaN anyway)
    double dm[V][4], dv[V][4];
    unsigned tm = 0, tv = 0;
#pragma unroll
    for (int x = 0; x < V; ++x)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double gj = (double)g[x][j];
        dm[x][j] = __builtin_fma(square_m(cm[x], j), bm, a.a1d * gj);
        dv[x][j] = __builtin_fma(fourth_v(cv[x], j), bv, a.a2d * (gj * gj));
        m[x][j] = (float)dm[x][j];
        v[x][j] = (float)dv[x][j];
        tm = umax(tm, abs_bits(m[x][j]));
        tv = umax(tv, __float_as_uint(v[x][j]));  // of v >= 0; a NaN is above every number with either sign
      }
    const float fs = scale_m(half_umax(tm)), fr = scale_v(half_umax(tv));
    const bool live_m = fs > 0.f, live_v = fr > 0.f;
    const float im = __builtin_amdgcn_rcpf(live_m ? fs : 1.f), ir = __builtin_amdgcn_rcpf(live_v ? fr : 1.f);
    unsigned om[V][4], ov[V][4];
    float rv[V][4];  // sqrt(v) over its scale
#pragma unroll
    for (int x = 0; x < V; ++x)
#pragma unroll
      for (int j = 0; j < 4; ++j) rv[x][j] = __builtin_amdgcn_sqrtf(v[x][j] * ir * ir);
    if constexpr (MOM == GL_MOMENTS_INT8) {
      const double dim = reciprocal(live_m ? fs : 1.f), dir = reciprocal(live_v ? fr : 1.f), dir2 = dir * dir;
#pragma unroll
      for (int x = 0; x < V; ++x) {
        const uv4 noise = code_noise((unsigned long long)(t.first + base + i[x]) >> 2, p[x], m[x], v[x], c.bc1, c.bc2, t.seed);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const unsigned q = drawn_m((float)(__builtin_fabs(dm[x][j]) * dim), noise[j] & 0x3fffu);
          const unsigned u = drawn_v((float)(dv[x][j] * dir2), noise[j] >> 14);
          om[x][j] = dm[x][j] < 0.0 ? 0u - q : q;
          ov[x][j] = u == 0 && dv[x][j] > 0.0 ? 1u : u;
        }
      }
    } else {
      float near = 0.f;
#pragma unroll
      for (int x = 0; x < V; ++x)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          om[x][j] = code_of(__builtin_copysignf(__builtin_amdgcn_sqrtf(__builtin_fabsf(m[x][j]) * im), m[x][j]), near);
          ov[x][j] = code_of(__builtin_fmaxf(__builtin_amdgcn_sqrtf(rv[x][j]), dv[x][j] > 0.0 ? 0.75f : 0.f), near);
        }
      if (__builtin_amdgcn_ballot_w64(near > 0.5f - CODE_NEAR)) {
        const double dim = reciprocal(live_m ? fs : 1.f), dir = reciprocal(live_v ? fr : 1.f);
#pragma unroll
        for (int x = 0; x < V; ++x)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const unsigned q = live_m ? code_m(__builtin_fabs(dm[x][j]) * dim) : 0u, u = live_v ? code_v(dv[x][j] * dir * dir) : 0u;
            om[x][j] = dm[x][j] < 0.0 ? 0u - q : q;
            ov[x][j] = u == 0 && dv[x][j] > 0.0 ? 1u : u;
          }
      }
    }
#pragma unroll
    for (int x = 0; x < V; ++x) {
      adam_store_codes(M, i[x], n[x], live_m ? low_bytes(om[x]) : 0u);
      adam_store_codes(U, i[x], n[x], live_v ? low_bytes(ov[x]) : 0u);
    }
    if ((lane & 31) == 0 && here) {
      scale_of_m[half] = fs;
      scale_of_v[half] = fr;
    }
    // the update by the root that v's code has and an estimated quotient, within a few last places; bc1 and bc2 come as
    // lr / bc1 and 1 / sqrt(bc2)
    const float up = (live_v ? fr : 1.f) * c.bc2, keep = 1.f - c.lr * c.wd;
#pragma unroll
    for (int x = 0; x < V; ++x)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        p[x][j] = __builtin_fmaf(-(m[x][j] * c.bc1), __builtin_amdgcn_rcpf(__builtin_fmaf(rv[x][j], up, c.eps)), p[x][j] * keep);
  } else {
    adam_load<BM>(M, i[0], n[0], m[0]);
    adam_load<BM>(U, i[0], n[0], v[0]);
#pragma unroll
    for (int j = 0; j < 4; ++j) adam_elem(c, p[0][j], g[0][j], m[0][j], v[0][j]);
    if constexpr (BM) {
      adam_store((unsigned short*)M, i[0], n[0], to_bf16x2(m[0][0], m[0][1]), to_bf16x2(m[0][2], m[0][3]));
      adam_store((unsigned short*)U, i[0], n[0], to_bf16x2(v[0][0], v[0][1]), to_bf16x2(v[0][2], v[0][3]));
    } else {
      adam_store((float*)M, i[0], n[0], m[0]);
      adam_store((float*)U, i[0], n[0], v[0]);
    }
  }
#pragma unroll
  for (int x = 0; x < V; ++x) {
    if constexpr (!GBF) {
      const float none[4] = {0.f, 0.f, 0.f, 0.f};
      if (a.clear) adam_store((float*)G, i[x], n[x], none);
    }
    if constexpr (PM == PM_F32 || PM == PM_BF16_MASTER) adam_store((float*)P, i[x], n[x], p[x]);
    unsigned short* O = (unsigned short*)t.p + base;
    if constexpr (PM == PM_BF16_SR) {
      unsigned o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = round_stochastic(p[x][j], t.seed, t.first + base + i[x] + j);
      adam_store(O, i[x], n[x], o[0] | o[1] << 16, o[2] | o[3] << 16);
    } else if constexpr (PM != PM_F32) {
      adam_store(O, i[x], n[x], to_bf16x2(p[x][0], p[x][1]), to_bf16x2(p[x][2], p[x][3]));
    }
  }
}
constexpr int STEP_THREADS = 256;
template <int MOM, int PM, bool GBF>
__global__ void __launch_bounds__(STEP_THREADS) adam_kernel(AdamTable a) {
  constexpr int WAVE = 256 * adam_vectors(MOM);  // elements of a wave
  const int ti = adam_tensor(a);
  const AdamTensorK& t = a.t[ti];
  const long long base = (long long)(blockIdx.x - a.first[ti]) * (4 * WAVE) + wave_uniform(threadIdx.x >> 6) * WAVE;
  if (base + WAVE <= t.n) adam_vector<MOM, PM, GBF, true>(a, t, base);
  else if (base < t.n) adam_vector<MOM, PM, GBF, false>(a, t, base);
}

// The fp32 values of 8-bit moments (into g: m's, into p: v's), a vector a thread.  150M: 237 us, 6.3 TB/s.
constexpr int VALUES_THREADS = 512;
__global__ void __launch_bounds__(VALUES_THREADS) adam_values_kernel(AdamTable a) {
  const int ti = adam_tensor(a);
  const AdamTensorK& t = a.t[ti];
  const long long block = (long long)(blockIdx.x - a.first[ti]) * adam_chunk(GL_MOMENTS_INT8) + wave_uniform(threadIdx.x >> 6) * ADAM_BLOCK;
  const unsigned i = 4 * (threadIdx.x & 63);
  const long long left = t.n - block - i;
  if (left <= 0) return;
  const int n = left > 4 ? 4 : (int)left;
  const unsigned cm = adam_load_codes((char*)t.m + block, i, n), cv = adam_load_codes((char*)t.v + block, i, n);
  const double sm = (double)t.m_scale[block / ADAM_BLOCK], sv = (double)t.v_scale[block / ADAM_BLOCK], sv2 = sv * sv;
  float m[4], v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m[j] = (float)(square_m(cm, j) * sm);
    v[j] = (float)(fourth_v(cv, j) * sv2);
  }
  adam_store((float*)t.g + block, i, n, m);
  adam_store((float*)t.p + block, i, n, v);
}

template <int MOM, int PM>
void launch_adam_as(bool gbf, dim3 grid, hipStream_t s, const AdamTable& a) {
  if (gbf) GL_LAUNCH(GL_KERNEL_ADAM, (adam_kernel<MOM, PM, true>), grid, dim3(STEP_THREADS), 0, s, a);
  else GL_LAUNCH(GL_KERNEL_ADAM, (adam_kernel<MOM, PM, false>), grid, dim3(STEP_THREADS), 0, s, a);
}
template <int MOM>
void launch_adam_of(int pm, bool gbf, dim3 grid, hipStream_t s, const AdamTable& a) {
  if (pm == PM_F32) launch_adam_as<MOM, PM_F32>(gbf, grid, s, a);
  else if (pm == PM_BF16_RNE) launch_adam_as<MOM, PM_BF16_RNE>(gbf, grid, s, a);
  else if (pm == PM_BF16_MASTER) launch_adam_as<MOM, PM_BF16_MASTER>(gbf, grid, s, a);
  else launch_adam_as<MOM, PM_BF16_SR>(gbf, grid, s, a);
}

// one launch for every ADAM_TENSORS of the tensors; `values`: their moments' values instead of a step
int launch_adam(const GlAdamArgs* a, const GlAdamTensor* tensors, int count, bool values, hipStream_t s) {
  AdamTable k{};
  k.lr = a->lr;
  k.b1 = a->beta1;
  k.b2 = a->beta2;
  k.eps = a->eps;
  k.wd = a->weight_decay;
  k.clear = !a->keep_g;
  k.b1d = a->beta1_64;
  k.a1d = 1.0 - a->beta1_64;
  k.b2d = a->beta2_64;
  k.a2d = 1.0 - a->beta2_64;
  // workgroups of a launch: 2^31 threads, of the 2^32 - 1 that one may have
  const long long most = (1LL << 31) / (values ? VALUES_THREADS : STEP_THREADS);
  const bool i8 = a->moments_dtype == GL_MOMENTS_INT8;
  const int chunk = adam_chunk(a->moments_dtype);
  int next = 0;
  long long done = 0;  // of the next tensor, which takes several launches where it has more chunks than one takes
  while (next < count) {
    long long groups = 0;
    k.count = 0;
    while (next < count && k.count < ADAM_TENSORS && groups < most) {
      const GlAdamTensor& t = tensors[next];
      const long long left = t.n - done, room = (most - groups) * chunk, n = left < room ? left : room;
      if (n > 0) {
        AdamTensorK& d = k.t[k.count];
        k.first[k.count++] = (unsigned)groups;
        const auto at = [&](void* p, int bytes) { return (void*)((char*)p + done * bytes); };
        const int pe = values || a->p_dtype == GL_DTYPE_F32 ? 4 : 2, ge = values || a->g_dtype == GL_DTYPE_F32 ? 4 : 2;
        const int me = i8 ? 1 : a->moments_dtype == GL_DTYPE_F32 ? 4 : 2;
        d = AdamTensorK{at(t.p, pe), at(t.g, ge), at(t.m, me), at(t.v, me), t.master ? t.master + done : nullptr,
                        i8 ? t.m_scale + done / ADAM_BLOCK : nullptr, i8 ? t.v_scale + done / ADAM_BLOCK : nullptr, n, done,
                        (unsigned long long)t.seed, t.bc1, t.bc2};
        if (i8) {  // as that update takes them
          d.bc1 = (float)((double)a->lr / t.bc1);
          d.bc2 = (float)(1.0 / __builtin_sqrt((double)t.bc2));
        }
        groups += (n + chunk - 1) / chunk;
      }
      done = n < left ? done + n : 0;
      next += n >= left;
    }
    if (groups == 0) continue;
    k.first[k.count] = (unsigned)groups;
    const dim3 grid((unsigned)groups);
    if (values) {
      GL_LAUNCH(GL_KERNEL_ADAM_VALUES, adam_values_kernel, grid, dim3(VALUES_THREADS), 0, s, k);
    } else {
      const int pm = a->p_dtype == GL_DTYPE_F32 ? PM_F32 : (k.t[0].master ? PM_BF16_MASTER : (a->stochastic ? PM_BF16_SR : PM_BF16_RNE));
      const bool gbf = a->g_dtype == GL_DTYPE_BF16;
      if (a->moments_dtype == GL_DTYPE_F32) launch_adam_of<GL_DTYPE_F32>(pm, gbf, grid, s, k);
      else if (a->moments_dtype == GL_DTYPE_BF16) launch_adam_of<GL_DTYPE_BF16>(pm, gbf, grid, s, k);
      else if (a->nearest_codes) launch_adam_of<MOMENTS_INT8_NEAREST>(pm, gbf, grid, s, k);
      else launch_adam_of<GL_MOMENTS_INT8>(pm, gbf, grid, s, k);
    }
    GL_CHECK_LAUNCH();
  }
  return 0;
}

int check_tensors(const GlAdamArgs* a, bool values) {
  if (a->count < 0 || !a->tensors) return GL_ERR_ARG;
  if (a->moments_dtype != GL_DTYPE_F32 && a->moments_dtype != GL_DTYPE_BF16 && a->moments_dtype != GL_MOMENTS_INT8)
    return GL_ERR_UNSUPPORTED;
  const bool i8 = a->moments_dtype == GL_MOMENTS_INT8;
  if (values && !i8) return GL_ERR_ARG;
  if (!values) {
    if ((a->p_dtype != GL_DTYPE_F32 && a->p_dtype != GL_DTYPE_BF16) || (a->g_dtype != GL_DTYPE_F32 && a->g_dtype != GL_DTYPE_BF16))
      return GL_ERR_UNSUPPORTED;
    if (a->p_dtype == GL_DTYPE_F32 && a->stochastic) return GL_ERR_ARG;  // fp32 parameters round nothing
  }
  const uintptr_t pe = values || a->p_dtype == GL_DTYPE_F32 ? 3 : 1, ge = values || a->g_dtype == GL_DTYPE_F32 ? 3 : 1;
  const uintptr_t me = i8 ? 0 : (a->moments_dtype == GL_DTYPE_F32 ? 3 : 1);
  int master = -1;  // not known yet
  for (int i = 0; i < a->count; ++i) {
    const GlAdamTensor& t = a->tensors[i];
    if (t.n < 0) return GL_ERR_ARG;
    if (t.n == 0) continue;
    if (t.n > GL_ADAM_MAX_ELEMENTS) return GL_ERR_UNSUPPORTED;
    if (!t.p || !t.g || !t.m || !t.v || (i8 && (!t.m_scale || !t.v_scale))) return GL_ERR_ARG;
    if (!values) {
      if (master >= 0 && (t.master != nullptr) != (master == 1)) return GL_ERR_ARG;
      master = t.master != nullptr;
      if (t.master && a->p_dtype == GL_DTYPE_F32) return GL_ERR_ARG;
    }
    if (((uintptr_t)t.p & pe) || ((uintptr_t)t.g & ge) || (((uintptr_t)t.m | (uintptr_t)t.v) & me) ||
        (((uintptr_t)t.master | (uintptr_t)t.m_scale | (uintptr_t)t.v_scale) & 3))
      return GL_ERR_ARG;
  }
  return 0;
}

}  // namespace gl

using namespace gl;

extern "C" int gl_adam_values(const GlAdamArgs* a, void* stream) {
  if (!a) return GL_ERR_ARG;
  GL_TRY(check_tensors(a, true));
  return launch_adam(a, a->tensors, a->count, true, (hipStream_t)stream);
}

extern "C" int gl_adam(const GlAdamArgs* a, void* stream) {
  if (!a) return GL_ERR_ARG;
  if (a->tensors) {
    GL_TRY(check_tensors(a, false));
    return launch_adam(a, a->tensors, a->count, false, (hipStream_t)stream);
  }
  if (a->n < 0) return GL_ERR_ARG;
  if (a->n == 0) return 0;
  if (!a->p || !a->g || !a->m || !a->v) return GL_ERR_ARG;
  if (a->moments_dtype != GL_DTYPE_F32 && a->moments_dtype != GL_DTYPE_BF16) return GL_ERR_UNSUPPORTED;
  if (a->p_dtype != GL_DTYPE_F32 && a->p_dtype != GL_DTYPE_BF16) return GL_ERR_UNSUPPORTED;
  if (a->p_dtype == GL_DTYPE_F32 && (a->master || a->stochastic)) return GL_ERR_ARG;  // fp32 parameters round nothing
  const bool f32p = a->p_dtype == GL_DTYPE_F32;
  // one tensor is at whole vectors: 16-byte fp32 streams, 8-byte bf16 streams
  const uintptr_t a16 = (uintptr_t)a->g | (f32p ? (uintptr_t)a->p : 0) | (uintptr_t)a->master;
  const uintptr_t a8 = f32p ? 0 : (uintptr_t)a->p;
  const uintptr_t alm = (uintptr_t)a->m | (uintptr_t)a->v;
  if ((a16 & 15) || (a8 & 7) || (alm & (a->moments_dtype == GL_DTYPE_F32 ? 15 : 7))) return GL_ERR_ARG;
  const GlAdamTensor t{a->p, a->g, a->m, a->v, a->master, nullptr, nullptr, a->n, a->seed, a->bc1, a->bc2};
  GlAdamArgs k = *a;
  k.g_dtype = GL_DTYPE_F32;
  k.keep_g = 0;
  return launch_adam(&k, &t, 1, false, (hipStream_t)stream);
}
