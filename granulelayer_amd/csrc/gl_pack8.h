// The 8-bit form of an activation tensor, shared by the kernels that write and read it.
//
// Along a row, blocks of 32 values share a power of two (the last block of a row may be shorter).
// With a = max |x| over the block:
//     e    = ((bits(a) + 0x10000) >> 23) - 6, between 1 and 248    stored, one byte a block
//     step = 2^(e - 127)
//     q    = rint(x / step), between -127 and 127                  stored, one byte a value
// a lies in [64, 128) steps; the added 0x10000 carries a's whose quotient would round to 128
// (mantissas of 127.5 / 64 and more) into the next power, so |x - q step| <= step / 2 for every
// value; only the last 1/256 below the largest fp32 number is cut to 127 steps (a step more would
// be past fp32).  Scaling by a power of two is exact, so q does not depend on the order or width of any
// arithmetic, and q step has 7 significant bits: it is exact in bf16 as well as in fp32.  A block
// that holds an infinity or a NaN has e = 255 and reads back as NaN.
#pragma once

#include "gl_common.h"

namespace gl {

constexpr int P8_BLOCK = 32;

// e of a block whose largest |x| has the bits `amax` (integer order is the values' order, with the
// infinities and NaN above every number)
__device__ __forceinline__ int p8_exp(unsigned amax) {
  if (amax >= 0x7f800000u) return 255;
  const int e = (int)((amax + 0x10000u) >> 23) - 6;
  return e < 1 ? 1 : (e > 248 ? 248 : e);
}
// 1 / step; 0 for a block without a finite maximum (its codes stand for nothing)
__device__ __forceinline__ float p8_inv_step(int e) { return e == 255 ? 0.f : __uint_as_float((unsigned)(254 - e) << 23); }
__device__ __forceinline__ float p8_step(int e) { return __uint_as_float(e == 255 ? 0x7fc00000u : (unsigned)e << 23); }

// Four codes.  1.5 x 2^23 has a last place of one: adding it rounds to a whole number (nearest even) and
// leaves it in the low byte, two's complement; the product is exact, so the fused add rounds once.
__device__ __forceinline__ unsigned p8_code(float x, float inv_step) {
  constexpr float LIMIT = 127.f * 0x1p121f;  // of the largest step
  return __float_as_uint(__builtin_fmaf(__builtin_amdgcn_fmed3f(x, -LIMIT, LIMIT), inv_step, 12582912.f));
}
__device__ __forceinline__ unsigned p8_codes4(float a, float b, float c, float d, float inv_step) {
  const unsigned lo = __builtin_amdgcn_perm(p8_code(b, inv_step), p8_code(a, inv_step), 0x0c0c0400u);
  const unsigned hi = __builtin_amdgcn_perm(p8_code(d, inv_step), p8_code(c, inv_step), 0x04000c0cu);
  return lo | hi;
}
// value i of four packed codes
__device__ __forceinline__ float p8_value(unsigned codes, int i, float step) {
  return (float)((int)(codes << (24 - 8 * i)) >> 24) * step;
}

__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }

// ---- bf16 and fp32 storage -----------------------------------------------------------------------
// nearest even; the inputs' own conversion, NaN included
__device__ __forceinline__ unsigned short to_bf16(float x) {
  return __builtin_bit_cast(unsigned short, __float2bfloat16(x));
}
__device__ __forceinline__ unsigned to_bf16x2(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
}
// vectors at an element's own alignment: global memory takes 8- and 16-byte accesses at any address
// that is a multiple of the element's size
typedef unsigned uv2 __attribute__((ext_vector_type(2)));
typedef unsigned uv4 __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(2))) bytes16 { uv4 v; };
struct __attribute__((packed, aligned(2))) bytes8 { uv2 v; };

// eight values from p (element type T) into fp32, of which the first n are there and the rest are 0
template <bool BF>
__device__ __forceinline__ void load8(const void* p, long long i, int n, float (&v)[8]) {
  if (n >= 8) {
    if constexpr (BF) {
      const uv4 w = reinterpret_cast<const bytes16*>((const char*)p + 2 * i)->v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uv4 w = reinterpret_cast<const bytes16*>((const char*)p + 4 * i + 16 * h)->v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * h + j] = __uint_as_float(w[j]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? ld_param_t<BF>((const float*)p, i + j) : 0.f;
  }
}
template <bool BF>
__device__ __forceinline__ void store8(void* p, long long i, int n, const float (&v)[8]) {
  if (n >= 8) {
    if constexpr (BF) {
      uv4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = to_bf16x2(v[2 * j], v[2 * j + 1]);
      reinterpret_cast<bytes16*>((char*)p + 2 * i)->v = w;
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uv4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(v[4 * h + j]);
        reinterpret_cast<bytes16*>((char*)p + 4 * i + 16 * h)->v = w;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) {
        if constexpr (BF) ((unsigned short*)p)[i + j] = to_bf16(v[j]);
        else ((float*)p)[i + j] = v[j];
      }
  }
}

// enqueue the unpack of [rows, cols] codes / exponents (contiguous, rows of round_up(cols, 32) codes)
// into x, rows sx elements apart
int launch_unpack8(const uint8_t* q, const uint8_t* e, long long rows, int cols, void* x, long long sx, int x_dtype,
                   hipStream_t s);

}  // namespace gl
