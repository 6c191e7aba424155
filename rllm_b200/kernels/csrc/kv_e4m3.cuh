// A cache kept in 8 bits: what its writer, its reader and its attention share.
//
// A row (a token's key or value of one kv head, d numbers x_i) is kept as d e4m3 numbers c_i and one power of two 2^e,
// x_i ~ c_i 2^e.  e is the least whole number with max|x_i| <= 448 * 2^e (448: the largest e4m3 number), at least -127;
// c_i is x_i 2^-e rounded once, to the nearest with ties to even.  2^-e is exact in float32, so that rounding is the only
// one, and nothing saturates.  The scale is kept as a byte, e + 127 (e8m0): 255, which stands for NaN, marks a row that had
// an infinity or a NaN; its numbers are then zeros, and everything that is computed from the row is NaN.
//
// A power of two rather than max / 448: the rounding of a floating type is relative, so the scale's finer steps would buy
// nothing but at the subnormal end (numbers below 2^-14 of the row's largest), and with it a row's values are exact in
// bfloat16 and its scale can be moved between factors without a rounding.
//
// Layout: codes [pages, kv heads, page size, d], one byte each, and scales [pages, kv heads, page size], for keys and for
// values.  The rows of a (page, head) follow one another.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#define KV8_NAN_SCALE 255

// What a kernel of the attention may take for granted of the kernel ahead of it in the stream (`known`):
//   KV8_ANY      nothing.  The kernel ahead may be the one that makes the step's lengths, row ranges and block table (decode_advance lets
//                the next kernel in and then counts the lengths up), so they too are read behind the wait for it (kv8_inputs).
//   KV8_LENGTHS  it leaves those alone: every kernel but the one directly ahead is complete when this one starts, so they are read, and
//                tiles looked up, while that one ends.
//   KV8_BESIDE   it is the first kernel of the same call, of which this one reads nothing (the portions' attention behind the single
//                tokens').  This one does not wait before it begins but before it ends: what was written ahead of both is there when it
//                starts, for the first has let it in behind its own wait, and whoever comes after it finds both complete.  It lets
//                nobody in itself.
#define KV8_ANY 0
#define KV8_BESIDE 1
#define KV8_LENGTHS 2
template <typename... P>
__device__ __forceinline__ void kv8_inputs(int known, P&... ptrs) {
  if (known == KV8_ANY) {
    pdl_wait();
    (pdl_fresh_in_place(ptrs), ...);
  }
}
template <typename... P>
__device__ __forceinline__ void kv8_begin(int known, P&... ptrs) {
  if (known != KV8_BESIDE) pdl_wait();
  (pdl_fresh_in_place(ptrs), ...);
}
__device__ __forceinline__ void kv8_let_in(int known) { if (known != KV8_BESIDE) pdl_launch(); }
__device__ __forceinline__ void kv8_end(int known) { if (known == KV8_BESIDE) pdl_wait(); }

// the scale byte of a row whose largest magnitude is `top` (finite): (bits + 0x1FFFFF) >> 23 is top's biased exponent, one
// more where its mantissa lies above 1.75 = 448 / 256
__device__ __forceinline__ int kv8_scale_byte(float top) {
  const int e = (int)((__float_as_uint(top) + 0x1FFFFFu) >> 23) - 8;
  return e > 0 ? e : 0;
}
// 2^-e of a byte (0 .. 247): a normal float32
__device__ __forceinline__ float kv8_inverse(int byte) { return __uint_as_float((unsigned)(254 - byte) << 23); }
// 2^e of a byte; NaN for 255
__device__ __forceinline__ float kv8_power(int byte) {
  const unsigned bits = byte == 0 ? 0x00400000u : (byte == KV8_NAN_SCALE ? 0x7FC00000u : (unsigned)byte << 23);
  return __uint_as_float(bits);
}
// 2^x of a whole x of up to 127; 0 where it is below the normal numbers'
__device__ __forceinline__ float kv8_two_to(float x) {
  return __uint_as_float((unsigned)((int)fminf(fmaxf(x, -127.f), 127.f) + 127) << 23);
}
// A row's two references, top of its scores and high, relative to top, of its weights with their values' powers, joined with those of another
// part of its keys
__device__ __forceinline__ void kv8_join(float& top, float& high, float m, float t) {
  const float both = fmaxf(top, m);
  high = fmaxf(high + (top - both), t + (m - both));
  top = both;
}
// two numbers as e4m3, the first in the low byte
__device__ __forceinline__ unsigned kv8_pack2(float a, float b) {
  return (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ unsigned kv8_pack4(float a, float b, float c, float d) { return kv8_pack2(a, b) | (kv8_pack2(c, d) << 16); }
// the two e4m3 numbers of 16 bits as a pair of halves (exact)
__device__ __forceinline__ unsigned kv8_halves(unsigned short two) {
  unsigned r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(two));
  return r;
}
__device__ __forceinline__ unsigned kv8_halves_lo(unsigned four) { return kv8_halves((unsigned short)(four & 0xffffu)); }
__device__ __forceinline__ unsigned kv8_halves_hi(unsigned four) { return kv8_halves((unsigned short)(four >> 16)); }
__device__ __forceinline__ void kv8_floats(unsigned four, float* o) {
  const unsigned lo = kv8_halves_lo(four), hi = kv8_halves_hi(four);
  const float2 a = __half22float2(*(const __half2*)&lo), b = __half22float2(*(const __half2*)&hi);
  o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y;
}
