// What the kernels of the 8-bit and 4-bit formats share.
//
// 8 bits: a row is e4m3 codes and one fp32 scale, value = code * scale, scale = max(max |x|, 2^-100) / 448, so that the row's largest
// entry becomes e4m3's largest value. The lower bound keeps an all-zero row (and one of nothing but entries too small to matter) away
// from a division by zero; its codes are zeros or tiny. A code is rounded to nearest (ties to even): off by at most 2^-4 of its value.
//
// 4 bits: entry (n, k) of a matrix is scales[n, k / group] * (q - z), q in 0 .. 15, z = zeros[n, k / group] or 8. Eight entries of a row
// share an int32 word, entry i of the eight at bit 4 (i / 2) + 16 (i % 2): neighbours lie sixteen bits apart, so that one mask takes a
// neighbouring pair out of a word into the two halves of a register, where the pairs of 16-bit types live.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#define SI_E4M3_MAX 448.f
#define SI_Q8_LEAST 7.888609052210118e-31f      // 2^-100

// What a row's entries are divided by on their way to codes: y / scale, rounded to fp32 as a division would, then to e4m3. A product with the inverse rounded
// to fp32 is up to two units off, and puts entries halfway between two codes on either side: of bf16 entries below a bf16 maximum one in 3,000. So the inverse
// is kept in two parts, the hardware's approximation (2^-23) and what is left of one behind it; the fused sum of their products with y is off by half a unit
// and 2^-45 of the value, and exact where the quotient is. Two entries at a time: as many instructions as one product an entry. The scale's own quotient is a
// product and its exact remainder. An infinite maximum leaves zeros, and NaN of infinite entries.
struct Q8Row {
  float scale, inverse, rest;
  __device__ __forceinline__ explicit Q8Row(float amax) {
    constexpr float part = 1.f / SI_E4M3_MAX;
    amax = fmaxf(amax, SI_Q8_LEAST);
    const bool finite = amax <= 3.4028234663852886e38f;
    const float q = amax * part;
    scale = finite ? __fmaf_rn(__fmaf_rn(q, -SI_E4M3_MAX, amax), part, q) : amax;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(scale));
    rest = finite ? __fmaf_rn(-inverse, scale, 1.f) * inverse : 0.f;
  }
  __device__ __forceinline__ float operator()(float y) const { return __fmaf_rn(y, inverse, y * rest); }
  __device__ __forceinline__ void operator()(float& a, float& b) const {
    asm("{\n.reg .b64 y, f, g;\nmov.b64 y, {%0, %1};\nmov.b64 f, {%2, %2};\nmov.b64 g, {%3, %3};\n"
        "mul.rn.f32x2 g, y, g;\nfma.rn.f32x2 y, y, f, g;\nmov.b64 {%0, %1}, y;\n}\n" : "+f"(a), "+f"(b) : "f"(inverse), "f"(rest));
  }
};
// A product's sum times the row's and the column's scale. Scales reach from 2^-100 / 448 to 2^119 and a sum from 2^-18 up, so that each of the two
// orders in fp32 loses some result that is an ordinary number: the product of the scales may be subnormal, zero or infinite, and so may the sum times
// one of them. Where the product of the scales is a normal number it is taken; else 64 bits are, which hold all of it.
__device__ __forceinline__ bool q8_normal(float p) { return fabsf(p) >= 1.1754943508222875e-38f && fabsf(p) <= 3.4028234663852886e38f; }
__device__ __forceinline__ float q8_scaled_wide(float sum, float sa, float sw) { return (float)((double)sum * (double)sa * (double)sw); }
__device__ __forceinline__ float q8_scaled(float sum, float sa, float sw) {
  const float p = sa * sw;
  return q8_normal(p) ? sum * p : q8_scaled_wide(sum, sa, sw);
}
// The least and the largest size of the scales s[from .. to), for every lane of a warp (as whole numbers, which order sizes alike; NaN is the largest). A
// tile asks once, before it waits for its sums: with a test an output 61 x 28,672 x 4,096 took 27.0 us for 24.5.
__device__ __forceinline__ float2 q8_range(const float* s, int from, int to) {
  unsigned least = 0x7fffffffu, most = 0;
  for (int i = from + (int)(threadIdx.x & 31); i < to; i += 32) {
    const unsigned b = __float_as_uint(s[i]) & 0x7fffffffu;
    least = min(least, b);
    most = max(most, b);
  }
  return make_float2(__uint_as_float(__reduce_min_sync(0xffffffffu, least)), __uint_as_float(__reduce_max_sync(0xffffffffu, most)));
}
// Whether the product of `scale` and any of that range is a normal number.
__device__ __forceinline__ bool q8_plain(float scale, float2 range) { return q8_normal(scale * range.x) && q8_normal(scale * range.y); }

__device__ __forceinline__ unsigned q8_pack2(float a, float b) {      // two codes, a in the low byte
  return (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint2 q8_pack8(const Q8Row& to, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) to(v[i], v[i + 1]);
  return make_uint2(q8_pack2(v[0], v[1]) | (q8_pack2(v[2], v[3]) << 16), q8_pack2(v[4], v[5]) | (q8_pack2(v[6], v[7]) << 16));
}
__device__ __forceinline__ unsigned char q8_pack1(const Q8Row& to, float a) { return (unsigned char)__nv_cvt_float_to_fp8(to(a), __NV_SATFINITE, __NV_E4M3); }

// Pair p (entries 2p, 2p + 1) of a word of eight 4-bit entries as two bf16 of value 128 + q: bf16 counts in ones from 128 to 255, so
// the four bits go straight into the mantissa (a widely known way of widening 4-bit entries; the constants follow from the two formats).
// (Written as one instruction: the compiler makes two of the mask and the or, and such instructions are what bounds the kernels that widen.)
__device__ __forceinline__ unsigned w4_pair_raw(unsigned word, int p) {
  unsigned v;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;\n" : "=r"(v) : "r"(word >> (4 * p)), "r"(0x000f000fu), "r"(0x43004300u));
  return v;
}
// The same less 128 + z, exact: `bias` holds 128 + z twice.
__device__ __forceinline__ unsigned w4_pair(unsigned word, int p, __nv_bfloat162 bias) {
  const unsigned raw = w4_pair_raw(word, p);
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&raw), bias);
  return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ __nv_bfloat162 w4_bias(int z) { return __float2bfloat162_rn(128.f + (float)z); }
