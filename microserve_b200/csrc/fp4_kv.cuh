// The 4-bit KV-cache format ("fp4_e2m1"), shared by its writer, reader and attentions.
//
// Per (token, kv head) of head_dim 128: 128 codes e2m1 (1 sign, 2 exponent, 1 mantissa
// bit: 0 .5 1 1.5 2 3 4 6), element 2i in the low nibble of byte i (64 bytes), and 8
// scale bytes, one per 16 elements. A scale byte is an unsigned float of 5 exponent and
// 3 mantissa bits, the top bits of an fp16 number: its fp16 value has the bits byte << 7
// (subnormals included), so a reader decodes it with a shift, and the fp16 exponent
// range (2^-17 .. 61440) makes a second scale per token unnecessary for fp16 data.
//   a = max |x| of the 16,  s = min(rn(a / 6), 10240),  code = rn(x / s), saturating at 6
// with ties to even in both roundings. 10240 is the largest scale for which 6 s is a
// finite fp16 number. Every value code * s has at most 6 significant bits and is exact
// in fp16, subnormal or not (smallest: 0.5 * 2^-17), so attention multiplies codes by
// scales in fp16 without rounding. Infinities count as the largest fp16 number; a group
// that holds a NaN gets the scale byte 0xFF (fp16 NaN) and zero codes, so a NaN reaches
// the reader as NaNs of that group. A group whose max is below 6 * 2^-18 rounds to scale 0.
//
// Codes and scales are bit-exact whatever the arithmetic: x has 11 significant bits, a
// rounding boundary of x / s at most 3 + 4, so unequal x and boundary differ by more than
// 2^-12 relative, far above fp32's error, and equal ones are found exactly (encode8).
//
// Cache: codes [num_blocks, kv_heads, block_size, 64], scales [num_blocks, kv_heads,
// block_size, 8]. The tokens of one head are contiguous within a page, so an attention
// tile of 64 tokens is one 4 KB piece of codes and one 512-byte piece of scales.
#pragma once

#include "common.cuh"

namespace ms {

constexpr int kFp4Dim = 128;         // head_dim
constexpr int kFp4RowBytes = 64;     // codes of one (token, head)
constexpr int kFp4ScaleBytes = 8;    // scales of one (token, head)
constexpr int kFp4MaxScaleCode = 226;  // 10240
constexpr int kFp4NanScaleCode = 255;

// 8 codes (one 32-bit word) -> 4 half2 in element order, exact (no scale applied).
__device__ __forceinline__ void fp4x8_to_f16x2(uint32_t w, uint32_t (&o)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
      : "r"(w));
}

__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Scale byte in both halves of an f16x2.
__device__ __forceinline__ uint32_t fp4_scale_h2(uint32_t byte) { return byte * 0x00800080u; }

// Pairs of floats in one 64-bit register: one instruction for two.
__device__ __forceinline__ uint64_t f32x2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Softmax references are kept as scores r, and a weight is 2^((s - r) c + b) (c: the softmax scale times log2 e, b: a
// constant). s c - (r c - b) is one fma a score, but r c is rounded by 2^-24 of itself, a factor that all weights
// of a row share: harmless until it drives a weight out of f16's range. So where |r| c is above this, s - r is formed first.
constexpr float kFarScore = 4194304.f;  // 2^22: the factor is below 2^(1/4)
__device__ __forceinline__ bool far_score(float r, float c) {
  return fabsf(r) * c > kFarScore && fabsf(r) < INFINITY;  // (r infinite: nothing seen yet, or an infinite query)
}

// Scale byte of a group whose largest |x| has the fp16 bits `amax` (0..0x7FFF).
// a / 6 is taken as a * h + a * l with h + l = 1/6 to 48 bits: exact where it is a rounding
// boundary (5 bits), right to 2^-24 elsewhere.
__device__ __forceinline__ uint32_t fp4_scale_code(uint32_t amax) {
  constexpr float kSixthHi = 1.f / 6.f, kSixthLo = (float)(1.0 / 6.0 - (double)kSixthHi);
  const float a = __half2float(__ushort_as_half((unsigned short)min(amax, 0x7BFFu)));
  const float v = __fmaf_rn(a, kSixthHi, __fmul_rn(a, kSixthLo));
  // keep 3 mantissa bits, ties to even; rebias 127 -> 15
  uint32_t b = __float_as_uint(v);
  b += 0x7FFFFu + ((b >> 20) & 1u);
  const uint32_t normal = (b >> 20) - ((127u - 15u) << 3);
  const uint32_t tiny = (uint32_t)__float2int_rn(v * 131072.f);  // below 2^-14: steps of 2^-17
  const uint32_t code = min(v < 6.103515625e-05f ? tiny : normal, (uint32_t)kFp4MaxScaleCode);
  return amax > 0x7C00u ? (uint32_t)kFp4NanScaleCode : code;
}

// Codes of 8 fp16 elements (4 words) under scale byte `sc`, packed in one word; amax as above.
// x / s is taken as x * h + x * l with h + l = 1 / s to 48 bits: exact where it is a rounding
// boundary (the only place where the last bit matters).
__device__ __forceinline__ uint32_t fp4_encode8(const uint32_t (&x)[4], uint32_t sc, uint32_t amax) {
  uint32_t h[4] = {x[0], x[1], x[2], x[3]};
  if (amax >= 0x7C00u) {  // rare
    if (amax > 0x7C00u) return 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // an infinity counts as the largest number
      if ((h[i] & 0x7FFFu) == 0x7C00u) h[i] -= 1u;
      if ((h[i] & 0x7FFF0000u) == 0x7C000000u) h[i] -= 0x10000u;
    }
  }
  const float s = __half2float(__ushort_as_half((unsigned short)(sc << 7)));
  const float r = sc == 0 ? 0.f : __frcp_rn(s);
  const float rl = __fmul_rn(__fmaf_rn(-r, s, 1.f), r);
  const uint64_t r2 = f32x2(r, r), l2 = f32x2(rl, rl);
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __half2 p;
    memcpy(&p, &h[i], 4);
    const float2 f = __half22float2(p);
    const uint64_t f2 = f32x2(f.x, f.y);
    float qx, qy;
    unpack2(fma2(f2, r2, mul2(f2, l2)), qx, qy);
    qx = copysignf(qx, f.x);  // the sign of a zero is x's
    qy = copysignf(qy, f.y);
    asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tcvt.u32.u8 %0, t;\n\t}"
        : "=r"(b[i])
        : "f"(qy), "f"(qx));
  }
  return prmt(prmt(b[0], b[1], 0x0040u), prmt(b[2], b[3], 0x0040u), 0x5410u);
}

}  // namespace ms
