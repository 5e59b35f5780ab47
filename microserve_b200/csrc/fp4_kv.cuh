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

// Scale byte of a group whose largest |x| has the fp16 bits `amax` (0..0x7FFF).
__device__ __forceinline__ uint32_t fp4_scale_code(uint32_t amax) {
  if (amax > 0x7C00u) return kFp4NanScaleCode;
  const float a = fminf(__half2float(__ushort_as_half((unsigned short)amax)), 65504.f);
  const float v = __fdiv_rn(a, 6.f);
  uint32_t code;
  if (v < 6.103515625e-05f) {  // below 2^-14: steps of 2^-17
    code = (uint32_t)__float2int_rn(v * 131072.f);
  } else {  // keep 3 mantissa bits, ties to even; rebias 127 -> 15
    uint32_t b = __float_as_uint(v);
    b += 0x7FFFFu + ((b >> 20) & 1u);
    code = (b >> 20) - ((127u - 15u) << 3);
  }
  return min(code, (uint32_t)kFp4MaxScaleCode);
}

// Codes of 8 fp16 elements (4 words) under scale byte `sc`, packed in one word.
// x / s is taken as q0 = x * (1/s) and one correction by the remainder x - q0 s: exact
// where x / s is a rounding boundary (the only place where the last bit matters).
__device__ __forceinline__ uint32_t fp4_encode8(const uint32_t (&h)[4], uint32_t sc) {
  if (sc == (uint32_t)kFp4NanScaleCode) return 0u;
  const float s = __half2float(__ushort_as_half((unsigned short)(sc << 7)));
  const float r = sc == 0 ? 0.f : __frcp_rn(s);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __half2 p;
    memcpy(&p, &h[i], 4);
    float2 f = __half22float2(p);
    f.x = fminf(fmaxf(f.x, -65504.f), 65504.f);
    f.y = fminf(fmaxf(f.y, -65504.f), 65504.f);
    const float qx = __fmul_rn(f.x, r), qy = __fmul_rn(f.y, r);
    // the sign of a zero (or of a quotient that rounds to zero) is x's
    const float cx = copysignf(__fmaf_rn(__fmaf_rn(-qx, s, f.x), r, qx), f.x);
    const float cy = copysignf(__fmaf_rn(__fmaf_rn(-qy, s, f.y), r, qy), f.y);
    uint32_t b;
    asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tcvt.u32.u8 %0, t;\n\t}"
        : "=r"(b)
        : "f"(cy), "f"(cx));
    w |= b << (8 * i);
  }
  return w;
}

}  // namespace ms
