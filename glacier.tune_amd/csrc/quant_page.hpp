// quant_page.hpp -- device side of the 4-bit formats: a cache's groups of 32
// columns as they are quantised and read, and words of eight numbers unpacked for
// the matrix cores.
//
// A number n (0 .. 15) stands for (n - 8) s.  s has five significant bits and n - 8
// three, so a held value is exact in bf16 and in fp16, and no kernel rounds it.  A
// word's eight numbers lie so that (word >> 4 j) & 0x000f000f are neighbouring
// columns 2 j and 2 j + 1 in the two halves of a register: one more OR makes them
// floats 128 + n (bf16) or 1024 + n (fp16; bits 4 to 7 of a half 64 + n), exact, without
// a conversion.
#pragma once

#include "attn_common.hpp"
#include "quant_launch.hpp"

namespace glacier {

constexpr float kQuantScaleMax = 2688.0f;  // the format's largest scale: 21 x 2^7, five bits
constexpr unsigned kQuantNan = 0x7e00u;    // scale of a group that is not finite
constexpr unsigned kQuantZero = 0x88888888u;  // a word of zeros

typedef _Float16 f16;
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

__device__ inline float half_at(unsigned w, int hi) {  // fp16 in a register's half
  return (float)__builtin_bit_cast(f16x2, w)[hi];
}

// s (fp32) at five significant bits, ties to even, within +-kQuantScaleMax, as fp16.
__device__ inline f16 quant_scale(float s) {
  unsigned u = __builtin_bit_cast(unsigned, s);
  u = (u + 0x3ffffu + ((u >> 19) & 1u)) & ~0x7ffffu;
  return (f16)fminf(fmaxf(__builtin_bit_cast(float, u), -kQuantScaleMax), kQuantScaleMax);
}

// The number of x: floor(x / s + 1/2) + 8 within 0 .. 15.  size: |s|; sign: s's sign bit;
// inv: about 1 / |s|.  The product may land on the wrong side of a border: it is held
// below it (by more than its error), and the remainder tells whether x has passed it (it
// is exact there: x and n s agree in their leading bits).
__device__ inline unsigned quant_number(float x, unsigned sign, float size, float inv) {
  x = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) ^ sign);
  const float n = floorf(fmaf(x, inv, 0.5f - 0x1p-18f));
  const float up = fmaf(-n, size, x) >= 0.5f * size ? 9.0f : 8.0f;
  return static_cast<unsigned>(fminf(fmaxf(n + up, 0.0f), 15.0f));
}

// Eight columns (of a group of 32 that four neighbouring lanes hold) as a word and
// the group's scale.
__device__ inline unsigned quantise8(const float (&x)[8], f16& scale) {
  float top = x[0], low = x[0], zero = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    top = fmaxf(top, x[e]);
    low = fminf(low, x[e]);
    zero = fmaf(x[e], 0.0f, zero);  // NaN where an element is not finite
  }
#pragma unroll
  for (int d = 1; d < 4; d *= 2) {
    top = fmaxf(top, __shfl_xor(top, d));
    low = fminf(low, __shfl_xor(low, d));
    zero += __shfl_xor(zero, d);
  }
  const bool odd = zero != 0.0f;
  scale = odd ? __builtin_bit_cast(f16, static_cast<unsigned short>(kQuantNan))
              : quant_scale((top >= -low ? top : low) * -0.125f);
  const float s = (float)scale;
  if (odd || s == 0.0f) return kQuantZero;
  const unsigned sign = __builtin_bit_cast(unsigned, s) & 0x80000000u;
  const float size = fabsf(s), inv = __builtin_amdgcn_rcpf(size);
  unsigned w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) w |= quant_number(x[e], sign, size, inv) << (4 * (e / 2) + 16 * (e % 2));
  return w;
}

// A word's columns as floats (n - 8) s.
__device__ inline void dequantise8(unsigned w, float s, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    x[e] = (float)(static_cast<int>((w >> (4 * (e / 2) + 16 * (e % 2))) & 15u) - 8) * s;
}

// Where a token's head lies in a page's head part of 18 G P bytes: `row` the token's
// place in the page.  Words in units of 4 bytes, scales in units of 2 behind them.
__device__ inline int k_word(int row, int G, int col8) { return (row * 4 + col8 % 4) * G + col8 / 4; }
__device__ inline int k_scale(int row, int G, int i) { return row * G + i; }
__device__ inline int v_word(int row, int G, int col8) { return ((row >> 2) * 4 * G + col8) * 4 + (row & 3); }
__device__ inline int v_scale(int row, int G, int i) { return ((row >> 2) * G + i) * 4 + (row & 3); }

// The constants of raw numbers: a register each, since and-or takes one constant from
// elsewhere only (as a literal each would be an operation of its own).
struct QuantMagic {
  unsigned bf128 = 0x43004300u;  // bf16 128
  unsigned h1024 = 0x64006400u, h64 = 0x54005400u;  // fp16 1024, 64
  __device__ inline QuantMagic() {
    asm("" : "+v"(bf128));
    asm("" : "+v"(h1024));
    asm("" : "+v"(h64));
  }
};
// Two numbers n, n' (in bits 0-3 and 16-19 of w >> shift) as bf16 128 + n, 128 + n'.
__device__ inline unsigned pair_bf16(unsigned w, int shift, const QuantMagic& c) {
  return ((w >> shift) & 0x000f000fu) | c.bf128;
}
// A word's columns as a bf16 operand of 128 + n.
__device__ inline bf16x8 raw8_bf16(unsigned w, const QuantMagic& c) {
  return __builtin_bit_cast(bf16x8, u32x4{pair_bf16(w, 0, c), pair_bf16(w, 4, c), pair_bf16(w, 8, c), pair_bf16(w, 12, c)});
}
// Upper halves of two floats (bf16 values) as a pair.
__device__ inline unsigned upper_pair(float lo, float hi) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, hi), __builtin_bit_cast(unsigned, lo), 0x07060302u);
}
// A word's columns as a bf16 operand of n - 8.
__device__ inline unsigned exact_pair(unsigned w, int shift, const QuantMagic& c) {
  const unsigned p = pair_bf16(w, shift, c);
  return upper_pair(__builtin_bit_cast(float, p << 16) - 136.0f, __builtin_bit_cast(float, p & 0xffff0000u) - 136.0f);
}
__device__ inline bf16x8 exact8_bf16(unsigned w, const QuantMagic& c) {
  return __builtin_bit_cast(bf16x8, u32x4{exact_pair(w, 0, c), exact_pair(w, 4, c), exact_pair(w, 8, c), exact_pair(w, 12, c)});
}

}  // namespace glacier
