// Rows in 4-bit floating point: the one rule by which activations, weights, keys and values are quantised.
//
// A row x (a token's activations, an output channel of a weight, a token's key or value of one head), a = max(max |x|, 2^-100):
//   E      the least exponent with a <= 2688 * 2^E, -111 .. 117, kept as the byte E + 127 (255: a row with an infinity or a NaN)
//   b      of each block of 16 values: e4m3(max |x| of the block / (6 * 2^E)), at most 448 (2688 = 6 * 448)
//   code   e2m1(x / (2^E * b)), at most 6; 0 where b is 0
// Both roundings are to the nearest, ties to even; quotients are rounded to float32 first, as torch divides tensors.  A code
// stands for code * b * 2^E, exactly (6 digits).  2^E being a power of two, the only roundings are those of b and of the code, so
// that all paths make the same codes, and so does the same rule in 64 bits but for quotients within 2^-24 of a tie.
// Dividing by b is a product with its reciprocal and one correction step: with a correctly rounded reciprocal the result is
// the correctly rounded quotient (Markstein's theorem), in three instructions a value.
#pragma once

#include "common.cuh"

constexpr int FP4_BLOCK = 16;
constexpr float FP4_ROW_FLOOR = 7.888609052210118e-31f;      // 2^-100
constexpr unsigned FP4_NO_NUMBER = 255;                      // exponent byte of a row that holds no finite numbers

// The exponent byte of a row, from the largest |x| as an unsigned number (infinities and NaN order above every finite one).
__device__ __forceinline__ unsigned fp4_row_exponent(unsigned bits) {
  if (bits >= 0x7f800000u) return FP4_NO_NUMBER;
  bits = max(bits, __float_as_uint(FP4_ROW_FLOOR));
  return (bits >> 23) - 11u + ((bits & 0x7fffffu) > 0x280000u ? 1u : 0u);      // 2688 = 1.3125 * 2^11
}
// 2^(byte - 127), NaN for 255
__device__ __forceinline__ float fp4_unit(unsigned byte) {
  return __uint_as_float(byte == FP4_NO_NUMBER ? 0x7fc00000u : byte == 0 ? 0x00400000u : byte << 23);
}
// 2^(127 - byte) for a byte that the rule makes (16 .. 244; 0 for 255)
__device__ __forceinline__ float fp4_down(unsigned byte) {
  return byte == FP4_NO_NUMBER ? 0.f : __uint_as_float((254u - byte) << 23);
}
__device__ __forceinline__ unsigned fp4_magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// e4m3 of a number from 0 to 448, and back
__device__ __forceinline__ unsigned fp4_scale_code(float x) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(x));
  return r;
}
__device__ __forceinline__ float fp4_scale_value(unsigned code) {
  unsigned two;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(two) : "h"((unsigned short)code));
  float y;
  asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.f32.f16 %0, lo; }" : "=f"(y) : "r"(two));
  return y;
}
// x / d for a constant d, correctly rounded where x is not within 2^-24 of the smallest normal numbers
__device__ __forceinline__ float fp4_divide(float x, float d, float inv) {
  const float q = x * inv;
  return fmaf(fmaf(-q, d, x), inv, q);
}
// The scale's code of a block whose largest |x| is `top` (finite, or down is 0).
__device__ __forceinline__ unsigned fp4_block_scale(unsigned top, float down) {
  if (down == 0.f) return 0;
  return fp4_scale_code(fp4_divide(__uint_as_float(top) * down, 6.f, 1.f / 6.f));
}
// Eight values' codes, the first in the lowest four bits.
__device__ __forceinline__ unsigned fp4_pack8(const float* y) {
  unsigned r;
  asm("{\n\t"
      ".reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t"
      "}" : "=r"(r) : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  return r;
}
// four values' codes in the low 16 bits
__device__ __forceinline__ unsigned fp4_pack4(const float* y) {
  const float x[8] = {y[0], y[1], y[2], y[3], 0.f, 0.f, 0.f, 0.f};
  return fp4_pack8(x) & 0xffffu;
}
// What the values of a block are divided by, 2^E b (2^-120 .. 448 * 2^117), and its reciprocal (0: all codes are 0).  Both are
// exact multiples, by a power of two, of b and of b's rounded reciprocal: the division rounds as that of x 2^-E by b does.
struct Fp4Scaler {
  float b, inv;
};
__device__ __forceinline__ Fp4Scaler fp4_scaler(unsigned scale_code, float down) {
  Fp4Scaler s;
  const float b = fp4_scale_value(scale_code);
  s.b = b * __uint_as_float(0x7f000000u - __float_as_uint(down));
  s.inv = scale_code == 0 ? 0.f : __frcp_rn(b) * down;
  return s;
}
__device__ __forceinline__ float fp4_quotient(float x, const Fp4Scaler& s) { return fp4_divide(x, s.b, s.inv); }
// Eight codes of values of one block, two values a product.  (A block of zeros, and one of a row without finite numbers: codes of
// zero, whatever 0 times an infinity makes.)
__device__ __forceinline__ unsigned fp4_codes8(const float* x, const Fp4Scaler& s) {
  if (s.inv == 0.f) return 0;
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    asm("{\n\t"
        ".reg .b64 x, b, v, q, r;\n\t"
        "mov.b64 x, {%2, %3};\n\t"
        "mov.b64 b, {%4, %4};\n\t"
        "mov.b64 v, {%5, %5};\n\t"
        "mul.rn.f32x2 q, x, v;\n\t"
        "fma.rn.f32x2 r, q, b, x;\n\t"
        "fma.rn.f32x2 q, r, v, q;\n\t"
        "mov.b64 {%0, %1}, q;\n\t"
        "}" : "=f"(y[i]), "=f"(y[i + 1]) : "f"(x[i]), "f"(x[i + 1]), "f"(-s.b), "f"(s.inv));
  return fp4_pack8(y);
}
// A sum of products of two rows' codes and block scales (2^-20 .. 2^48, or 0) times the rows' units, the smaller one first: it
// overflows where the result does, and what a small unit makes too small for all digits is 2^-40 of the products' magnitude.
__device__ __forceinline__ float fp4_times_units(float sum, float ua, float ub) {
  float less, more;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(less) : "f"(ua), "f"(ub));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(more) : "f"(ua), "f"(ub));
  return sum * less * more;
}
// Eight codes as numbers, times `scale`.
__device__ __forceinline__ void fp4_values8(unsigned w, float scale, float* x) {
  unsigned h[4];
  asm("{\n\t"
      ".reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t"
      "}" : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; cvt.f32.f16 %0, l; cvt.f32.f16 %1, h; }" : "=f"(lo), "=f"(hi) : "r"(h[i]));
    x[2 * i] = lo * scale;
    x[2 * i + 1] = hi * scale;
  }
}

// 16 values of a row from `at` on, zeros behind K; kept as they came (bfloat16 two a word).
template <typename T> struct Block16 {
  static constexpr int WORDS = 16 * (int)sizeof(T) / 4;
  unsigned w[WORDS];
  template <bool WIDE> __device__ __forceinline__ void load(const T* row, int at, int K) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0;
    if (at >= K) return;
    if (WIDE) {      // rows on 32 bytes, K a multiple of 16
#pragma unroll
      for (int i = 0; i < WORDS / 8; ++i)
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w[8 * i]), "=r"(w[8 * i + 1]), "=r"(w[8 * i + 2]), "=r"(w[8 * i + 3]), "=r"(w[8 * i + 4]),
                       "=r"(w[8 * i + 5]), "=r"(w[8 * i + 6]), "=r"(w[8 * i + 7])
                     : "l"(reinterpret_cast<const char*>(row + at) + 32 * i));
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (at + e < K) {
          if (sizeof(T) == 4) w[e % WORDS] = __float_as_uint(Elem<T>::load(row + at + e));
          else w[e >> 1] |= (unsigned)*reinterpret_cast<const unsigned short*>(row + at + e) << (16 * (e & 1));
        }
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if (sizeof(T) == 4) return __uint_as_float(w[e % WORDS]);
    return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
  }
  __device__ __forceinline__ unsigned top() const {
    unsigned t = 0;
    if (sizeof(T) == 2) {      // two at a time: as 16-bit integers magnitudes order like the numbers
#pragma unroll
      for (int i = 0; i < WORDS; ++i) asm("max.u16x2 %0, %0, %1;" : "+r"(t) : "r"(w[i] & 0x7fff7fffu));
      t = max(t << 16, t & 0xffff0000u);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) t = max(t, fp4_magnitude(get(e)));
    }
    return t;
  }
};
// 16 values, on 32 bytes
template <typename T> __device__ __forceinline__ void store16(T* dst, const float (&x)[16]) {
  constexpr int WORDS = 16 * (int)sizeof(T) / 4;
  unsigned y[16];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (sizeof(T) == 4) {
      y[2 * e] = __float_as_uint(x[2 * e]);
      y[2 * e + 1] = __float_as_uint(x[2 * e + 1]);
    } else {
      const __nv_bfloat162 p = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
      y[e] = *reinterpret_cast<const unsigned*>(&p);
    }
  }
#pragma unroll
  for (int w = 0; w < WORDS; w += 8)
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(reinterpret_cast<unsigned*>(dst) + w), "r"(y[w]),
                 "r"(y[w + 1]), "r"(y[w + 2]), "r"(y[w + 3]), "r"(y[w + 4]), "r"(y[w + 5]), "r"(y[w + 6]), "r"(y[w + 7])
                 : "memory");
}

// ---- block scales of a matrix's rows as the tensor cores' block-scaled products take them: tiles of 128 rows x 64 values, 512
// bytes each, in which row r's scales of its four blocks lie at (r % 32) * 16 + (r / 32) * 4.  Tiles of 128 rows follow one
// another; within them those along k, whose number is a multiple of four (256 values, one stage of a product).
__host__ __device__ __forceinline__ int fp4_k_tiles(int k) { return (k + 255) / 256 * 4; }
__device__ __forceinline__ long long fp4_scale_at(long long row, int block, int k_tiles) {
  return ((row >> 7) * k_tiles + (block >> 2)) * 512 + (row & 31) * 16 + (row >> 5 & 3) * 4 + (block & 3);
}
