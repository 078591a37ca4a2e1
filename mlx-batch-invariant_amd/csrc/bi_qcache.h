// bi_qcache.h — rows of a cache held in 8 or 4 bits. A row of D values is D codes
// (8 bits: a byte each; 4 bits: two to a byte, the low half first) and one (scale,
// bias) pair of type T for each group of 32, 64 or 128 values; code c stands for
// T(fma(c, scale, bias)), as in the quantized matmul.
#pragma once

#include "bi_common.h"

namespace bi {

template <typename T> struct Pair { float s, b; };        // a group's scale and bias

template <typename T>
__device__ __forceinline__ Pair<T> unpack_pair(const uint32_t* u) {
  Pair<T> g;
  if constexpr (sizeof(T) == 2) {
    g.s = to_f32(__builtin_bit_cast(T, (uint16_t)u[0]));
    g.b = to_f32(__builtin_bit_cast(T, (uint16_t)(u[0] >> 16)));
  } else {
    g.s = __builtin_bit_cast(float, u[0]);
    g.b = __builtin_bit_cast(float, u[1]);
  }
  return g;
}
template <typename T>
__device__ __forceinline__ Pair<T> load_pair(const T* p) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
    return unpack_pair<T>(&u);
  } else {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
    const uint32_t u[2] = {v[0], v[1]};
    return unpack_pair<T>(u);
  }
}

// Eight and sixteen consecutive codes.
template <int BITS> struct Codes8;
template <> struct Codes8<8> { uint32_t w[2]; };
template <> struct Codes8<4> { uint32_t w[1]; };
template <int BITS> struct Codes16 {
  uint32_t w[BITS / 2];
  __device__ __forceinline__ Codes8<BITS> half(int h) const {
    Codes8<BITS> c;
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) c.w[i] = w[h * (BITS / 4) + i];
    return c;
  }
};

template <int BITS>
__device__ __forceinline__ Codes8<BITS> load_codes8(const char* p) {
  Codes8<BITS> c;
  if constexpr (BITS == 8) {
    const u32x2 u = *reinterpret_cast<const u32x2*>(p);
    c.w[0] = u[0];
    c.w[1] = u[1];
  } else {
    c.w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
  return c;
}

template <int BITS>
__device__ __forceinline__ Codes16<BITS> load_codes16(const char* p) {
  Codes16<BITS> c;
  if constexpr (BITS == 8) {
    const u32x4 u = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) c.w[i] = u[i];
  } else {
    const u32x2 u = *reinterpret_cast<const u32x2*>(p);
    c.w[0] = u[0];
    c.w[1] = u[1];
  }
  return c;
}

// The values of 8 codes, as floats that hold T's before the rounding.
template <int BITS>
__device__ __forceinline__ void code_floats(Codes8<BITS> c, float (&x)[8]) {
  if constexpr (BITS == 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)(c.w[e / 4] >> (8 * (e % 4)) & 255u);
  } else {
    uint32_t even = c.w[0] & 0x0f0f0f0fu, odd = c.w[0] >> 4 & 0x0f0f0f0fu;
    // (three instructions for eight codes, which are converted from bytes then; seen
    // through, each code costs one of its own)
    asm("" : "+v"(even), "+v"(odd));
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)((e & 1 ? odd : even) >> (8 * (e / 2)) & 255u);
  }
}

// Codes of 4 bits as fp16 numbers instead, n 2^-24 (denormals; odd ones n 2^-20): an fma
// takes such a number as it is (v_fma_mix_f32, which keeps denormals), so with the
// scale times code_factor() a code needs no conversion, and two are cut out of a word
// at once. The product is exact either way, so the fma rounds the same sum. Decode over
// 4 bits, 64 sequences of up to 8192 keys, in turn: fp16 112 -> 110 us, bf16 113 -> 108,
// four tokens 129 -> 122, heads of 64 63 -> 60. (Bytes, which a conversion takes out of
// the word by itself, gained nothing.)
__device__ __forceinline__ void code_halves(Codes8<4> c, _Float16 (&h)[8]) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f16x2 x = __builtin_bit_cast(f16x2, c.w[0] >> (i / 2 * 8) & (i % 2 ? 0x00f000f0u : 0x000f000fu));
    h[i] = x[0];
    h[i + 4] = x[1];
  }
}
template <int BITS>
__device__ __forceinline__ float code_factor(int e) { return BITS == 8 ? 1.0f : e & 1 ? 0x1p20f : 0x1p24f; }

// x[e] = fma(code, scale, bias), rounded to T.
template <typename T>
__device__ __forceinline__ typename Frag<T>::type round_frag8(float (&x)[8]) {
  typedef float f32x2v __attribute__((ext_vector_type(2)));
  typedef T tx2 __attribute__((ext_vector_type(2)));
  typename Frag<T>::type f;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int e = 0; e < 8; ++e) asm("" : "+v"(x[e]));
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const tx2 y = __builtin_convertvector(f32x2v{x[e], x[e + 1]}, tx2);
      f[e] = y[0];
      f[e + 1] = y[1];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f.lo[e] = x[e];
      f.hi[e] = x[4 + e];
    }
  }
  return f;
}

// T(fma(code, scale, bias)) of 8 codes, each with a pair of its own or all of one
// group. The fma's result is kept in a register of its own: folded into the conversion
// (v_fma_mixlo_f16) it would round once where the quantized matmul rounds twice.
template <typename T, int BITS>
__device__ __forceinline__ typename Frag<T>::type dequant_frag8(Codes8<BITS> c, const float (&s)[8], const float (&b)[8]) {
  float x[8];
  code_floats<BITS>(c, x);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __builtin_fmaf(x[e], s[e], b[e]);
  return round_frag8<T>(x);
}
// The same from s[e] = scale code_factor(e), where that is finite.
template <typename T, int BITS>
__device__ __forceinline__ typename Frag<T>::type dequant_scaled8(Codes8<BITS> c, const float (&s)[8], const float (&b)[8]) {
  if constexpr (BITS == 8) {
    return dequant_frag8<T, 8>(c, s, b);
  } else {
    _Float16 h[8];
    code_halves(c, h);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __builtin_fmaf((float)h[e], s[e], b[e]);
    return round_frag8<T>(x);
  }
}
template <typename T, int BITS>
__device__ __forceinline__ typename Frag<T>::type dequant_frag(Codes8<BITS> c, Pair<T> g) {
  const float s[8] = {g.s, g.s, g.s, g.s, g.s, g.s, g.s, g.s}, b[8] = {g.b, g.b, g.b, g.b, g.b, g.b, g.b, g.b};
  return dequant_frag8<T, BITS>(c, s, b);
}

}  // namespace bi
