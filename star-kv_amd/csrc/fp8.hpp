// Device helpers of the e4m3 kernels: block scales and conversions.
#pragma once
#include "common.hpp"

namespace starkv {

// scale types: one byte 2^(b - 127) (255: NaN), or fp32
struct ScaleE8 { typedef uint8_t T; static constexpr bool pow2 = true; };
struct ScaleF32 { typedef float T; static constexpr bool pow2 = false; };

__device__ inline float scale_f32(uint8_t b) {
  // 2^-127 is subnormal; 255 << 23 would be infinity
  const uint32_t u = b == 255 ? 0x7fc00000u : b == 0 ? 0x00400000u : (uint32_t)b << 23;
  return __uint_as_float(u);
}
__device__ inline float scale_f32(float s) { return s; }

// The scale of a block from the bits of its largest |x| (as fp32), and the
// factor that its values take before they are rounded to e4m3.  A maximum
// that is not finite makes both NaN.
template <typename S> __device__ inline typename S::T block_scale(uint32_t amax_bits, float& inv);
template <> __device__ inline uint8_t block_scale<ScaleE8>(uint32_t amax_bits, float& inv) {
  // e = least integer with a <= 448 2^e = 1.75 2^(e + 8); subnormal a clamp
  int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = max(e, -126);
  if (amax_bits == 0) e = 0;
  const bool bad = amax_bits >= 0x7f800000u;
  inv = bad ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)(127 - e) << 23);
  return bad ? (uint8_t)255 : (uint8_t)(e + 127);
}
template <> __device__ inline float block_scale<ScaleF32>(uint32_t amax_bits, float& inv) {
  if (amax_bits >= 0x7f800000u) return inv = __uint_as_float(0x7fc00000u);
  const float a = fmaxf(__uint_as_float(amax_bits), FP8_AMAX_FLOOR);
  inv = FP8_MAX / a;                               // both divisions correctly rounded
  return amax_bits == 0 ? 1.0f : a / FP8_MAX;
}

// four fp32 values of at most 448 (1 + 2^-23) in magnitude, or NaN, to e4m3 (nearest even)
__device__ inline uint32_t pack_e4m3(float a, float b, float c, float d) {
  int v = 0;
  v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, v, false);
  v = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
  return (uint32_t)v;
}

// the two 16-bit values of a dword, in fp32
template <typename T> __device__ inline void unpack2(uint32_t w, float& a, float& b);
template <> __device__ inline void unpack2<_Float16>(uint32_t w, float& a, float& b) {
  const kh2 h = __builtin_bit_cast(kh2, w);
  a = (float)h[0];
  b = (float)h[1];
}
template <> __device__ inline void unpack2<__bf16>(uint32_t w, float& a, float& b) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}

// Largest |x| of the two 16-bit values of each dword, kept packed: their
// magnitudes order as unsigned integers (a NaN above infinity).
__device__ inline uint32_t max2_u16(uint32_t a, uint32_t b) {
  typedef uint16_t u2 __attribute__((ext_vector_type(2)));
  const u2 x = __builtin_bit_cast(u2, a), y = __builtin_bit_cast(u2, b);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(x, y));
}
// bits of the fp32 value of a 16-bit magnitude (NaN and infinity stay above 0x7f800000)
template <typename T> __device__ inline uint32_t mag_bits(uint32_t h);
template <> __device__ inline uint32_t mag_bits<_Float16>(uint32_t h) {
  const uint32_t f = __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)h));
  return h > 0x7c00u ? 0x7fc00000u : f;
}
template <> __device__ inline uint32_t mag_bits<__bf16>(uint32_t h) { return h << 16; }

// zero the bytes of a 16-byte chunk from nv on (nv may be negative or over 16)
__device__ inline uint4 keep_bytes(uint4 v, int nv) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = nv - 4 * i;
    w[i] = n >= 4 ? w[i] : n <= 0 ? 0u : w[i] & ((1u << (8 * n)) - 1u);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 16 consecutive act-dtype values of a row from column c0 on as 8 dwords;
// columns at or past k are zero.  vec: the row is 16-byte aligned (pieces
// wholly past k are not read).
template <typename T>
__device__ inline void load16(const uint8_t* row, int c0, int k, bool vec, uint32_t (&w)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c = c0 + 8 * h, nv = k - c;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (vec) {
      if (nv > 0) v = *(const uint4*)(row + 2 * (int64_t)c);
      if (nv < 8) v = keep_bytes(v, 2 * nv);
    } else if (nv >= 8) {
      __builtin_memcpy(&v, row + 2 * (int64_t)c, 16);      // one load at any alignment (2157 x 15550: 62 us by elements, 21)
    } else {
      uint16_t e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = i < nv ? ((const uint16_t*)row)[c + i] : (uint16_t)0;
      __builtin_memcpy(&v, e, 16);
    }
    w[4 * h] = v.x; w[4 * h + 1] = v.y; w[4 * h + 2] = v.z; w[4 * h + 3] = v.w;
  }
}

// packed |x| maximum of 16 values
__device__ inline uint32_t amax16(const uint32_t (&w)[8]) {
  uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max2_u16(m, w[i] & 0x7fff7fffu);
  return m;
}

// Two 16-bit values of a dword divided by the power of two `scale` and rounded to e4m3, into the low or high half of v
typedef short short2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
template <typename T, bool HI> __device__ inline uint32_t cvt2_pow2(uint32_t v, uint32_t w, float scale);
template <> __device__ inline uint32_t cvt2_pow2<_Float16, false>(uint32_t v, uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(__builtin_bit_cast(short2v, v), __builtin_bit_cast(kh2, w), scale, false));
}
template <> __device__ inline uint32_t cvt2_pow2<_Float16, true>(uint32_t v, uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(__builtin_bit_cast(short2v, v), __builtin_bit_cast(kh2, w), scale, true));
}
template <> __device__ inline uint32_t cvt2_pow2<__bf16, false>(uint32_t v, uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(__builtin_bit_cast(short2v, v), __builtin_bit_cast(bf16x2, w), scale, false));
}
template <> __device__ inline uint32_t cvt2_pow2<__bf16, true>(uint32_t v, uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(__builtin_bit_cast(short2v, v), __builtin_bit_cast(bf16x2, w), scale, true));
}

// 16 values to e4m3 by block_scale()'s result: one instruction for two values where the scale is a power of two,
// else the product with the reciprocal, rounded to fp32, first
template <typename T, typename S> __device__ inline uint4 quant16(const uint32_t (&w)[8], float inv, float scale) {
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (S::pow2) {
      o[i] = cvt2_pow2<T, true>(cvt2_pow2<T, false>(0u, w[2 * i], scale), w[2 * i + 1], scale);
    } else {
      float a, b, c, d;
      unpack2<T>(w[2 * i], a, b);
      unpack2<T>(w[2 * i + 1], c, d);
      o[i] = pack_e4m3(a * inv, b * inv, c * inv, d * inv);
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// sum of squares of 16 values, added in fp32
template <typename T> __device__ inline float sumsq16(const uint32_t (&w)[8], float ss);
template <> __device__ inline float sumsq16<_Float16>(const uint32_t (&w)[8], float ss) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const kh2 h = __builtin_bit_cast(kh2, w[i]);
    ss = __builtin_amdgcn_fdot2(h, h, ss, false);
  }
  return ss;
}
template <> __device__ inline float sumsq16<__bf16>(const uint32_t (&w)[8], float ss) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bf16x2 h = __builtin_bit_cast(bf16x2, w[i]);
    ss = __builtin_amdgcn_fdot2_f32_bf16(h, h, ss, false);
  }
  return ss;
}

// D (16 x 16) = A (16 rows) B^T (16 rows) over 128 e4m3 columns: lane (r = l
// % 16, g = l / 16) gives 32 bytes of row r of each operand (the same columns
// in both, in any order over g), and gets rows 4g .. 4g + 3 of A against row r of B.
__device__ inline intx8 frag8(uint4 lo, uint4 hi) {
  return intx8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}
__device__ inline floatx4 mfma8(intx8 a, intx8 b, floatx4 c, int scale_a, int scale_b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, scale_a, 0, scale_b);
}
constexpr int E8_ONE = 0x7f7f7f7f;                 // scale 2^0

// The 8-bit instruction adds the eight products of each run of 8 columns with
// about 14 bits below the largest of them (measured: 2^16 + 2^2 gives 2^16
// within a run, 2^16 + 2^-7 is exact across runs), an error of 1.5e-5 of the
// result.  Next to the rounding of a 16-bit output (fp16: 2e-4, bf16: 1.7e-3)
// that is nothing; fp32 outputs take 16-bit instructions instead, whose sums
// hold 24 bits: e4m3 values are fp16 values, and their products are exact.
// Values 8q .. 8q + 7 of a lane's 32, in fp16:
__device__ inline half8 half_of(intx8 v, int q) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  half8 h;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[2 * q + w], 1.0f, false);
    const h2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[2 * q + w], 1.0f, true);
    h[4 * w] = a[0]; h[4 * w + 1] = a[1]; h[4 * w + 2] = b[0]; h[4 * w + 3] = b[1];
  }
  return h;
}
__device__ inline floatx4 mfma8_exact(intx8 a, intx8 b) {
  floatx4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(half_of(a, q), half_of(b, q), c, 0, 0, 0);
  return c;
}

// Four consecutive outputs of type O, nv of them inside the row, at any alignment: whole ones go in one access, which
// the hardware takes at any address (8192 x 8191 outputs by elements cost 35 to 65 % of the product more).
template <typename O> __device__ inline void store4(O* p, const float (&v)[4], int nv) {
  const O t[4] = {(O)v[0], (O)v[1], (O)v[2], (O)v[3]};
  if (nv >= 4) {
    __builtin_memcpy(p, t, sizeof(t));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < nv) p[e] = t[e];
  }
}
template <typename O> __device__ inline void load4(const O* p, float (&v)[4], int nv) {
  if (nv >= 4) {
    O t[4];
    __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)t[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < nv ? (float)p[e] : 0.f;
  }
}
// SiLU(g) u = g u / (1 + exp(-g)); for g far below zero exp is infinite and the reciprocal 0.  exp2 and the
// reciprocal are the instructions' (1 unit of fp32 each), a 16th of what a 16-bit rounding leaves.
__device__ inline float silu_mul_f32(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.4426950408889634f)) * u;
}

}  // namespace starkv
