// e4m3 numbers (OCP form: 4 exponent bits, 3 of mantissa, largest 448, no infinities) with
// a scale per block of a cache's positions (form: include/saga_amd.h).
#pragma once

#include "common.cuh"

namespace saga {

constexpr float kFp8Max = 448.f;

// Two of a word's four e4m3 numbers as a pair of 16-bit numbers (exact in bf16 and f16).
template <int DT, bool HI>
__device__ __forceinline__ uint32_t fp8_pair(uint32_t w) {
  if constexpr (DT == SAGA_DTYPE_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HI));
}

// 8 e4m3 numbers as an MFMA operand.
template <int DT>
__device__ __forceinline__ u32x4 fp8_frag(uint32_t w0, uint32_t w1) {
  return u32x4{fp8_pair<DT, false>(w0), fp8_pair<DT, true>(w0), fp8_pair<DT, false>(w1), fp8_pair<DT, true>(w1)};
}

__device__ __forceinline__ void fp8_open(uint32_t w, float (&f)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  f[0] = lo[0], f[1] = lo[1], f[2] = hi[0], f[3] = hi[1];
}

// c s of finite c and s: e4m3 may round the largest magnitudes of bf16 and f32 up to 2^128.
__device__ __forceinline__ float fp8_value(float c, float s) {
  constexpr float kBf16Max = 0x1.fep127f;
  const float v = c * s;
  return fabsf(v) == __builtin_inff() && s < __builtin_inff() ? copysignf(kBf16Max, v) : v;
}

// Four floats rounded to e4m3 (to the nearest, ties to even; at most 448 in magnitude, or NaN).
__device__ __forceinline__ uint32_t fp8_round(float a, float b, float c, float d) {
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}

// 16 e4m3 numbers times a power of two, rounded again.
__device__ __forceinline__ u32x4 fp8_rescaled(u32x4 v, float by) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[4];
    fp8_open(v[i], f);
    v[i] = fp8_round(f[0] * by, f[1] * by, f[2] * by, f[3] * by);
  }
  return v;
}

// The scale that a largest magnitude asks for: 2^(floor(log2 top) - 5), so that top / scale lies in
// [32, 64).  Rounding in a floating form does not gain from a tighter scale: three powers of two
// are left for later tokens of a block (a rise of the scale rounds what the block holds again),
// and numbers turn subnormal only below 2^-11 of the largest.
__device__ __forceinline__ float fp8_scale(float top) {
  if (!(top > 0.f)) return 0.f;
  int e;
  frexpf(top, &e);
  return __uint_as_float(static_cast<uint32_t>(max(e - 6, -100) + 127) << 23);
}

// 1 / s of a power of two s, 0 for a block of zeros.
__device__ __forceinline__ float fp8_inverse(float s) { return s > 0.f ? 1.f / s : 0.f; }

// |x| where it counts for a scale: infinities and NaN are held as NaN whatever the scale.
__device__ __forceinline__ float fp8_size(float x) { return fabsf(x) < __builtin_inff() ? fabsf(x) : 0.f; }

// A double rounded to a float whose last bit tells that more follows (round to odd): rounding
// that once more to few bits gives what rounding the double would.
__device__ __forceinline__ float odd_float(double v) {
  const float f = static_cast<float>(v);
  const double d = static_cast<double>(f);
  uint32_t u = __float_as_uint(f);
  u -= fabs(d) > fabs(v) ? 1u : 0u;  // towards zero
  u |= d != v ? 1u : 0u;
  return __uint_as_float(u);
}

}  // namespace saga
