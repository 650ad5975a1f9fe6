// 4-bit codes on the way to matrix products (layouts: include/saga_amd.h).
//
// A code c enters an MFMA as a bf16 number b + c, where one or two instructions
// make that for two codes of a word: nibbles 0 and 4 are merged in place with the
// bits of b = 128 (a bf16 mantissa's unit there is 1), the others are shifted to
// bits 3..6 of their half, where the unit at b = 16 is 1/8.  Products with bf16
// numbers are then exact, and what b adds is taken out of the fp32 sums.
#pragma once

#include "common.cuh"

namespace saga {

constexpr uint32_t kBf16Ones = 0x3f803f80u;

// The masks and b's of two codes, in registers: as literals each code pair took an and
// and an or (a three-operand instruction holds no literal).
struct Q4Const {
  uint32_t mask0, mask, base0, base;
  __device__ __forceinline__ Q4Const() : mask0(0x000f000fu), mask(0x00780078u), base0(0x43004300u), base(0x41804180u) {
    asm("" : "+s"(mask0), "+s"(mask), "+v"(base0), "+v"(base));
  }
};

// b + nibble P of each half of w: b = 128 for P = 0, else 16.
template <int P>
__device__ __forceinline__ uint32_t q4_pair(uint32_t w, const Q4Const& c) {
  if constexpr (P == 0) return (w & c.mask0) | c.base0;
  else return ((w >> (4 * P - 3)) & c.mask) | c.base;
}

// The 8 codes of a word as an MFMA operand: slots 2 p and 2 p + 1 are nibbles p and p + 4.
__device__ __forceinline__ u32x4 q4_frag(uint32_t w, const Q4Const& c) {
  return u32x4{q4_pair<0>(w, c), q4_pair<1>(w, c), q4_pair<2>(w, c), q4_pair<3>(w, c)};
}

// The same with b = 16 in every slot.
template <int P>
__device__ __forceinline__ uint32_t q4_pair16(uint32_t w, const Q4Const& c) {
  if constexpr (P == 0) return ((w << 3) & c.mask) | c.base;
  else return q4_pair<P>(w, c);
}
__device__ __forceinline__ u32x4 q4_frag16(uint32_t w, const Q4Const& c) {
  return u32x4{q4_pair16<0>(w, c), q4_pair16<1>(w, c), q4_pair16<2>(w, c), q4_pair16<3>(w, c)};
}

// -b of each slot of q4_frag.
__device__ __forceinline__ u32x4 q4_minus_base() { return u32x4{0xc300c300u, 0xc180c180u, 0xc180c180u, 0xc180c180u}; }

__device__ __forceinline__ float q4_lo(uint32_t sz) { return f16_bits_to_f32(sz & 0xffffu); }  // scale
__device__ __forceinline__ float q4_hi(uint32_t sz) { return f16_bits_to_f32(sz >> 16); }      // offset

// What a result of type dt holds of v.  A group's scale is rounded up (4 bits), or the value itself (e4m3), so that
// the largest value may read as up to 65536 although what was stored fits f16: finite results end at f16's range.
__device__ __forceinline__ float q4_in_range(float v, int dt) {
  return dt == SAGA_DTYPE_F16 && fabsf(v) > 65504.f && fabsf(v) < __builtin_inff() ? copysignf(65504.f, v) : v;
}

// Two floats rounded to a pair of bf16 numbers.
__device__ __forceinline__ uint32_t q4_bf16_pair(float a, float b) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2_t));
}

}  // namespace saga
