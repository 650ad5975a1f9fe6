// 4-bit codes on the way to matrix products (layouts: include/saga_amd.h).
//
// A code c enters an MFMA as the bf16 number 16 + c, which two instructions make
// for two codes: shifted to bits 3..6 of each half (a bf16 mantissa's unit at 16
// is 1/8, bit 0) and merged with 16's bits.  Products with bf16 numbers are then
// exact, and what the 16 adds is taken out of the fp32 sums.
#pragma once

#include "common.cuh"

namespace saga {

constexpr uint32_t kQ4Mask = 0x00780078u, kQ4Base = 0x41804180u;  // two of 4 bits at bit 3; two of 16.0
constexpr uint32_t kBf16Ones = 0x3f803f80u;

// 16 + nibble P of each half of w.
template <int P>
__device__ __forceinline__ uint32_t q4_pair(uint32_t w) {
  if constexpr (P == 0) return ((w << 3) & kQ4Mask) | kQ4Base;
  else return ((w >> (4 * P - 3)) & kQ4Mask) | kQ4Base;
}

// The 8 codes of a word as an MFMA operand: slots 2 p and 2 p + 1 are nibbles p and p + 4.
__device__ __forceinline__ u32x4 q4_frag(uint32_t w) {
  return u32x4{q4_pair<0>(w), q4_pair<1>(w), q4_pair<2>(w), q4_pair<3>(w)};
}

__device__ __forceinline__ float q4_lo(uint32_t sz) { return f16_bits_to_f32(sz & 0xffffu); }  // scale
__device__ __forceinline__ float q4_hi(uint32_t sz) { return f16_bits_to_f32(sz >> 16); }      // offset

}  // namespace saga
