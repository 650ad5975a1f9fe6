// Pieces of 8 elements of token and cache rows, to and from fp32.
#pragma once

#include "q4.cuh"

namespace saga {

// 8 consecutive elements of a row as floats.
__device__ __forceinline__ void load8(const void* base, int dt, int64_t off, bool vec, float (&f)[8]) {
  if (vec && dt != SAGA_DTYPE_F32) {
    const u32x4 v = ld16(static_cast<const uint16_t*>(base) + off);
    if (dt == SAGA_DTYPE_BF16) unpack16<SAGA_DTYPE_BF16>(v, f);
    else unpack16<SAGA_DTYPE_F16>(v, f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = load_as_f32(base, dt, off + e);
  }
}

__device__ __forceinline__ void store8(void* base, int dt, int64_t off, bool vec, const float (&f)[8]) {
  if (vec && dt != SAGA_DTYPE_F32) {
    u32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (dt == SAGA_DTYPE_BF16) v[e] = q4_bf16_pair(f[2 * e], f[2 * e + 1]);
      else v[e] = f32_to_f16_bits(f[2 * e]) | (static_cast<uint32_t>(f32_to_f16_bits(f[2 * e + 1])) << 16);
    }
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(base) + off) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) store_from_f32(base, dt, off + e, f[e]);
  }
}

}  // namespace saga
