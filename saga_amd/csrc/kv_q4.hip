// The 4-bit key / value cache around its attention: rotary embedding with the
// append of new tokens, and rows read back as values.  Formats: saga_amd.h.
#include "kernels.h"
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
      const uint32_t lo = dt == SAGA_DTYPE_BF16 ? f32_to_bf16_bits(f[2 * e]) : f32_to_f16_bits(f[2 * e]);
      const uint32_t hi = dt == SAGA_DTYPE_BF16 ? f32_to_bf16_bits(f[2 * e + 1]) : f32_to_f16_bits(f[2 * e + 1]);
      v[e] = lo | (hi << 16);
    }
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(base) + off) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) store_from_f32(base, dt, off + e, f[e]);
  }
}

// The largest f16 that is at most x, and the smallest that is at least x (|x| at most 65504).
__device__ __forceinline__ uint16_t f16_down(float x) {
  const uint16_t h = f32_to_f16_bits(x);
  if (!(f16_bits_to_f32(h) > x)) return h;
  return (h & 0x7fffu) == 0 ? 0x8001u : (h & 0x8000u) ? h + 1 : h - 1;
}
__device__ __forceinline__ uint16_t f16_up(float x) { return f16_down(-x) ^ 0x8000u; }

// One thread per 8 consecutive dims of a (token, head); the d / 8 threads of a
// head are neighbours, so a group's extremes and a value row's transposition are
// lane exchanges.  A query or key thread reads its dims and their rotary partners.
__global__ void __launch_bounds__(256) rope_kv_append_q4_kernel(RopeQ4Params p) {
  const int per = p.kv.d / 8, heads = p.n_q + p.kv.n_k + p.kv.n_v;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = min(item / per, static_cast<int64_t>(p.N) * heads - 1);  // threads past the end repeat the last head
  const bool live = item < static_cast<int64_t>(p.N) * heads * per;
  const int t = static_cast<int>(item % per);
  const int n = static_cast<int>(row / heads), hh = static_cast<int>(row - static_cast<int64_t>(n) * heads);
  const int d = p.kv.d, half = d / 2;
  const int pos = p.pos[n], b = p.batch ? p.batch[n] : n;
  const bool ok = pos >= 0 && pos < p.kv.Lmax && b >= 0 && b < p.kv.B;
  const int64_t src = static_cast<int64_t>(n) * p.qkv_ld + static_cast<int64_t>(hh) * d;
  float x[8];
  load8(p.qkv, p.dt, src + 8 * t, p.vec, x);
  if (hh < p.n_q + p.kv.n_k) {
    const bool second = 8 * t >= half;
    const int i = 8 * t - (second ? half : 0);
    float o[8];
    load8(p.qkv, p.dt, src + (second ? i : i + half), p.vec, o);
    const f32x4* rot = reinterpret_cast<const f32x4*>(p.table + static_cast<int64_t>(n) * d) + i / 2;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f32x4 r = rot[e];  // cos, sin of two pairs
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float cs = r[2 * k], sn = r[2 * k + 1], a = x[2 * e + k], w = o[2 * e + k];
        x[2 * e + k] = second ? a * cs + w * sn : a * cs - w * sn;
      }
    }
    if (hh < p.n_q) {
      if (!ok) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __builtin_nanf("");
      }
      if (live) store8(p.q_out, p.dt, static_cast<int64_t>(n) * p.q_sn + static_cast<int64_t>(hh) * p.q_sh + 8 * t, p.vec, x);
    }
  }
  // every thread takes part in the exchanges below: a wave may hold query and cache heads
  float lo = x[0], hi = x[0];
  int bad = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo = fminf(lo, x[e]);
    hi = fmaxf(hi, x[e]);
    bad |= !(fabsf(x[e]) <= 65504.f);
  }
  for (int m = 1; m < p.kv.group / 8; m <<= 1) {
    lo = fminf(lo, __shfl_xor(lo, m));
    hi = fmaxf(hi, __shfl_xor(hi, m));
    bad |= __shfl_xor(bad, m);
  }
  uint16_t zb = 0x7e00, sb = 0x7e00;
  uint32_t w = 0;
  if (!bad) {
    zb = f16_down(lo);
    const float z = f16_bits_to_f32(zb);
    sb = f16_up((hi - z) / 15.f);
    const float s = f16_bits_to_f32(sb), by = s > 0.f ? s : 1.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= static_cast<uint32_t>(fminf(fmaxf(rintf((x[e] - z) / by), 0.f), 15.f)) << (4 * e);
  }
  const bool is_v = hh >= p.n_q + p.kv.n_k;
  // values: nibble e of unit c is dim 16 e + c, held by thread 2 e + c / 8 as its nibble c % 8
  uint32_t vw = 0;
  const int lane = threadIdx.x & 63, head0 = lane - t;
  if (per == 16) {
#pragma unroll
    for (int e = 0; e < 8; ++e) vw |= ((__shfl(w, head0 + 2 * e + (t >> 3)) >> (4 * (t & 7))) & 15u) << (4 * e);
  } else {  // two units of 4 nibbles per thread
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t two = __shfl(w, head0 + 2 * e + (t >> 2)) >> (8 * (t & 3));
      vw |= ((two & 15u) << (4 * e)) | (((two >> 4) & 15u) << (16 + 4 * e));
    }
  }
  if (!live || !ok || hh < p.n_q) return;
  const int h = hh - p.n_q - (is_v ? p.kv.n_k : 0);
  char* codes = const_cast<char*>(is_v ? p.kv.vc + b * p.kv.vc_sb + h * p.kv.vc_sh + pos * p.kv.vc_sl
                                       : p.kv.kc + b * p.kv.kc_sb + h * p.kv.kc_sh + pos * p.kv.kc_sl);
  char* scales = const_cast<char*>(is_v ? p.kv.vs + b * p.kv.vs_sb + h * p.kv.vs_sh + pos * p.kv.vs_sl
                                        : p.kv.ks + b * p.kv.ks_sb + h * p.kv.ks_sh + pos * p.kv.ks_sl);
  const int word = is_v ? t : (t & 3) * (d / 32) + (t >> 2);
  *reinterpret_cast<uint32_t*>(codes + 4 * word) = is_v ? vw : w;
  const int tg = p.kv.group / 8;
  if (t % tg == 0) *reinterpret_cast<uint32_t*>(scales + 4 * (t / tg)) = sb | (static_cast<uint32_t>(zb) << 16);
}

hipError_t launch_rope_kv_append_q4(const RopeQ4Params& p, hipStream_t st) {
  const int64_t items = static_cast<int64_t>(p.N) * (p.n_q + p.kv.n_k + p.kv.n_v) * (p.kv.d / 8);
  hipLaunchKernelGGL(rope_kv_append_q4_kernel, dim3(static_cast<unsigned>((items + 255) / 256)), dim3(256), 0, st, p);
  return hipGetLastError();
}

// One thread per 8 consecutive dims of a (token, head): one code word and one
// pair (s, z); a value thread picks its dims out of 8 units.
__global__ void __launch_bounds__(256) kv_q4_read_kernel(KvQ4ReadParams p) {
  const int per = p.kv.d / 8, heads = p.kv.n_k + p.kv.n_v;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (item >= static_cast<int64_t>(p.N) * heads * per) return;
  const int64_t row = item / per;
  const int t = static_cast<int>(item - row * per);
  const int n = static_cast<int>(row / heads), hh = static_cast<int>(row - static_cast<int64_t>(n) * heads);
  const int pos = p.pos[n], b = p.batch ? p.batch[n] : n;
  const bool is_v = hh >= p.kv.n_k;
  const int h = hh - (is_v ? p.kv.n_k : 0);
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __builtin_nanf("");
  if (pos >= 0 && pos < p.kv.Lmax && b >= 0 && b < p.kv.B) {
    const char* codes = is_v ? p.kv.vc + b * p.kv.vc_sb + h * p.kv.vc_sh + pos * p.kv.vc_sl
                             : p.kv.kc + b * p.kv.kc_sb + h * p.kv.kc_sh + pos * p.kv.kc_sl;
    const char* scales = is_v ? p.kv.vs + b * p.kv.vs_sb + h * p.kv.vs_sh + pos * p.kv.vs_sl
                              : p.kv.ks + b * p.kv.ks_sb + h * p.kv.ks_sh + pos * p.kv.ks_sl;
    const uint32_t sz = *reinterpret_cast<const uint32_t*>(scales + 4 * (8 * t / p.kv.group));
    const float s = q4_lo(sz), z = q4_hi(sz);
    if (!is_v) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + 4 * ((t & 3) * (p.kv.d / 32) + (t >> 2)));
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = s * static_cast<float>((w >> (4 * e)) & 15u) + z;
    } else {
      const int sh = 4 * (t >> 1), c0 = 8 * (t & 1);  // dims 16 (t / 2) + c0 + e: nibble t / 2 of units c0 + e
      if (per == 16) {
        const u32x4* q = reinterpret_cast<const u32x4*>(codes + 4 * c0);
        const u32x4 a[2] = {q[0], q[1]};
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = s * static_cast<float>((a[e >> 2][e & 3] >> sh) & 15u) + z;
      } else {
        const u32x4 a = *reinterpret_cast<const u32x4*>(codes + 2 * c0);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = s * static_cast<float>((a[e >> 1] >> (16 * (e & 1) + sh)) & 15u) + z;
      }
    }
  }
  if (is_v) store8(p.v, p.dt, static_cast<int64_t>(n) * p.v_sn + static_cast<int64_t>(h) * p.v_sh + 8 * t, p.vec, x);
  else store8(p.k, p.dt, static_cast<int64_t>(n) * p.k_sn + static_cast<int64_t>(h) * p.k_sh + 8 * t, p.vec, x);
}

hipError_t launch_kv_q4_read(const KvQ4ReadParams& p, hipStream_t st) {
  const int64_t items = static_cast<int64_t>(p.N) * (p.kv.n_k + p.kv.n_v) * (p.kv.d / 8);
  hipLaunchKernelGGL(kv_q4_read_kernel, dim3(static_cast<unsigned>((items + 255) / 256)), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace saga
