// The 4-bit key / value cache around its attention: rotary embedding with the
// append of new tokens, and rows read back as values.  Formats: saga_amd.h.
#include "kernels.h"
#include "rows.cuh"

namespace saga {

// The largest f16 that is at most x, and the smallest that is at least x (|x| at most 65504).
__device__ __forceinline__ uint16_t f16_down(float x) {
  const uint16_t h = f32_to_f16_bits(x);
  if (!(f16_bits_to_f32(h) > x)) return h;
  return (h & 0x7fffu) == 0 ? 0x8001u : (h & 0x8000u) ? h + 1 : h - 1;
}
__device__ __forceinline__ uint16_t f16_up(float x) { return f16_down(-x) ^ 0x8000u; }

// NW x 8 floats of one group as codes (word i, nibble e: value 8 i + e) and its (s, z); the
// TG threads of a group are neighbours.
template <int TG, int NW>
__device__ __forceinline__ void quantise(const float (&x)[NW][8], uint32_t (&w)[NW], uint32_t& sz) {
  float lo = x[0][0], hi = x[0][0];
  int bad = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo = fminf(lo, x[i][e]);
      hi = fmaxf(hi, x[i][e]);
      bad |= !(fabsf(x[i][e]) <= 65504.f);
    }
#pragma unroll
  for (int m = 1; m < TG; m <<= 1) {
    lo = fminf(lo, __shfl_xor(lo, m));
    hi = fmaxf(hi, __shfl_xor(hi, m));
    bad |= __shfl_xor(bad, m);
  }
#pragma unroll
  for (int i = 0; i < NW; ++i) w[i] = 0u;
  sz = 0x7e007e00u;
  if (bad) return;
  const uint16_t zb = f16_down(lo);
  const float z = f16_bits_to_f32(zb);
  const uint16_t sb = f16_up((hi - z) / 15.f);
  const float s = f16_bits_to_f32(sb), by = s > 0.f ? s : 1.f, r = 1.f / by;
  sz = sb | (static_cast<uint32_t>(zb) << 16);
#pragma unroll
  for (int i = 0; i < NW; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // (x - z) / by, correctly rounded: with the correctly rounded reciprocal r, one
      // correction of the product by its exact remainder is (Markstein)
      const float a = x[i][e] - z, q0 = a * r;
      const float q = __builtin_fmaf(__builtin_fmaf(-q0, by, a), r, q0);
      w[i] |= static_cast<uint32_t>(fminf(fmaxf(rintf(q), 0.f), 15.f)) << (4 * e);
    }
}

// T = d / 16 threads per head take dims 8 t .. and d / 2 + 8 t .. , the rotary partners; a
// wave takes 64 / T heads of one token at a time, with the token's rotations in registers
// for all of them; few tokens spread their heads over blocks (grid y).  A group's extremes
// and a value row's transposition are lane exchanges.  4001 tokens of 15 heads, d 128
// (31 MB): 11.0 us, bound by the quantisation's VALU work beside the projection's bytes: of a
// wave's second pass here (12 / 1 / 2 heads) 24 lanes hold keys or values and 40 queries or
// repeats (a thread per 8 dims that read its rotations per head and divided per value: 16.8;
// heads over blocks here too: 12.4); 8 tokens 4.7 us, a launch and two round trips.
template <int D, int G>
__global__ void __launch_bounds__(256) rope_kv_append_q4_kernel(RopeQ4Params p) {
  constexpr int T = D / 16, HW = 64 / T;
  const int lane = threadIdx.x & 63, t = lane % T, heads = p.n_q + p.kv.n_k + p.kv.n_v;
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= p.N) return;
  const int pos = p.pos[n], b = p.batch ? p.batch[n] : n;
  const bool ok = pos >= 0 && pos < p.kv.Lmax && b >= 0 && b < p.kv.B;
  f32x4 rot[4];  // (cos, sin) of pairs 8 t .. 8 t + 7
#pragma unroll
  for (int e = 0; e < 4; ++e) rot[e] = reinterpret_cast<const f32x4*>(p.table + static_cast<int64_t>(n) * D)[4 * t + e];
  for (int h0 = blockIdx.y * HW; h0 < heads; h0 += gridDim.y * HW) {
    const int hh = min(h0 + lane / T, heads - 1);  // lanes past the last head repeat it
    const bool live = h0 + lane / T < heads;
    const int64_t src = static_cast<int64_t>(n) * p.qkv_ld + static_cast<int64_t>(hh) * D + 8 * t;
    float x[2][8];  // dims 8 t .. and D / 2 + 8 t ..
    load8(p.qkv, p.dt, src, p.vec, x[0]);
    load8(p.qkv, p.dt, src + D / 2, p.vec, x[1]);
    if (hh < p.n_q + p.kv.n_k) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float cs = rot[e / 2][2 * (e & 1)], sn = rot[e / 2][2 * (e & 1) + 1], x1 = x[0][e], x2 = x[1][e];
        x[0][e] = x1 * cs - x2 * sn;
        x[1][e] = x2 * cs + x1 * sn;
      }
    }
    if (hh < p.n_q && live) {
      if (!ok) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[0][e] = x[1][e] = __builtin_nanf("");
      }
      const int64_t dst = static_cast<int64_t>(n) * p.q_sn + static_cast<int64_t>(hh) * p.q_sh + 8 * t;
      store8(p.q_out, p.dt, dst, p.vec, x[0]);
      store8(p.q_out, p.dt, dst + D / 2, p.vec, x[1]);
    }
    if (h0 + HW <= p.n_q) continue;  // the whole wave holds queries
    uint32_t w[2], sz[2];
    if constexpr (G <= D / 2) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float (&xi)[1][8] = reinterpret_cast<const float (&)[1][8]>(x[i]);
        quantise<G / 8>(xi, reinterpret_cast<uint32_t (&)[1]>(w[i]), sz[i]);
      }
    } else {  // one group over both halves
      quantise<T>(x, w, sz[0]);
      sz[1] = sz[0];
    }
    const bool is_v = hh >= p.n_q + p.kv.n_k;
    if (__any(is_v)) {
      // values: nibble e of unit c (of 16) is dim 16 e + c, value (c & 7) of word 2 e + c / 8,
      // which thread (2 e + c / 8) mod T holds as its word (2 e + c / 8) / T
      uint32_t v[2] = {0u, 0u};
      const int head0 = lane - t;
      if constexpr (D == 128) {  // units t and t + 8
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            v[i] |= ((__shfl(w[e / 4], head0 + (2 * e + i) % 8) >> (4 * t)) & 15u) << (4 * e);
      } else {  // two units of 4 nibbles a word: 2 t, 2 t + 1 and 2 t + 8, 2 t + 9
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t two = __shfl(w[e / 2], head0 + (2 * e + i) % 4) >> (8 * t);
            v[i] |= ((two & 15u) << (4 * e)) | (((two >> 4) & 15u) << (16 + 4 * e));
          }
      }
      if (is_v) w[0] = v[0], w[1] = v[1];
    }
    if (!live || !ok || hh < p.n_q) continue;
    const int h = hh - p.n_q - (is_v ? p.kv.n_k : 0);
    char* codes = const_cast<char*>(is_v ? p.kv.vc + b * p.kv.vc_sb + h * p.kv.vc_sh + pos * p.kv.vc_sl
                                         : p.kv.kc + b * p.kv.kc_sb + h * p.kv.kc_sh + pos * p.kv.kc_sl);
    char* scales = const_cast<char*>(is_v ? p.kv.vs + b * p.kv.vs_sb + h * p.kv.vs_sh + pos * p.kv.vs_sl
                                          : p.kv.ks + b * p.kv.ks_sb + h * p.kv.ks_sh + pos * p.kv.ks_sl);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int u = t + i * T;  // dims 8 u ..
      const int word = is_v ? u : (u & 3) * (D / 32) + (u >> 2);
      *reinterpret_cast<uint32_t*>(codes + 4 * word) = w[i];
      if (u % (G / 8) == 0) *reinterpret_cast<uint32_t*>(scales + 4 * (u / (G / 8))) = sz[i];
    }
  }
}

template <int D, int G>
static void launch_rope_kv_append_q4_typed(const RopeQ4Params& p, hipStream_t st) {
  const int passes = (p.n_q + p.kv.n_k + p.kv.n_v + 64 / (D / 16) - 1) / (64 / (D / 16));
  const dim3 grid(static_cast<unsigned>((p.N + 3) / 4), p.N < 1024 ? passes : 1);
  hipLaunchKernelGGL((rope_kv_append_q4_kernel<D, G>), grid, dim3(256), 0, st, p);
}

hipError_t launch_rope_kv_append_q4(const RopeQ4Params& p, hipStream_t st) {
  if (p.kv.d == 128) {
    if (p.kv.group == 32) launch_rope_kv_append_q4_typed<128, 32>(p, st);
    else launch_rope_kv_append_q4_typed<128, 64>(p, st);
  } else {
    if (p.kv.group == 32) launch_rope_kv_append_q4_typed<64, 32>(p, st);
    else launch_rope_kv_append_q4_typed<64, 64>(p, st);
  }
  return hipGetLastError();
}

// One thread per 8 consecutive dims of a (token, head): one code word and one
// pair (s, z); a value thread picks its dims out of 8 units.  4001 tokens of 3 heads, d 128
// (4 MB): 4.9 us, two dependent round trips (the index, then the row).
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
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = q4_in_range(x[e], p.dt);
  if (is_v) store8(p.v, p.dt, static_cast<int64_t>(n) * p.v_sn + static_cast<int64_t>(h) * p.v_sh + 8 * t, p.vec, x);
  else store8(p.k, p.dt, static_cast<int64_t>(n) * p.k_sn + static_cast<int64_t>(h) * p.k_sh + 8 * t, p.vec, x);
}

hipError_t launch_kv_q4_read(const KvQ4ReadParams& p, hipStream_t st) {
  const int64_t items = static_cast<int64_t>(p.N) * (p.kv.n_k + p.kv.n_v) * (p.kv.d / 8);
  hipLaunchKernelGGL(kv_q4_read_kernel, dim3(static_cast<unsigned>((items + 255) / 256)), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace saga
