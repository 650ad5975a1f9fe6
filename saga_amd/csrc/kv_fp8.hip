// New tokens into a cache: norms of queries and keys per head, rotary embedding and append
// in one pass, into a cache of the tokens' own type or one of 8 bits; rows of an
// 8-bit cache read back.  Formats: saga_amd.h.
//
// A token's head x [d]: y = x / sqrt(mean x^2 + eps) * w, then the pairs (i, i + d / 2) turned by
// the token's rotations; values are stored as they come.  T = d / 16 threads take a head, dims
// 8 t .. and d / 2 + 8 t .., the rotary partners: the mean is a sum over T lanes, everything
// else stays in a thread.  Bound by the projection read once and written once.
#include "fp8.cuh"
#include "kernels.h"
#include "rows.cuh"

namespace saga {

// Sum over the T lanes of a head (T = 4 or 8, neighbours).
template <int T>
__device__ __forceinline__ float head_sum(float v) {
  v += dpp_f<kDppQuadXor1>(v);
  v += dpp_f<kDppQuadXor2>(v);
  if constexpr (T == 8) v += dpp_f<kDppRowHalfMirror>(v);
  return v;
}
template <int T>
__device__ __forceinline__ double head_sum(double v) {
#pragma unroll
  for (int m = 1; m < T; m <<= 1) v += __shfl_xor(v, m);
  return v;
}
template <int T>
__device__ __forceinline__ float head_max(float v) {
  v = fmaxf(v, dpp_f<kDppQuadXor1>(v));
  v = fmaxf(v, dpp_f<kDppQuadXor2>(v));
  if constexpr (T == 8) v = fmaxf(v, dpp_f<kDppRowHalfMirror>(v));
  return v;
}

__device__ __forceinline__ float root(float v) { return sqrtf(v); }
__device__ __forceinline__ double root(double v) { return sqrt(v); }
__device__ __forceinline__ float rounded(float v) { return v; }
__device__ __forceinline__ float rounded(double v) { return odd_float(v); }

// Norm (w not null) and rotation of a head's dims x in A; keys on their way to e4m3 in
// double, so that they round as the formula's values do (fp32 moves one in 2^19 across a
// rounding's border, and the next one to read the cache sees 2^-3 of it).
template <int D, class A>
__device__ __forceinline__ void norm_rope(float (&x)[2][8], const float (*w)[8], float eps, const f32x4* rot) {
  A y[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) y[i][e] = static_cast<A>(x[i][e]);
  if (w) {
    A sq = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) sq += y[i][e] * y[i][e];
    const A r = A(1) / root(head_sum<D / 16>(sq) / A(D) + A(eps));
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) y[i][e] = y[i][e] * r * static_cast<A>(w[i][e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const A cs = rot[e / 2][2 * (e & 1)], sn = rot[e / 2][2 * (e & 1) + 1];
    x[0][e] = rounded(y[0][e] * cs - y[1][e] * sn);
    x[1][e] = rounded(y[1][e] * cs + y[0][e] * sn);
  }
}

template <int D>
__device__ __forceinline__ void load_head(const NormRopeParams& p, int64_t n, int hh, int t, float (&x)[2][8]) {
  const int64_t src = n * p.qkv_ld + static_cast<int64_t>(hh) * D + 8 * t;
  load8(p.qkv, p.dt, src, p.vec, x[0]);
  load8(p.qkv, p.dt, src + D / 2, p.vec, x[1]);
}

template <int D>
__device__ __forceinline__ void load_weight(const void* w, const NormRopeParams& p, int t, float (&f)[2][8]) {
  load8(w, p.dt, 8 * t, p.vec, f[0]);
  load8(w, p.dt, D / 2 + 8 * t, p.vec, f[1]);
}

template <int D>
__device__ __forceinline__ void load_rot(const NormRopeParams& p, int64_t n, int t, f32x4* rot) {
#pragma unroll
  for (int e = 0; e < 4; ++e) rot[e] = reinterpret_cast<const f32x4*>(p.table + n * D)[4 * t + e];
}

template <int D>
__device__ __forceinline__ void store_query(const NormRopeParams& p, int64_t n, int hh, int t, bool ok, float (&x)[2][8]) {
  if (!ok) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[0][e] = x[1][e] = __builtin_nanf("");
  }
  const int64_t dst = n * p.q_sn + static_cast<int64_t>(hh) * p.q_sh + 8 * t;
  store8(p.q_out, p.dt, dst, p.vec, x[0]);
  store8(p.q_out, p.dt, dst + D / 2, p.vec, x[1]);
}

// 8 values over a scale, as e4m3 numbers.
__device__ __forceinline__ u32x2 fp8_codes(const float (&x)[8], float inv) {
  float c[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = fabsf(x[e]) < __builtin_inff() ? x[e] * inv : __builtin_nanf("");
  return u32x2{fp8_round(c[0], c[1], c[2], c[3]), fp8_round(c[4], c[5], c[6], c[7])};
}

// One head of an 8-bit cache: its codes and scales.
struct Fp8Head {
  char* codes;
  float* scales;
  int64_t sl;
};
__device__ __forceinline__ Fp8Head fp8_head(const KvFp8& kv, bool is_v, int64_t b, int h) {
  return is_v ? Fp8Head{const_cast<char*>(kv.vc) + b * kv.vc_sb + h * kv.vc_sh, const_cast<float*>(kv.vs) + b * kv.vs_sb + h * kv.vs_sh, kv.vc_sl}
              : Fp8Head{const_cast<char*>(kv.kc) + b * kv.kc_sb + h * kv.kc_sh, const_cast<float*>(kv.ks) + b * kv.ks_sb + h * kv.ks_sh, kv.kc_sl};
}

// Scale of a block after tokens of largest magnitude `top`: a block that holds earlier tokens keeps
// its own while they fit.
__device__ __forceinline__ float fp8_next_scale(bool held, float old, float top) {
  return held && top <= kFp8Max * old ? old : fp8_scale(top);
}

// A wave per token (the caches' own type, any tokens; 8 bits, one token of each row), 64 / T
// heads of it at a time; few tokens spread their heads over blocks (grid y).
template <int D, bool FP8>
__global__ void __launch_bounds__(256) norm_rope_kv_append_kernel(NormRopeParams p) {
  constexpr int T = D / 16, HW = 64 / T;
  const int lane = threadIdx.x & 63, t = lane % T, heads = p.n_q + p.n_k + p.n_v;
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= p.N) return;
  const int pos = FP8 ? p.start[n] : p.pos[n], b = !FP8 && p.batch ? p.batch[n] : n;
  const bool ok = pos >= 0 && pos < p.Lmax && b >= 0 && b < p.B;
  f32x4 rot[4];  // (cos, sin) of pairs 8 t .. 8 t + 7
  load_rot<D>(p, n, t, rot);
  for (int h0 = blockIdx.y * HW; h0 < heads; h0 += gridDim.y * HW) {
    const int hh = min(h0 + lane / T, heads - 1);  // lanes past the last head repeat it
    const bool live = h0 + lane / T < heads;
    const bool is_q = hh < p.n_q, is_v = hh >= p.n_q + p.n_k;
    float x[2][8];
    load_head<D>(p, n, hh, t, x);
    if (!is_v) {
      const void* wp = is_q ? p.q_norm : p.k_norm;
      float w[2][8];
      if (wp) load_weight<D>(wp, p, t, w);
      if constexpr (FP8) norm_rope<D, double>(x, wp ? w : nullptr, p.eps, rot);
      else norm_rope<D, float>(x, wp ? w : nullptr, p.eps, rot);
    }
    if (is_q) {
      if (live) store_query<D>(p, n, hh, t, ok, x);
      continue;
    }
    if (!live || !ok) continue;
    const int h = hh - p.n_q - (is_v ? p.n_k : 0);
    if constexpr (!FP8) {
      const int64_t dst = is_v ? b * p.v_sb + h * p.v_sh + pos * p.v_sl + 8 * t : b * p.k_sb + h * p.k_sh + pos * p.k_sl + 8 * t;
      void* cache = is_v ? p.v_cache : p.k_cache;
      store8(cache, p.dt, dst, p.vec, x[0]);
      store8(cache, p.dt, dst + D / 2, p.vec, x[1]);
    } else {
      const Fp8Head c = fp8_head(p.kv, is_v, b, h);
      const int block = pos >> p.kv.shift, first = block << p.kv.shift;
      const float old = c.scales[block];
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fmaxf(fp8_size(x[0][e]), fp8_size(x[1][e])));
      top = head_max<T>(top);
      const float s = fp8_next_scale(pos > first, old, top), inv = fp8_inverse(s);
      char* row = c.codes + pos * c.sl + 8 * t;
      *reinterpret_cast<u32x2*>(row) = fp8_codes(x[0], inv);
      *reinterpret_cast<u32x2*>(row + D / 2) = fp8_codes(x[1], inv);
      if (s != old) {
        if (t == 0) c.scales[block] = s;
        for (int i = first; i < pos; ++i) {  // one 16-byte piece of a row per thread
          u32x4* at = reinterpret_cast<u32x4*>(c.codes + i * c.sl + 16 * t);
          *at = fp8_rescaled(*at, old * inv);
        }
      }
    }
  }
}

static int head_passes(const NormRopeParams& p) {
  const int hw = 64 / (p.d / 16);
  return p.N < 1024 ? (p.n_q + p.n_k + p.n_v + hw - 1) / hw : 1;
}

hipError_t launch_norm_rope_kv_append(const NormRopeParams& p, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>((p.N + 3) / 4), head_passes(p));
  if (p.d == 128) hipLaunchKernelGGL((norm_rope_kv_append_kernel<128, false>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((norm_rope_kv_append_kernel<64, false>), grid, dim3(256), 0, st, p);
  return hipGetLastError();
}

// Several tokens of a row into an 8-bit cache: a block of threads per block of positions that the
// call touches and head (grid y), its tokens' values in registers until their largest is known.
// Blocks of positions are counted off row by row: row i with tokens o_i .. touches at most
// o_(i+1) / S - o_i / S + 2 blocks of S, so that block w belongs to the last row whose
// o_i / S + 2 i is at most w.
template <int D, int TPT, int NT>
__global__ void __launch_bounds__(NT) norm_rope_kv_append_fp8_kernel(NormRopeParams p) {
  constexpr int T = D / 16, HEADS = NT / T;  // tokens side by side
  __shared__ float red[NT / kWave], old_sh;
  const int tid = threadIdx.x, lane = tid & 63, t = tid % T, hh = blockIdx.y, shift = p.kv.shift;
  int row = 0;
  int64_t w = blockIdx.x, o0, o1;
  if (p.offsets) {
    int below = 0;
    for (int i0 = 0; i0 < p.rows; i0 += 64) {
      const int i = i0 + lane;
      const bool hit = i < p.rows && (max(p.offsets[min(i, p.rows - 1)], 0) >> shift) + 2LL * i <= w;
      below += __popcll(__ballot(hit));
    }
    row = max(below - 1, 0);
    o0 = max(p.offsets[row], 0);
    o1 = p.offsets[row + 1];
    w -= (o0 >> shift) + 2LL * row;
  } else {
    const int per = p.N / p.rows, each = (per >> shift) + 2;
    row = static_cast<int>(w / each);
    w -= static_cast<int64_t>(row) * each;
    o0 = static_cast<int64_t>(row) * per;
    o1 = o0 + per;
  }
  o1 = min(o1, static_cast<int64_t>(p.N));
  const int64_t at = p.start[row], start = max(at, static_cast<int64_t>(0)), len = o1 - o0;
  const bool ok = at >= 0 && at + len <= p.Lmax;
  const int64_t first = ((start >> shift) + w) << shift;  // the block's first position
  if (w < 0 || len <= 0 || first >= start + len) return;
  const bool is_q = hh < p.n_q, is_v = hh >= p.n_q + p.n_k;
  if (!is_q && !ok) return;

  float x[TPT][2][8];
  bool live[TPT];
#pragma unroll
  for (int i = 0; i < TPT; ++i) {
    const int64_t pos = first + i * HEADS + tid / T;
    live[i] = pos >= start && pos < start + len;
    if (live[i]) load_head<D>(p, o0 + (pos - start), hh, t, x[i]);
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][0][e] = x[i][1][e] = 0.f;
    }
  }
  if (!is_v) {
    const void* wp = is_q ? p.q_norm : p.k_norm;
    float nw[2][8];
    if (wp) load_weight<D>(wp, p, t, nw);
#pragma unroll
    for (int i = 0; i < TPT; ++i) {
      f32x4 rot[4];
      const int64_t n = o0 + first + i * HEADS + tid / T - start;
      load_rot<D>(p, live[i] ? n : o0, t, rot);
      if (is_q) {
        norm_rope<D, float>(x[i], wp ? nw : nullptr, p.eps, rot);
        if (live[i]) store_query<D>(p, n, hh, t, ok, x[i]);
      } else {
        norm_rope<D, double>(x[i], wp ? nw : nullptr, p.eps, rot);
      }
    }
    if (is_q) return;
  }
  const Fp8Head c = fp8_head(p.kv, is_v, row, hh - p.n_q - (is_v ? p.n_k : 0));
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < TPT; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (live[i]) top = fmaxf(top, fmaxf(fp8_size(x[i][0][e]), fp8_size(x[i][1][e])));
  top = wave_max(top);
  if (lane == 0) red[tid >> 6] = top;
  if (tid == 0) old_sh = c.scales[first >> shift];
  __syncthreads();
  top = red[0];
#pragma unroll
  for (int i = 1; i < NT / kWave; ++i) top = fmaxf(top, red[i]);
  const float old = old_sh, s = fp8_next_scale(first < start, old, top), inv = fp8_inverse(s);
#pragma unroll
  for (int i = 0; i < TPT; ++i) {
    if (!live[i]) continue;
    char* dst = c.codes + (first + i * HEADS + tid / T) * c.sl + 8 * t;
    *reinterpret_cast<u32x2*>(dst) = fp8_codes(x[i][0], inv);
    *reinterpret_cast<u32x2*>(dst + D / 2) = fp8_codes(x[i][1], inv);
  }
  if (s != old) {
    if (tid == 0) c.scales[first >> shift] = s;
    for (int64_t pos = first + tid / T; pos < start; pos += HEADS) {
      u32x4* piece = reinterpret_cast<u32x4*>(c.codes + pos * c.sl + 16 * t);
      *piece = fp8_rescaled(*piece, old * inv);
    }
  }
}

template <int D, int TPT, int NT>
static void launch_append_fp8(const NormRopeParams& p, hipStream_t st) {
  const int64_t blocks = p.offsets ? (p.N >> p.kv.shift) + 2LL * p.rows : ((p.N / p.rows >> p.kv.shift) + 2LL) * p.rows;
  const dim3 grid(static_cast<unsigned>(blocks), p.n_q + p.n_k + p.n_v);
  hipLaunchKernelGGL((norm_rope_kv_append_fp8_kernel<D, TPT, NT>), grid, dim3(NT), 0, st, p);
}

hipError_t launch_norm_rope_kv_append_fp8(const NormRopeParams& p, hipStream_t st) {
  if (!p.offsets && p.N == p.rows) {
    const dim3 grid(static_cast<unsigned>((p.N + 3) / 4), head_passes(p));
    if (p.d == 128) hipLaunchKernelGGL((norm_rope_kv_append_kernel<128, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((norm_rope_kv_append_kernel<64, true>), grid, dim3(256), 0, st, p);
  } else if (p.d == 128) {
    if (p.kv.shift == 5) launch_append_fp8<128, 1, 256>(p, st);
    else if (p.kv.shift == 6) launch_append_fp8<128, 2, 256>(p, st);
    else launch_append_fp8<128, 4, 256>(p, st);
  } else {
    if (p.kv.shift == 5) launch_append_fp8<64, 1, 128>(p, st);
    else if (p.kv.shift == 6) launch_append_fp8<64, 1, 256>(p, st);
    else launch_append_fp8<64, 2, 256>(p, st);
  }
  return hipGetLastError();
}

// One thread per 8 consecutive dims of a (token, head).
__global__ void __launch_bounds__(256) kv_fp8_read_kernel(KvFp8ReadParams p) {
  const int per = p.kv.d / 8, heads = p.kv.n_k + p.kv.n_v;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (item >= static_cast<int64_t>(p.N) * heads * per) return;
  const int64_t rowi = item / per;
  const int t = static_cast<int>(item - rowi * per);
  const int n = static_cast<int>(rowi / heads), hh = static_cast<int>(rowi - static_cast<int64_t>(n) * heads);
  const int pos = p.pos[n], b = p.batch ? p.batch[n] : n;
  const bool is_v = hh >= p.kv.n_k;
  const int h = hh - (is_v ? p.kv.n_k : 0);
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __builtin_nanf("");
  if (pos >= 0 && pos < p.kv.Lmax && b >= 0 && b < p.kv.B) {
    const Fp8Head c = fp8_head(p.kv, is_v, b, h);
    const float s = c.scales[pos >> p.kv.shift];
    const u32x2 v = *reinterpret_cast<const u32x2*>(c.codes + pos * c.sl + 8 * t);
    float f[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fp8_open(v[i], f);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = q4_in_range(fp8_value(f[e], s), p.dt);
    }
  }
  if (is_v) store8(p.v, p.dt, static_cast<int64_t>(n) * p.v_sn + static_cast<int64_t>(h) * p.v_sh + 8 * t, p.vec, x);
  else store8(p.k, p.dt, static_cast<int64_t>(n) * p.k_sn + static_cast<int64_t>(h) * p.k_sh + 8 * t, p.vec, x);
}

hipError_t launch_kv_fp8_read(const KvFp8ReadParams& p, hipStream_t st) {
  const int64_t items = static_cast<int64_t>(p.N) * (p.kv.n_k + p.kv.n_v) * (p.kv.d / 8);
  hipLaunchKernelGGL(kv_fp8_read_kernel, dim3(static_cast<unsigned>((items + 255) / 256)), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace saga
