// New tokens into a cache: norms of queries and keys per head, rotary embedding and append
// in one pass, into a cache of the tokens' own type or one of 8 bits; rows of an
// 8-bit cache read back.  Formats: saga_amd.h.
//
// A token's head x [d]: y = x / sqrt(mean x^2 + eps) * w, then the pairs (i, i + d / 2) turned by
// the token's rotations; values are stored as they come.  T = d / 16 threads take a head, dims
// 8 t .. and d / 2 + 8 t .., the rotary partners: the mean is a sum over T lanes, everything
// else stays in a thread.  Bound by the projection read once and written once: 4001 tokens of 15 heads
// of 128 (32.8 MB) 9.3 us, few tokens by a launch and two round trips (one token 2.7, 8 tokens into 8
// bits 4.6), 8-bit appends of prompts besides by the keys' doubles and a barrier per head (9001 tokens
// of 25 heads of 64, 52 MB, 19.4 us).  A token that raises its block's scale rounds the rows before it one
// after another: 8 tokens, the last of their blocks of 32, 64 or 128 positions, 17.6, 29.0 and 54.2 us.
#include <algorithm>

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

// 8 elements of a row on their way from memory: of a 16-bit type in 16-byte vectors (VT its code), or of
// any type and alignment (VT 0).
template <int VT>
struct Piece {
  u32x4 v;
  __device__ __forceinline__ void load(const void* base, int, int64_t off) { v = ld16(static_cast<const uint16_t*>(base) + off); }
  __device__ __forceinline__ void open(float (&f)[8]) const { unpack16<VT>(v, f); }
};
template <>
struct Piece<0> {
  float f[8];
  __device__ __forceinline__ void load(const void* base, int dt, int64_t off) { load8(base, dt, off, false, f); }
  __device__ __forceinline__ void open(float (&o)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = f[e];
  }
};

// A thread's dims of a head, of the norms, and the rotations of its pairs.
template <int VT>
struct HeadDims {
  Piece<VT> p[2];
  template <int D>
  __device__ __forceinline__ void load(const void* base, int dt, int64_t off, int t) {
    p[0].load(base, dt, off + 8 * t);
    p[1].load(base, dt, off + D / 2 + 8 * t);
  }
  __device__ __forceinline__ void open(float (&f)[2][8]) const {
    p[0].open(f[0]);
    p[1].open(f[1]);
  }
};
struct Rotations {
  f32x4 r[4];  // (cos, sin) of pairs 8 t .. 8 t + 7
  template <int D>
  __device__ __forceinline__ void load(const NormRopeParams& p, int64_t n, int t) {
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = reinterpret_cast<const f32x4*>(p.table + n * D)[4 * t + e];
  }
};

// The norms, loaded without a branch (which would be waited for): where there is none, other memory
// of at least its size.
template <int VT>
struct Norms {
  HeadDims<VT> q, k;
  template <int D>
  __device__ __forceinline__ void load(const NormRopeParams& p, int t) {
    q.template load<D>(p.q_norm ? p.q_norm : p.table, p.dt, 0, t);
    k.template load<D>(p.k_norm ? p.k_norm : p.table, p.dt, 0, t);
  }
};

// Norm (w: its weights, where `normed`) and rotation of a head's dims x.
template <int D>
__device__ __forceinline__ void norm_rope(float (&x)[2][8], bool normed, const float (&w)[2][8], float eps, const Rotations& rot) {
  if (normed) {
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) sq = __builtin_fmaf(x[i][e], x[i][e], sq);
    const float r = 1.f / sqrtf(head_sum<D / 16>(sq) / D + eps);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = x[i][e] * r * w[i][e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float cs = rot.r[e / 2][2 * (e & 1)], sn = rot.r[e / 2][2 * (e & 1) + 1], x0 = x[0][e], x1 = x[1][e];
    x[0][e] = x0 * cs - x1 * sn;
    x[1][e] = x1 * cs + x0 * sn;
  }
}

// The same for keys on their way to e4m3, in double and rounded to odd floats, so that they round as
// the formula's values do (fp32 moves one in 2^19 across a rounding's border, and whoever reads
// the cache sees 2^-3 of it).  F16: products of two f16 numbers are floats (22 bits from 2^-48 to 2^32);
// those of bf16 numbers leave a float's range.
template <int D, bool F16>
__device__ __forceinline__ void norm_rope_exact(float (&x)[2][8], bool normed, const float (&w)[2][8], float eps, const Rotations& rot) {
  double r = 1.0;
  if (normed) {
    double sq = 0.0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (F16) sq += static_cast<double>(x[i][e] * x[i][e]);
        else sq = __builtin_fma(static_cast<double>(x[i][e]), static_cast<double>(x[i][e]), sq);
      }
    r = 1.0 / sqrt(head_sum<D / 16>(sq) / D + static_cast<double>(eps));
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    double y[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (F16) {
        y[i] = normed ? x[i][e] * w[i][e] : x[i][e];
      } else {
        float xe = x[i][e], we = w[i][e];
        // (doubles made here: those of the sum, or of the norm ahead of the heads' loop, cost 40 registers)
        asm volatile("" : "+v"(xe), "+v"(we));
        y[i] = normed ? static_cast<double>(xe) * static_cast<double>(we) : static_cast<double>(xe);
      }
    }
    const double cs = rot.r[e / 2][2 * (e & 1)], sn = rot.r[e / 2][2 * (e & 1) + 1];
    x[0][e] = odd_float(__builtin_fma(y[0], cs, -(y[1] * sn)) * r);
    x[1][e] = odd_float(__builtin_fma(y[1], cs, y[0] * sn) * r);
    __builtin_amdgcn_sched_barrier(0);  // one pair's doubles at a time
  }
}

template <int VT, int D>
__device__ __forceinline__ void store_dims(void* base, int dt, int64_t off, int t, const float (&x)[2][8]) {
  store8(base, VT ? VT : dt, off + 8 * t, VT != 0, x[0]);
  store8(base, VT ? VT : dt, off + D / 2 + 8 * t, VT != 0, x[1]);
}

template <int VT, int D>
__device__ __forceinline__ void store_query(const NormRopeParams& p, int64_t n, int hh, int t, bool ok, float (&x)[2][8]) {
  if (!ok) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[0][e] = x[1][e] = __builtin_nanf("");
  }
  store_dims<VT, D>(p.q_out, p.dt, n * p.q_sn + static_cast<int64_t>(hh) * p.q_sh, t, x);
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
// heads of it at a time, the next ones' loads in flight; few tokens spread their heads over
// blocks (grid y).
template <int VT, int D, bool FP8>
__global__ void __launch_bounds__(256) norm_rope_kv_append_kernel(NormRopeParams p) {
  constexpr int T = D / 16, HW = 64 / T;
  const int lane = threadIdx.x & 63, t = lane % T, heads = p.n_q + p.n_k + p.n_v;
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= p.N) return;
  const int pos = FP8 ? p.start[n] : p.pos[n], b = !FP8 && p.batch ? p.batch[n] : n;
  const int64_t src = static_cast<int64_t>(n) * p.qkv_ld;
  const int step = gridDim.y * HW;
  HeadDims<VT> next;
  next.template load<D>(p.qkv, p.dt, src + static_cast<int64_t>(min(static_cast<int>(blockIdx.y) * HW + lane / T, heads - 1)) * D, t);
  Rotations rot;
  rot.template load<D>(p, n, t);
  Norms<VT> norms;
  norms.template load<D>(p, t);
  const bool ok = pos >= 0 && pos < p.Lmax && b >= 0 && b < p.B;
  for (int h0 = blockIdx.y * HW; h0 < heads; h0 += step) {
    const int hh = min(h0 + lane / T, heads - 1);  // lanes past the last head repeat it
    const bool live = h0 + lane / T < heads;
    const bool is_q = hh < p.n_q, is_v = hh >= p.n_q + p.n_k;
    const int h = hh - p.n_q - (is_v ? p.n_k : 0);
    Fp8Head c{};
    int block = 0;
    float old = 0.f;
    if constexpr (FP8) {
      c = fp8_head(p.kv, is_v, ok ? b : 0, max(h, 0));
      block = ok ? pos >> p.kv.shift : 0;
      old = c.scales[block];
    }
    float x[2][8];
    next.open(x);
    if (h0 + step < heads)
      next.template load<D>(p.qkv, p.dt, src + static_cast<int64_t>(min(h0 + step + lane / T, heads - 1)) * D, t);
    if (!is_v) {
      float w[2][8], wk[2][8];
      norms.q.open(w);
      norms.k.open(wk);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) w[i][e] = is_q ? w[i][e] : wk[i][e];
      const bool normed = is_q ? p.q_norm != nullptr : p.k_norm != nullptr;
      if constexpr (FP8) norm_rope_exact<D, VT == SAGA_DTYPE_F16>(x, normed, w, p.eps, rot);
      else norm_rope<D>(x, normed, w, p.eps, rot);
    }
    if (is_q) {
      if (live) store_query<VT, D>(p, n, hh, t, ok, x);
      continue;
    }
    if (!live || !ok) continue;
    if constexpr (!FP8) {
      store_dims<VT, D>(is_v ? p.v_cache : p.k_cache, p.dt,
                        is_v ? b * p.v_sb + h * p.v_sh + pos * p.v_sl : b * p.k_sb + h * p.k_sh + pos * p.k_sl, t, x);
    } else {
      const int first = block << p.kv.shift;
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

template <int D, bool FP8>
static void launch_append(const NormRopeParams& p, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>((p.N + 3) / 4), head_passes(p));
  if (!p.vec) hipLaunchKernelGGL((norm_rope_kv_append_kernel<0, D, FP8>), grid, dim3(256), 0, st, p);
  else if (p.dt == SAGA_DTYPE_BF16) hipLaunchKernelGGL((norm_rope_kv_append_kernel<SAGA_DTYPE_BF16, D, FP8>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((norm_rope_kv_append_kernel<SAGA_DTYPE_F16, D, FP8>), grid, dim3(256), 0, st, p);
}

hipError_t launch_norm_rope_kv_append(const NormRopeParams& p, hipStream_t st) {
  if (p.d == 128) launch_append<128, false>(p, st);
  else launch_append<64, false>(p, st);
  return hipGetLastError();
}

// Several tokens of a row into an 8-bit cache: a block of threads per block of S positions that the
// call touches and run of heads (grid y).  T threads a token, HS heads side by side, a token's
// rotations in registers for all heads, the next head's values in flight, a head's in
// registers until the largest of its block is known.  Blocks of positions are counted off row by
// row: row i with tokens o_i .. touches at most o_(i+1) / S - o_i / S + 2 of them, so
// that block w belongs to the last row whose o_i / S + 2 i is at most w.
template <int D, int S>
struct AppendShape {
  static constexpr int T = D / 16, NT = S * T < 256 ? 256 : S * T;
  static constexpr int HS = NT / (S * T), HW = NT / kWave / HS;  // heads side by side, waves of a head
};

template <int VT, int D, int S>
__global__ void __launch_bounds__((AppendShape<D, S>::NT)) norm_rope_kv_append_fp8_kernel(NormRopeParams p) {
  using A = AppendShape<D, S>;
  constexpr int T = A::T, HS = A::HS;
  constexpr int shift = S == 32 ? 5 : S == 64 ? 6 : 7;
  __shared__ float red[2][A::NT / kWave], old_sh[2][HS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, t = tid % T;
  const int side = tid / T % S, hs = tid / (T * S);  // token of the block, head of those side by side (a wave's)
  int row = 0;
  int64_t w = blockIdx.x, o0, o1;
  if (p.offsets) {
    int below = 0;
    for (int i0 = 0; i0 < p.rows; i0 += 64) {
      const int i = i0 + lane;
      const bool hit = i < p.rows && (max(p.offsets[min(i, p.rows - 1)], 0) >> shift) + 2LL * i <= w;
      below += __popcll(__ballot(hit));
    }
    row = __builtin_amdgcn_readfirstlane(max(below - 1, 0));
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
  const int heads = ok ? p.n_q + p.n_k + p.n_v : p.n_q;
  const int run = (p.n_q + p.n_k + p.n_v + gridDim.y - 1) / gridDim.y;
  const int h0 = blockIdx.y * run, h1 = min(h0 + run, heads);
  if (h0 >= h1) return;

  const int64_t pos = first + side;
  const bool live = pos >= start && pos < start + len;
  const int64_t n = live ? o0 + (pos - start) : o0;  // this thread's token, the row's first one where there is none
  HeadDims<VT> next;
  auto load_next = [&](int hh) { next.template load<D>(p.qkv, p.dt, n * p.qkv_ld + static_cast<int64_t>(min(hh, h1 - 1)) * D, t); };
  load_next(h0 + hs);
  Rotations rot;
  rot.template load<D>(p, n, t);
  Norms<VT> norms;
  norms.template load<D>(p, t);

  int turn = 0;
  for (int hb = h0; hb < h1; hb += HS) {
    const int hh = min(hb + hs, h1 - 1);
    const bool mine = hb + hs < h1, is_q = hh < p.n_q, is_v = hh >= p.n_q + p.n_k;
    float x[2][8], nw[2][8];
    next.open(x);
    if (hb + HS < h1) load_next(hb + HS + hs);
    if (is_q) {
      norms.q.open(nw);
      norm_rope<D>(x, p.q_norm != nullptr, nw, p.eps, rot);
      if (live && mine) store_query<VT, D>(p, n, hh, t, ok, x);
    } else if (!is_v) {
      norms.k.open(nw);
      norm_rope_exact<D, VT == SAGA_DTYPE_F16>(x, p.k_norm != nullptr, nw, p.eps, rot);
    }
    if (min(hb + HS, h1) <= p.n_q) continue;  // the whole block holds queries
    const Fp8Head c = fp8_head(p.kv, is_v, row, is_q ? 0 : hh - p.n_q - (is_v ? p.n_k : 0));
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (live) top = fmaxf(top, fmaxf(fp8_size(x[0][e]), fp8_size(x[1][e])));
    top = wave_max(top);
    if (lane == 0) red[turn][wave] = top;
    if (side == 0 && t == 0 && !is_q) old_sh[turn][hs] = c.scales[first >> shift];  // (read before anyone writes it)
    __syncthreads();
    top = red[turn][hs * A::HW];
#pragma unroll
    for (int i = 1; i < A::HW; ++i) top = fmaxf(top, red[turn][hs * A::HW + i]);
    if (!is_q && mine) {
      const float old = old_sh[turn][hs], s = fp8_next_scale(first < start, old, top), inv = fp8_inverse(s);
      char* dst = c.codes + pos * c.sl;
      if (live) {
        *reinterpret_cast<u32x2*>(dst + 8 * t) = fp8_codes(x[0], inv);
        *reinterpret_cast<u32x2*>(dst + D / 2 + 8 * t) = fp8_codes(x[1], inv);
      }
      if (s != old) {
        if (side == 0 && t == 0) c.scales[first >> shift] = s;
        if (pos < start) {
          u32x4* piece = reinterpret_cast<u32x4*>(dst + 16 * t);
          *piece = fp8_rescaled(*piece, old * inv);
        }
      }
    }
    turn ^= 1;
  }
}

// Runs of four heads (the rotations and the row's search are paid per run: 9001 tokens of 25 heads of
// 64 in 1, 3, 7, 13 and 25 runs 23.2, 18.6, 17.3, 19.4 and 30.1 us; 4001 of 15 heads of 128 in 1, 2,
// 4, 8 and 15 19.5, 13.0, 10.0, 11.5 and 13.0), shorter ones where that leaves CUs idle.
template <int VT, int D, int S>
static void launch_append_fp8_typed(const NormRopeParams& p, hipStream_t st) {
  const int64_t blocks = p.offsets ? (p.N >> p.kv.shift) + 2LL * p.rows : ((p.N / p.rows >> p.kv.shift) + 2LL) * p.rows;
  const int heads = p.n_q + p.n_k + p.n_v, steps = (heads + AppendShape<D, S>::HS - 1) / AppendShape<D, S>::HS;
  const int64_t touched = (p.N >> p.kv.shift) + p.rows;
  const int runs = static_cast<int>(std::min<int64_t>(std::max<int64_t>(256 / touched, (heads + 3) / 4), steps));
  hipLaunchKernelGGL((norm_rope_kv_append_fp8_kernel<VT, D, S>), dim3(static_cast<unsigned>(blocks), runs), dim3(AppendShape<D, S>::NT), 0,
                     st, p);
}

template <int D, int S>
static void launch_append_fp8(const NormRopeParams& p, hipStream_t st) {
  if (!p.vec) launch_append_fp8_typed<0, D, S>(p, st);
  else if (p.dt == SAGA_DTYPE_BF16) launch_append_fp8_typed<SAGA_DTYPE_BF16, D, S>(p, st);
  else launch_append_fp8_typed<SAGA_DTYPE_F16, D, S>(p, st);
}

hipError_t launch_norm_rope_kv_append_fp8(const NormRopeParams& p, hipStream_t st) {
  if (!p.offsets && p.N == p.rows) {
    if (p.d == 128) launch_append<128, true>(p, st);
    else launch_append<64, true>(p, st);
  } else if (p.d == 128) {
    if (p.kv.shift == 5) launch_append_fp8<128, 32>(p, st);
    else if (p.kv.shift == 6) launch_append_fp8<128, 64>(p, st);
    else launch_append_fp8<128, 128>(p, st);
  } else {
    if (p.kv.shift == 5) launch_append_fp8<64, 32>(p, st);
    else if (p.kv.shift == 6) launch_append_fp8<64, 64>(p, st);
    else launch_append_fp8<64, 128>(p, st);
  }
  return hipGetLastError();
}

// One thread per 16 consecutive dims of a (token, head); bound by two dependent round trips (the index, then
// the row): 8 tokens 3.2 us, 9001 of 10 heads of 64 (17 MB) 7.9.
__global__ void __launch_bounds__(256) kv_fp8_read_kernel(KvFp8ReadParams p) {
  const uint32_t per = p.kv.d / 16, heads = p.kv.n_k + p.kv.n_v;
  const uint32_t item = blockIdx.x * 256 + threadIdx.x, rowi = item / per;
  const int t = static_cast<int>(item - rowi * per), n = static_cast<int>(rowi / heads), hh = static_cast<int>(rowi - n * heads);
  if (n >= p.N) return;
  const int pos = p.pos[n], b = p.batch ? p.batch[n] : n;
  const bool is_v = hh >= p.kv.n_k, ok = pos >= 0 && pos < p.kv.Lmax && b >= 0 && b < p.kv.B;
  const int h = hh - (is_v ? p.kv.n_k : 0), at = ok ? pos : 0;
  const Fp8Head c = fp8_head(p.kv, is_v, ok ? b : 0, h);
  const float s = c.scales[at >> p.kv.shift];
  const u32x4 v = ld16(c.codes + at * c.sl + 16 * t);
  float x[2][8], f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    fp8_open(v[i], f);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[i / 2][4 * (i % 2) + e] = ok ? q4_in_range(fp8_value(f[e], s), p.dt) : __builtin_nanf("");
  }
  void* to = is_v ? p.v : p.k;
  const int64_t off = is_v ? n * p.v_sn + h * p.v_sh + 16 * t : n * p.k_sn + h * p.k_sh + 16 * t;
  store8(to, p.dt, off, p.vec, x[0]);
  store8(to, p.dt, off + 8, p.vec, x[1]);
}

hipError_t launch_kv_fp8_read(const KvFp8ReadParams& p, hipStream_t st) {
  const int64_t items = static_cast<int64_t>(p.N) * (p.kv.n_k + p.kv.n_v) * (p.kv.d / 16);
  hipLaunchKernelGGL(kv_fp8_read_kernel, dim3(static_cast<unsigned>((items + 255) / 256)), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace saga
