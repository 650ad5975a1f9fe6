// Skinny GEMM with weights in 4 bits: y[m, n] = sum_k x[m, k] (s c + z)[n, k], m < 32.
//
// The weight stream of gemv.hip with a quarter of its bytes.  x is the A operand
// (token rows), 16 rows of W the B operand: a lane then holds one row n of the
// product and needs one (s, z) pair per group.  Per group of G columns
//   sum_k x (s c + z) = s (sum_k x (b + c) - sum_k x b) + z sum_k x,
// with the codes as b + c (q4.cuh): an MFMA chain each for the three sums, the first
// starting from the second, exact products summed in fp32.  The sums without codes are
// shared by a workgroup's tiles.  The RMSNorm's sum of squares is the diagonal of x x^T,
// an MFMA more per fragment.
//
// Bound by the weight stream from some 10 MB on (the LM head of 151936 x 1536, 131 MB,
// 28-29 us at up to 16 rows of x, 4.6 TB/s); below by a launch and two round trips (960 x
// 960 3.3 us in a graph), and with many rows by reading x: 96 tiles of K 8960 read 143 KB
// of x per workgroup at 8 rows.  Bias and residual are loaded behind the sums: 1536 x 1536 at
// 8 rows 3.9 us stored, 4.3 with norm and bias, 5.1 added to y.
#include <algorithm>

#include "kernels.h"
#include "q4.cuh"

namespace saga {

__device__ __forceinline__ f32x4 mfma_bf16(const u32x4& a, const u32x4& b, f32x4 c) {
  return mfma_16b<SAGA_DTYPE_BF16>(a, b, c);
}

// Finishes a (tile, token tile): lane (col, s) holds the sums v of row n = 16 tile + col of W
// and tokens m0 + r, sq their sums of squares (where the RMSNorm is fused).
template <int EPI>
__device__ __forceinline__ void gemv_q4_finish(const GemvQ4Params& p, int n, int m0, const f32x4& v, const f32x4& sq) {
  float bias = 0.f;
  if (EPI != SAGA_GEMV_SILU_PAIRS && p.bias) bias = bf16_bits_to_f32(static_cast<const uint16_t*>(p.bias)[n]);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int m = m0 + r;
    float o = v[r];
    if (p.rms) o *= rsqrtf(sq[r] / static_cast<float>(p.K) + p.eps);
    uint16_t* y = static_cast<uint16_t*>(p.y) + static_cast<int64_t>(m) * p.y_ld;
    if constexpr (EPI == SAGA_GEMV_SILU_PAIRS) {
      const float up = __shfl_xor(o, 1);  // rows (n, n + 1): gate, up
      if (m < p.M && (n & 1) == 0) y[n / 2] = f32_to_bf16_bits(o / (1.0f + expf(-o)) * up);
    } else {
      if (p.bias) o += bias;
      if (m < p.M) {
        if constexpr (EPI == SAGA_GEMV_ADD) o += bf16_bits_to_f32(y[n]);
        y[n] = f32_to_bf16_bits(o);
      }
    }
  }
}

// Workgroup: TPW tiles of 16 rows of W and (with several ranges) one range of the
// units of 128 columns, which its waves split (wave w takes units w, w + WAVES, ...)
// and join in LDS.  U units per wave in flight.  MT tiles of 16 token rows.  TAIL: K
// is no multiple of 128.
template <int EPI, int G, int MT, int WAVES, int TPW, int U, bool TAIL>
__global__ void __launch_bounds__(WAVES * 64) gemv_q4_kernel(GemvQ4Params p) {
  constexpr int NG = 128 / G;  // groups of a unit
  __shared__ float red[WAVES][TPW * MT][64][4];
  __shared__ float rsq[WAVES][16 * MT];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, s = lane >> 4;
  const int tile0 = blockIdx.x * TPW;
  const int units = (p.K + 127) / 128, steps = p.K / 32, groups = p.K / G;
  const int k0 = blockIdx.y * units / p.splits, k1 = (blockIdx.y + 1) * units / p.splits;
  const char* code = static_cast<const char*>(p.codes) + static_cast<int64_t>(tile0) * units * 1024 + lane * 16;
  const char* scale = static_cast<const char*>(p.scales) + static_cast<int64_t>(tile0) * groups * 64 + col * 4;
  const char* xrow[MT];  // rows past the last token repeat the first: their sums are not stored
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
    xrow[mt] = static_cast<const char*>(p.x) +
               (static_cast<int64_t>(col + 16 * mt < p.M ? col + 16 * mt : 0) * p.x_ld + 8 * s) * 2;
  f32x4 acc[TPW][MT], sq[MT];
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    sq[mt] = zero;
#pragma unroll
    for (int t = 0; t < TPW; ++t) acc[t][mt] = zero;
  }
  const u32x4 ones = {kBf16Ones, kBf16Ones, kBf16Ones, kBf16Ones};
  const Q4Const qc;
  for (int u0 = k0 + w; u0 < k1; u0 += U * WAVES) {
    u32x4 cw[U][TPW], xf[U][MT][4];
    uint32_t sz[U][TPW][NG];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int J = min(u0 + u * WAVES, k1 - 1);
#pragma unroll
      for (int t = 0; t < TPW; ++t) {
        cw[u][t] = ld16(code + (static_cast<int64_t>(t) * units + J) * 1024);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const int gi = TAIL ? min(J * NG + g, groups - 1) : J * NG + g;
          sz[u][t][g] = *reinterpret_cast<const uint32_t*>(scale + (static_cast<int64_t>(t) * groups + gi) * 64);
        }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          xf[u][mt][j] = ld16(xrow[mt] + static_cast<int64_t>(TAIL ? min(4 * J + j, steps - 1) : 4 * J + j) * 64);
          if (TAIL && 4 * J + j >= steps) xf[u][mt][j] = u32x4{0u, 0u, 0u, 0u};
        }
    }
    __builtin_amdgcn_sched_barrier(0);  // the whole burst is in flight
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u > 0 && u0 + u * WAVES >= k1) break;
      if (p.rms) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int j = 0; j < 4; ++j) sq[mt] = mfma_bf16(xf[u][mt][j], xf[u][mt][j], sq[mt]);
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        f32x4 xs[MT], xb[MT];  // sums of x, and of x times minus what the operand adds to its codes
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          xs[mt] = xb[mt] = zero;
#pragma unroll
          for (int j = g * (G / 32); j < (g + 1) * (G / 32); ++j) {
            xs[mt] = mfma_bf16(xf[u][mt][j], ones, xs[mt]);
            xb[mt] = mfma_bf16(xf[u][mt][j], q4_minus_base(), xb[mt]);
          }
        }
#pragma unroll
        for (int t = 0; t < TPW; ++t) {
          f32x4 d[MT];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) d[mt] = xb[mt];
#pragma unroll
          for (int j = g * (G / 32); j < (g + 1) * (G / 32); ++j) {
            const u32x4 b = q4_frag(cw[u][t][j], qc);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) d[mt] = mfma_bf16(xf[u][mt][j], b, d[mt]);
          }
          const float sc = q4_lo(sz[u][t][g]), z = q4_hi(sz[u][t][g]);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              acc[t][mt][r] = __builtin_fmaf(sc, d[mt][r], __builtin_fmaf(z, xs[mt][r], acc[t][mt][r]));
        }
      }
    }
  }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int t = 0; t < TPW; ++t)
      *reinterpret_cast<f32x4*>(red[w][t * MT + mt][lane]) = acc[t][mt];
    // the diagonal of x x^T: row 4 s + r of lane column 4 s + r
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (col == 4 * s + r) rsq[w][16 * mt + col] = sq[mt][r];
  }
  lds_sync();
  // one (tile, token tile) per wave
  for (int i = w; i < TPW * MT; i += WAVES) {
    const int t = i / MT, mt = i - t * MT;
    f32x4 v = zero, q2 = zero;
#pragma unroll
    for (int q = 0; q < WAVES; ++q) {
      v += *reinterpret_cast<const f32x4*>(red[q][i][lane]);
      if (p.rms) q2 += *reinterpret_cast<const f32x4*>(&rsq[q][16 * mt + 4 * s]);
    }
    if (p.splits > 1) {
      const int64_t tile = static_cast<int64_t>(blockIdx.y) * (p.N / 16) + tile0 + t;
      *reinterpret_cast<f32x4*>(p.part + ((tile * MT + mt) * 64 + lane) * 4) = v;
      if (p.rms && tile0 + t == 0 && col == 0)
        *reinterpret_cast<f32x4*>(p.part_sq + blockIdx.y * 32 + 16 * mt + 4 * s) = q2;
    } else {
      gemv_q4_finish<EPI>(p, (tile0 + t) * 16 + col, 16 * mt + 4 * s, v, q2);
    }
  }
}

// Weights of many tiles and short rows (the LM head): a workgroup keeps its x in
// registers, with its sums per group, and streams pairs of tiles (64-byte pieces of y rows),
// the next tile's codes in flight under a tile's products.  Its waves split K (UPW units
// each) and join through LDS, two buffers, a barrier per tile; a wave then finishes tokens
// 4 s + r of a token tile.  Here every code is 16 + c, so that one sum of x serves both corrections:
//   sum x w = s D + (z - 16 s) sum x.
// With two token tiles and groups of 32 (SUMS) the second term is a product of its own, fp32
// MFMAs over four groups each: a register per four groups and token tile in place of 16, and
// an instruction in place of 16 (LM head, 32 rows, 60 -> 49 us; with larger groups 5 % slower).
template <int EPI, int G, int MT, int WAVES, int UPW>
__global__ void __launch_bounds__(WAVES * 64, 8 / WAVES) gemv_q4_stream_kernel(GemvQ4Params p) {
  constexpr int NG = 128 / G, NS = UPW * NG, NC = (NS + 3) / 4;  // groups of a wave, in fours
  constexpr bool SUMS = MT == 2 && G == 32;
  __shared__ float red[2][WAVES][MT][4][64];
  __shared__ float rsq[WAVES][16 * MT];
  constexpr int NF = (4 * MT + WAVES - 1) / WAVES;  // (token tile, r) that a wave finishes: w, w + WAVES, ...
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, s = lane >> 4;
  const int units = (p.K + 127) / 128, steps = p.K / 32, groups = p.K / G, tiles = p.N / 16;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const u32x4 ones = {kBf16Ones, kBf16Ones, kBf16Ones, kBf16Ones};
  const Q4Const qc;

  struct Tile {
    u32x4 c[UPW];
    uint32_t sz[UPW][NG];
  };
  int64_t coff[UPW], soff[UPW][NG];  // units and groups past the row repeat its last (their x is zero)
#pragma unroll
  for (int u = 0; u < UPW; ++u) {
    const int J = min(w + WAVES * u, units - 1);
    coff[u] = static_cast<int64_t>(J) * 1024 + lane * 16;
#pragma unroll
    for (int g = 0; g < NG; ++g) soff[u][g] = static_cast<int64_t>(min(J * NG + g, groups - 1)) * 64 + col * 4;
  }
  // pairs blockIdx.x, + gridDim.x, ... of tiles: the workgroups read one region at a time
  const int pairs = (tiles + 1) / 2, grid = static_cast<int>(gridDim.x), b0 = static_cast<int>(blockIdx.x);
  const int mine = (pairs - b0 + grid - 1) / grid * 2;
  auto tile_of = [&](int i) { return ((i >> 1) * grid + b0) * 2 + (i & 1); };
  auto load_tile = [&](Tile& t, int tile) {
    const int at = min(tile, tiles - 1);
    const char* code = static_cast<const char*>(p.codes) + static_cast<int64_t>(at) * units * 1024;
    const char* scale = static_cast<const char*>(p.scales) + static_cast<int64_t>(at) * groups * 64;
#pragma unroll
    for (int u = 0; u < UPW; ++u) {
      t.c[u] = ld16(code + coff[u]);
#pragma unroll
      for (int g = 0; g < NG; ++g) t.sz[u][g] = *reinterpret_cast<const uint32_t*>(scale + soff[u][g]);
    }
  };
  Tile ta, tb;
  load_tile(ta, tile_of(0));

  u32x4 xf[UPW][MT][4];
  f32x4 xs[SUMS ? 1 : UPW][NG][MT];
  float xa[NC][MT];  // SUMS: the sum over group 4 c + s of token `col`, an A operand of four groups
  float* xsum = &red[0][w][0][0][0];  // SUMS: [MT][4 NC][16 tokens]
  static_assert(!SUMS || 4 * NC * 16 <= 256, "a wave's sums of x fit its part of red");
  {
    f32x4 sq[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      sq[mt] = zero;
      const bool row = col + 16 * mt < p.M;  // rows past the last token repeat the first: not stored
      const char* xrow = static_cast<const char*>(p.x) + (static_cast<int64_t>(row ? col + 16 * mt : 0) * p.x_ld + 8 * s) * 2;
#pragma unroll
      for (int u = 0; u < UPW; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = 4 * (w + WAVES * u) + j;
          xf[u][mt][j] = ld16(xrow + static_cast<int64_t>(min(k, steps - 1)) * 64);
          if (k >= steps) xf[u][mt][j] = u32x4{0u, 0u, 0u, 0u};
        }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int u = 0; u < UPW; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int g = j * 32 / G;
          f32x4& sum = xs[SUMS ? 0 : u][g][mt];  // tokens 4 s + r, in every column
          sum = mfma_bf16(xf[u][mt][j], ones, j * 32 % G == 0 ? zero : sum);
          if (SUMS && col == 0) *reinterpret_cast<f32x4*>(xsum + (mt * 4 * NC + u * NG + g) * 16 + 4 * s) = sum;
          if (p.rms) sq[mt] = mfma_bf16(xf[u][mt][j], xf[u][mt][j], sq[mt]);
        }
#pragma unroll
      for (int r = 0; r < 4; ++r)  // the diagonal of x x^T
        if (col == 4 * s + r) rsq[w][16 * mt + col] = sq[mt][r];
    }
  }
  lds_sync();
  if constexpr (SUMS) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) xa[c][mt] = xsum[(mt * 4 * NC + 4 * c + s) * 16 + col];
  }
  float scl[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const int i = min(w + f * WAVES, 4 * MT - 1);
    scl[f] = 1.f;
    if (p.rms) {
      float q2 = 0.f;
#pragma unroll
      for (int q = 0; q < WAVES; ++q) q2 += rsq[q][16 * (i / 4) + 4 * s + i % 4];
      scl[f] = rsqrtf(q2 / static_cast<float>(p.K) + p.eps);
    }
  }

  auto use_tile = [&](const Tile& t, int tile, int buf) {
    f32x4 acc[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[mt] = zero;
    if constexpr (SUMS) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {  // (NG 4: the groups of unit c)
        uint32_t sz = t.sz[c][0];  // of this lane's group
#pragma unroll
        for (int g = 1; g < NG; ++g) sz = s == g ? t.sz[c][g] : sz;
        const float zo = __builtin_fmaf(-16.f, q4_lo(sz), q4_hi(sz));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[mt] = __builtin_amdgcn_mfma_f32_16x16x4f32(xa[c][mt], zo, acc[mt], 0, 0, 0);
      }
    }
#pragma unroll
    for (int u = 0; u < UPW; ++u)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        f32x4 d[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) d[mt] = zero;
#pragma unroll
        for (int j = g * (G / 32); j < (g + 1) * (G / 32); ++j) {
          const u32x4 b = q4_frag16(t.c[u][j], qc);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) d[mt] = mfma_bf16(xf[u][mt][j], b, d[mt]);
        }
        const float sc = q4_lo(t.sz[u][g]), zo = __builtin_fmaf(-16.f, sc, q4_hi(t.sz[u][g]));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if constexpr (SUMS) acc[mt][r] = __builtin_fmaf(sc, d[mt][r], acc[mt][r]);
            else acc[mt][r] = __builtin_fmaf(sc, d[mt][r], __builtin_fmaf(zo, xs[u][g][mt][r], acc[mt][r]));
          }
      }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[buf][w][mt][r][lane] = acc[mt][r];
    lds_sync();
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const int i = w + f * WAVES;
      if (i >= 4 * MT) break;
      float o = 0.f;
#pragma unroll
      for (int q = 0; q < WAVES; ++q) o += red[buf][q][i / 4][i % 4][lane];
      o *= scl[f];
      const int m = 16 * (i / 4) + 4 * s + i % 4, n = tile * 16 + col;
      uint16_t* y = static_cast<uint16_t*>(p.y) + static_cast<int64_t>(m) * p.y_ld;
      if constexpr (EPI == SAGA_GEMV_SILU_PAIRS) {
        const float up = __shfl_xor(o, 1);
        if (m < p.M && (n & 1) == 0 && tile < tiles) y[n / 2] = f32_to_bf16_bits(o / (1.0f + expf(-o)) * up);
      } else {
        if (m < p.M && tile < tiles) y[n] = f32_to_bf16_bits(o);
      }
    }
  };
  for (int i = 0; i < mine; i += 2) {
    load_tile(tb, tile_of(i + 1));
    __builtin_amdgcn_sched_barrier(0);
    use_tile(ta, tile_of(i), 0);
    if (i + 1 >= mine) break;
    load_tile(ta, tile_of(i + 2));
    __builtin_amdgcn_sched_barrier(0);
    use_tile(tb, tile_of(i + 1), 1);
  }
}

// Adds up the ranges, one wave per (tile, token tile).
template <int EPI>
__global__ void __launch_bounds__(64) gemv_q4_join_kernel(GemvQ4Params p, int mts) {
  const int lane = threadIdx.x, col = lane & 15, s = lane >> 4;
  const int tile = blockIdx.x / mts, mt = blockIdx.x - tile * mts;
  const int64_t stride = static_cast<int64_t>(p.N / 16) * mts * 256;  // between ranges
  const float* part = p.part + (static_cast<int64_t>(blockIdx.x) * 64 + lane) * 4;
  f32x4 v = {0.f, 0.f, 0.f, 0.f}, q2 = v;
  for (int i0 = 0; i0 < p.splits; i0 += 8) {
    f32x4 a[8], b[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = min(i0 + u, p.splits - 1);
      a[u] = *reinterpret_cast<const f32x4*>(part + i * stride);
      if (p.rms) b[u] = *reinterpret_cast<const f32x4*>(p.part_sq + i * 32 + 16 * mt + 4 * s);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u < p.splits) {
        v += a[u];
        if (p.rms) q2 += b[u];
      }
  }
  gemv_q4_finish<EPI>(p, tile * 16 + col, 16 * mt + 4 * s, v, q2);
}

// Ranges of K: few tiles of long rows (the down projection: 96 tiles, 70 units) are
// spread over about one workgroup per CU, with at least 12 units each.  Measured
// (us in a graph, 1536 x 8960, groups of 64): one range 9.0 (8 rows of x) and 19.9 (32),
// five 7.7 and 10.2, join kernel included; below 8 rows what they gain (7.8 -> 7.4 at 5)
// is less than their second launch costs an eager caller (3.3).
static int gemv_q4_splits(int64_t M, int64_t N, int64_t K) {
  const int64_t units = (K + 127) / 128;
  return M < 8 ? 1 : static_cast<int>(std::max<int64_t>(std::min(256 / ((N / 16 + 1) / 2), units / 12), 1));
}

int64_t gemv_q4_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  const int64_t s = gemv_q4_splits(M, N, K);
  return s > 1 ? s * (N * 16 * (M > 16 ? 2 : 1) + 32) * 4 : 0;
}

template <int EPI, int G, int MT, int WAVES, int TPW, int U>
static void launch_gemv_q4_shape(const GemvQ4Params& p, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.N / 16 / TPW), p.splits);
  if (p.K % 128) hipLaunchKernelGGL((gemv_q4_kernel<EPI, G, MT, WAVES, TPW, U, true>), grid, dim3(WAVES * 64), 0, st, p);
  else hipLaunchKernelGGL((gemv_q4_kernel<EPI, G, MT, WAVES, TPW, U, false>), grid, dim3(WAVES * 64), 0, st, p);
}

// Two workgroups of 4 waves per CU, or one of 8 where the rows need more registers (x and
// its sums: 24 per unit and token tile; groups of 32: 32 with one token tile, 17 with two).  Measured against workgroups
// of a few tiles (us, groups of 64; 1, 8 and 32 rows of x): 8192 tiles, K 960 14.3, 15.5, 22.6
// against 16.7, 17.6, 29.6; K 2048 -, -, 41.9 against 31.8, 34.2, 52.2 (8 rows, streamed:
// 35.3); K 2944 -, -, 53.9 against 44.1, 47.6, 72.6; K 1536 with 1280 tiles 8.0, 8.1, 13.0
// against 8.7, 9.3, 16.1, 768 6.6, 7.2, 11.4 against 7.0, 7.8, 10.9, 320 4.9, 5.5, 8.9 against
// 4.7, 5.8, 9.6.  (1120 tiles are 560 pairs: 48 workgroups take two, the others one.)
template <int EPI, int G, int MT>
static void launch_gemv_q4_stream(const GemvQ4Params& p, int units, hipStream_t st) {
  if constexpr (EPI != SAGA_GEMV_ADD) {
    const int pairs = (p.N / 16 + 1) / 2;
    const dim3 two(std::min(pairs, 512)), one(std::min(pairs, 256));
    if (units <= 4) {
      hipLaunchKernelGGL((gemv_q4_stream_kernel<EPI, G, MT, 4, 1>), two, dim3(256), 0, st, p);
    } else if (units <= 8) {
      hipLaunchKernelGGL((gemv_q4_stream_kernel<EPI, G, MT, 4, 2>), two, dim3(256), 0, st, p);
    } else if (units <= 12) {
      hipLaunchKernelGGL((gemv_q4_stream_kernel<EPI, G, MT, 4, 3>), two, dim3(256), 0, st, p);
    } else if (units <= 16) {
      if constexpr (MT == 2) hipLaunchKernelGGL((gemv_q4_stream_kernel<EPI, G, MT, 8, 2>), one, dim3(512), 0, st, p);
    } else {
      if constexpr (MT == 2 && G > 32)
        hipLaunchKernelGGL((gemv_q4_stream_kernel<EPI, G, MT, 8, 3>), one, dim3(512), 0, st, p);
    }
  }
}

// Tiles per workgroup share its reads of x and their sums, workgroups share the CUs.
// Measured (us; 1, 8 and 32 rows of x; waves x tiles x units in flight):
//   9496 tiles, K 1536: 4x4x1 29.8, 33.9, 51.7; 4x2x1 32.3, 36.2, 67.3; 4x1x3 -, 42, 127;
//     streamed with x in registers 28.0, 29.5, 37.5 (tiles one by one 27.5, 28.9, 42.5)
//   1120 tiles, K 1536: 4x2x1 8.0, 9.1, 14.8; 8x2x1 8.0, 9.6, 14.7; 4x4x1 8.8, 10.4, 14.9; 4x1x3 7.9, 9.3, 20;
//     streamed 7.7, 8.0, 13.1
//   96 tiles, K 1536: 4x1x3 3.8 (8 rows), 4x2x3 4.4, 16x1x1 4.2
//   96 tiles, K 8960, five ranges: 8x2x2 7.7 and 10.5 (32 rows), 8x2x1 7.9 and 10.2, 4x1x3 8.4
template <int EPI, int G, int MT>
static void launch_gemv_q4_rows(const GemvQ4Params& p, hipStream_t st) {
  const int tiles = p.N / 16, units = (p.K + 127) / 128;
  if (p.splits > 1) {
    if (tiles % 2 == 0) launch_gemv_q4_shape<EPI, G, MT, 8, 2, 1>(p, st);
    else launch_gemv_q4_shape<EPI, G, MT, 8, 1, 1>(p, st);
  } else if (tiles >= 256 && units <= (MT == 1 ? 12 : G == 32 ? 16 : 24) && !p.bias && EPI != SAGA_GEMV_ADD) {
    launch_gemv_q4_stream<EPI, G, MT>(p, units, st);
  } else if (tiles >= 2048 && tiles % 4 == 0) {
    launch_gemv_q4_shape<EPI, G, MT, 4, 4, 1>(p, st);
  } else if (tiles >= 512 && tiles % 2 == 0) {
    launch_gemv_q4_shape<EPI, G, MT, 4, 2, 1>(p, st);
  } else if (units > 16) {
    launch_gemv_q4_shape<EPI, G, MT, 16, 1, 1>(p, st);
  } else {
    launch_gemv_q4_shape<EPI, G, MT, 4, 1, 3>(p, st);
  }
}

template <int EPI, int G>
static void launch_gemv_q4_group(const GemvQ4Params& p, hipStream_t st) {
  if (p.M > 16) launch_gemv_q4_rows<EPI, G, 2>(p, st);
  else launch_gemv_q4_rows<EPI, G, 1>(p, st);
  if (p.splits > 1) {
    const int mts = p.M > 16 ? 2 : 1;
    hipLaunchKernelGGL((gemv_q4_join_kernel<EPI>), dim3(p.N / 16 * mts), dim3(64), 0, st, p, mts);
  }
}

template <int EPI>
static void launch_gemv_q4_epi(const GemvQ4Params& p, hipStream_t st) {
  if (p.group == 32) launch_gemv_q4_group<EPI, 32>(p, st);
  else if (p.group == 64) launch_gemv_q4_group<EPI, 64>(p, st);
  else launch_gemv_q4_group<EPI, 128>(p, st);
}

hipError_t launch_gemv_q4(GemvQ4Params& p, void* ws, hipStream_t st) {
  p.splits = ws ? gemv_q4_splits(p.M, p.N, p.K) : 1;
  p.part = static_cast<float*>(ws);
  if (p.splits > 1) p.part_sq = p.part + p.splits * static_cast<int64_t>(p.N) * 16 * (p.M > 16 ? 2 : 1);
  if (p.epilogue == SAGA_GEMV_ADD) launch_gemv_q4_epi<SAGA_GEMV_ADD>(p, st);
  else if (p.epilogue == SAGA_GEMV_SILU_PAIRS) launch_gemv_q4_epi<SAGA_GEMV_SILU_PAIRS>(p, st);
  else launch_gemv_q4_epi<SAGA_GEMV_STORE>(p, st);
  return hipGetLastError();
}

// A block opens 16 rows of U units of 128 columns: thread (r, q) 8 columns of row r in each,
// four bytes in and 16 out, the 16 threads of a row 256 bytes of it; its loads are in flight
// together.  Bound by the bytes written: 17920 x 1536 (70 MB moved) 15.0 us with U 4, 18.2
// with U 1, which small weights take (960 x 2560: 4.0 against 4.5).
template <int U>
__global__ void __launch_bounds__(256) unpack_q4_kernel(UnpackQ4Params p) {
  int it = 0;
  while (it + 1 < p.n && static_cast<int>(blockIdx.x) >= p.item[it + 1].block0) ++it;
  const UnpackQ4Params::Item& w = p.item[it];
  const int units = (w.K + 127) / 128, runs = (units + U - 1) / U;
  const int blk = blockIdx.x - w.block0, tile = blk / runs, J0 = (blk - tile * runs) * U;
  const int r = threadIdx.x >> 4, q = threadIdx.x & 15;
  const char* codes = static_cast<const char*>(w.codes) + static_cast<int64_t>(tile) * units * 1024 + (16 * (q & 3) + r) * 16 + (q >> 2) * 4;
  const char* scales = static_cast<const char*>(w.scales) + static_cast<int64_t>(tile) * (w.K / w.group) * 64 + 4 * r;
  uint32_t c[U], sz[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int J = min(J0 + u, units - 1), k = min(128 * J + 8 * q, w.K - 8);
    c[u] = *reinterpret_cast<const uint32_t*>(codes + static_cast<int64_t>(J) * 1024);
    sz[u] = *reinterpret_cast<const uint32_t*>(scales + static_cast<int64_t>(k / w.group) * 64);
  }
  const int n = tile * 16 + r;
  int dst = n;
  if (w.head_rows > 0) {
    const int h = n / w.head_rows, j = n - h * w.head_rows;
    if (h < w.rot_heads) dst = h * w.head_rows + (j & 1) * (w.head_rows / 2) + j / 2;
  }
  uint16_t* out = static_cast<uint16_t*>(w.dst) + static_cast<int64_t>(dst) * w.dst_ld;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int k = 128 * (J0 + u) + 8 * q;
    if (k >= w.K) return;
    const float sc = q4_lo(sz[u]), z = q4_hi(sz[u]);
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // columns 2 e and 2 e + 1: nibbles e and e + 4
      const float a = sc * static_cast<float>((c[u] >> (4 * e)) & 15u) + z;
      const float b = sc * static_cast<float>((c[u] >> (4 * e + 16)) & 15u) + z;
      o[e] = q4_bf16_pair(a, b);
    }
    *reinterpret_cast<u32x4*>(out + k) = o;
  }
}

hipError_t launch_unpack_q4(UnpackQ4Params& p, hipStream_t st) {
  auto layout = [&](int u) {
    int64_t blocks = 0;
    for (int i = 0; i < p.n; ++i) {
      p.item[i].block0 = static_cast<int>(std::min<int64_t>(blocks, 1LL << 24));
      blocks += static_cast<int64_t>(p.item[i].N / 16) * ((p.item[i].K + 128 * u - 1) / (128 * u));
    }
    return blocks;
  };
  int64_t blocks = layout(4);
  const bool few = blocks < 1024;
  if (few) blocks = layout(1);
  if (blocks >= (1LL << 24)) return hipErrorInvalidValue;  // a launch holds less than 2^32 threads
  if (few) hipLaunchKernelGGL((unpack_q4_kernel<1>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((unpack_q4_kernel<4>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace saga
