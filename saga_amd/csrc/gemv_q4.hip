// Skinny GEMM with weights in 4 bits: y[m, n] = sum_k x[m, k] (s c + z)[n, k], m < 32.
//
// The weight stream of gemv.hip with a quarter of its bytes.  x is the A operand
// (token rows), 16 rows of W the B operand: a lane then holds one row n of the
// product and needs one (s, z) pair per group.  Per group of G columns
//   sum_k x (s c + z) = s sum_k x (16 + c) + (z - 16 s) sum_k x,
// the first sum an MFMA chain over the codes as 16 + c (q4.cuh), the second one
// over ones, both exact products summed in fp32.  The RMSNorm's sum of squares is
// the diagonal of x x^T, an MFMA more per fragment.
#include <algorithm>

#include "kernels.h"
#include "q4.cuh"

namespace saga {

__device__ __forceinline__ f32x4 mfma_bf16(const u32x4& a, const u32x4& b, f32x4 c) {
  return mfma_16b<SAGA_DTYPE_BF16>(a, b, c);
}

// Workgroup: TPW tiles of 16 rows of W, its waves split K by units of 128
// columns (wave w takes units w, w + WAVES, ...) and meet in LDS.  U units per
// wave in flight.  MT tiles of 16 token rows.
template <int EPI, int G, int MT, int WAVES, int TPW, int U>
__global__ void __launch_bounds__(WAVES * 64) gemv_q4_kernel(GemvQ4Params p) {
  constexpr int NG = 128 / G;  // groups of a unit
  __shared__ float red[WAVES][TPW * MT][64][4];
  __shared__ float rsq[WAVES][16 * MT];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int col = lane & 15, s = lane >> 4;
  const int tile0 = blockIdx.x * TPW;
  const int units = (p.K + 127) / 128, steps = p.K / 32, groups = p.K / G;
  const char* code = static_cast<const char*>(p.codes) + static_cast<int64_t>(tile0) * units * 1024 + lane * 16;
  const char* scale = static_cast<const char*>(p.scales) + static_cast<int64_t>(tile0) * groups * 64 + col * 4;
  const char* xrow[MT];
  bool xvalid[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    xvalid[mt] = col + 16 * mt < p.M;
    xrow[mt] = static_cast<const char*>(p.x) + (static_cast<int64_t>(xvalid[mt] ? col + 16 * mt : 0) * p.x_ld + 8 * s) * 2;
  }
  f32x4 acc[TPW][MT], sq[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    sq[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < TPW; ++t) acc[t][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const u32x4 ones = {kBf16Ones, kBf16Ones, kBf16Ones, kBf16Ones};
  for (int u0 = w; u0 < units; u0 += U * WAVES) {
    u32x4 cw[U][TPW], xf[U][MT][4];
    uint32_t sz[U][TPW][NG];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int J = min(u0 + u * WAVES, units - 1);
      const bool live = u0 + u * WAVES < units;
#pragma unroll
      for (int t = 0; t < TPW; ++t) {
        cw[u][t] = ld16(code + (static_cast<int64_t>(t) * units + J) * 1024);
#pragma unroll
        for (int g = 0; g < NG; ++g)
          sz[u][t][g] = *reinterpret_cast<const uint32_t*>(scale + (static_cast<int64_t>(t) * groups + min(J * NG + g, groups - 1)) * 64);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          xf[u][mt][j] = live && xvalid[mt] && 4 * J + j < steps ? ld16(xrow[mt] + static_cast<int64_t>(4 * J + j) * 64)
                                                                : u32x4{0u, 0u, 0u, 0u};
    }
    __builtin_amdgcn_sched_barrier(0);  // the whole burst is in flight
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p.rms) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int j = 0; j < 4; ++j) sq[mt] = mfma_bf16(xf[u][mt][j], xf[u][mt][j], sq[mt]);
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        f32x4 xs[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          xs[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = g * (G / 32); j < (g + 1) * (G / 32); ++j) xs[mt] = mfma_bf16(xf[u][mt][j], ones, xs[mt]);
        }
#pragma unroll
        for (int t = 0; t < TPW; ++t) {
          f32x4 d[MT];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) d[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = g * (G / 32); j < (g + 1) * (G / 32); ++j) {
            const u32x4 b = q4_frag(cw[u][t][j]);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) d[mt] = mfma_bf16(xf[u][mt][j], b, d[mt]);
          }
          const float sc = q4_lo(sz[u][t][g]), zo = __builtin_fmaf(-16.f, sc, q4_hi(sz[u][t][g]));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              acc[t][mt][r] = __builtin_fmaf(sc, d[mt][r], __builtin_fmaf(zo, xs[mt][r], acc[t][mt][r]));
        }
      }
    }
  }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int t = 0; t < TPW; ++t)
      *reinterpret_cast<f32x4*>(red[w][t * MT + mt][lane]) = acc[t][mt];
    // the diagonal: row 4 s + r of lane column 4 s + r
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (col == 4 * s + r) rsq[w][16 * mt + col] = sq[mt][r];
  }
  lds_sync();
  // one (tile, token tile) per wave: lane (col, s) holds rows n of tokens 4 s + r
  for (int i = w; i < TPW * MT; i += WAVES) {
    const int t = i / MT, mt = i - t * MT;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < WAVES; ++q) v += *reinterpret_cast<const f32x4*>(red[q][i][lane]);
    const int n = (tile0 + t) * 16 + col;
    float bias = 0.f;
    if (EPI != SAGA_GEMV_SILU_PAIRS && p.bias) bias = bf16_bits_to_f32(static_cast<const uint16_t*>(p.bias)[n]);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = 16 * mt + 4 * s + r;
      float scl = 1.f;
      if (p.rms) {
        float q2 = 0.f;
#pragma unroll
        for (int q = 0; q < WAVES; ++q) q2 += rsq[q][m];
        scl = rsqrtf(q2 / static_cast<float>(p.K) + p.eps);
      }
      float o = v[r] * scl;
      uint16_t* y = static_cast<uint16_t*>(p.y) + static_cast<int64_t>(m) * p.y_ld;
      if constexpr (EPI == SAGA_GEMV_SILU_PAIRS) {
        const float up = __shfl_xor(o, 1);  // rows (n, n + 1): gate, up
        if (m < p.M && (col & 1) == 0) y[n / 2] = f32_to_bf16_bits(o / (1.0f + expf(-o)) * up);
      } else {
        if (p.bias) o += bias;
        if (m < p.M) {
          if constexpr (EPI == SAGA_GEMV_ADD) o += bf16_bits_to_f32(y[n]);
          y[n] = f32_to_bf16_bits(o);
        }
      }
    }
  }
}

int64_t gemv_q4_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  (void)M, (void)N, (void)K;
  return 0;
}

template <int EPI, int G>
static void launch_gemv_q4_group(const GemvQ4Params& p, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.N / 16));
  if (p.M > 16) hipLaunchKernelGGL((gemv_q4_kernel<EPI, G, 2, 8, 1, 2>), grid, dim3(512), 0, st, p);
  else hipLaunchKernelGGL((gemv_q4_kernel<EPI, G, 1, 4, 1, 3>), grid, dim3(256), 0, st, p);
}

template <int EPI>
static void launch_gemv_q4_epi(const GemvQ4Params& p, hipStream_t st) {
  if (p.group == 32) launch_gemv_q4_group<EPI, 32>(p, st);
  else if (p.group == 64) launch_gemv_q4_group<EPI, 64>(p, st);
  else launch_gemv_q4_group<EPI, 128>(p, st);
}

hipError_t launch_gemv_q4(const GemvQ4Params& p, void* ws, hipStream_t st) {
  (void)ws;
  if (p.epilogue == SAGA_GEMV_ADD) launch_gemv_q4_epi<SAGA_GEMV_ADD>(p, st);
  else if (p.epilogue == SAGA_GEMV_SILU_PAIRS) launch_gemv_q4_epi<SAGA_GEMV_SILU_PAIRS>(p, st);
  else launch_gemv_q4_epi<SAGA_GEMV_STORE>(p, st);
  return hipGetLastError();
}

// A block opens 16 rows x 128 columns: thread (r, q) 8 columns of row r, four
// bytes in and 16 out, the 16 threads of a row 256 bytes of it.
__global__ void __launch_bounds__(256) unpack_q4_kernel(UnpackQ4Params p) {
  int it = 0;
  while (it + 1 < p.n && static_cast<int>(blockIdx.x) >= p.item[it + 1].block0) ++it;
  const UnpackQ4Params::Item& w = p.item[it];
  const int units = (w.K + 127) / 128;
  const int blk = blockIdx.x - w.block0, tile = blk / units, J = blk - tile * units;
  const int r = threadIdx.x >> 4, q = threadIdx.x & 15, k = 128 * J + 8 * q;
  if (k >= w.K) return;
  const uint32_t c = *reinterpret_cast<const uint32_t*>(static_cast<const char*>(w.codes) +
                                                        (static_cast<int64_t>(tile) * units + J) * 1024 +
                                                        (16 * (q & 3) + r) * 16 + (q >> 2) * 4);
  const uint32_t sz = *reinterpret_cast<const uint32_t*>(
      static_cast<const char*>(w.scales) + (static_cast<int64_t>(tile) * (w.K / w.group) + k / w.group) * 64 + 4 * r);
  const float sc = q4_lo(sz), z = q4_hi(sz);
  u32x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) {  // columns 2 e and 2 e + 1: nibbles e and e + 4
    const float a = sc * static_cast<float>((c >> (4 * e)) & 15u) + z;
    const float b = sc * static_cast<float>((c >> (4 * e + 16)) & 15u) + z;
    o[e] = f32_to_bf16_bits(a) | (static_cast<uint32_t>(f32_to_bf16_bits(b)) << 16);
  }
  const int n = tile * 16 + r;
  int dst = n;
  if (w.head_rows > 0) {
    const int h = n / w.head_rows, j = n - h * w.head_rows;
    if (h < w.rot_heads) dst = h * w.head_rows + (j & 1) * (w.head_rows / 2) + j / 2;
  }
  *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(w.dst) + static_cast<int64_t>(dst) * w.dst_ld + k) = o;
}

hipError_t launch_unpack_q4(UnpackQ4Params& p, hipStream_t st) {
  int64_t blocks = 0;
  for (int i = 0; i < p.n; ++i) {
    p.item[i].block0 = static_cast<int>(blocks);
    blocks += static_cast<int64_t>(p.item[i].N / 16) * ((p.item[i].K + 127) / 128);
    if (blocks >= (1LL << 24)) return hipErrorInvalidValue;  // a launch holds less than 2^32 threads
  }
  hipLaunchKernelGGL(unpack_q4_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace saga
