// Kernel 2 of the attention over 4- and 8-bit caches: the splits of a head joined.  P (DenseQ4Params,
// DenseFp8Params): b, q_h, nsplit; part: sums [b * q_h][nsplit][d], then (reference, sum of weights)
// [b * q_h][nsplit][2]; out.
#pragma once

#include "kernels.h"
#include "q4.cuh"

namespace saga {

// Joins a head's splits: one block per (batch row, head, JD dims), GR x JD threads; thread
// (grp, i) sums dim i of the splits grp, grp + GR, ..., the groups add up in a
// fixed order.  A round's sums are loaded before its references are known, so that a
// call of at most 8 GR splits waits for memory once.  More than 64 splits (few units, long
// rows) are read by more blocks, of 32 dims each: 1 x 32768 positions (12 heads, 256 splits)
// 15.1 -> 12.2 us with the first kernel; at 64 splits (8 x 32768) 21.3 -> 22.4.
constexpr int kJoinSplits = 1024;

template <class P, int D, int JD, int GR>
__device__ __forceinline__ void dense_join(const P& p, int block) {
  constexpr int NT = GR * JD;
  __shared__ float fm[kJoinSplits];
  __shared__ float red[NT / kWave];
  __shared__ float og[GR][JD];
  const int tid = threadIdx.x, grp = tid / JD, i = tid - grp * JD;
  const int row = block / (D / JD), d0 = (block - row * (D / JD)) * JD;
  const int bi = row / p.q_h, h = row - bi * p.q_h;
  const float* base = p.part + static_cast<int64_t>(row) * p.nsplit * D + d0 + i;
  const float2* ml = reinterpret_cast<const float2*>(p.part + static_cast<int64_t>(p.b) * p.q_h * p.nsplit * D) +
                     static_cast<int64_t>(row) * p.nsplit;
  float ov[8];
  auto load_round = [&](int q0) {
#pragma unroll
    for (int u = 0; u < 8; ++u) ov[u] = base[min(q0 + GR * u, p.nsplit - 1) * D];
  };
  load_round(grp);
  float2 v[kJoinSplits / NT];
  float mloc = kNegInf;
#pragma unroll
  for (int k = 0; k < kJoinSplits / NT; ++k) {
    const int q = tid + k * NT;
    v[k] = q < p.nsplit ? ml[q] : float2{kNegInf, 0.f};
    mloc = fmaxf(mloc, v[k].x);
  }
  const float M = block_max<NT / kWave>(mloc, red);
  float lloc = 0.f;
#pragma unroll
  for (int k = 0; k < kJoinSplits / NT; ++k) {
    const float f = v[k].x == kNegInf ? (v[k].y == 0.f ? 0.f : 1.f) : __expf(v[k].x - M);
    lloc += v[k].y * f;
    fm[tid + k * NT] = f;
  }
  const float l = block_sum<NT / kWave>(lloc, red);  // orders the writes of fm too
  float a = 0.f;
  for (int q0 = grp; q0 < p.nsplit; q0 += 8 * GR) {
    if (q0 != grp) load_round(q0);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (q0 + GR * u < p.nsplit) a += ov[u] * fm[q0 + GR * u];
  }
  og[grp][i] = a;
  __syncthreads();
  if (grp == 0) {
    float t = og[0][i];
#pragma unroll
    for (int q = 1; q < GR; ++q) t += og[q][i];
    store_from_f32(p.out, p.out_dt, bi * p.o_sb + static_cast<int64_t>(h) * p.o_sh + d0 + i, q4_in_range(t / l, p.out_dt));
  }
}

template <class P, int D, int JD, int GR>
__global__ void __launch_bounds__(GR * JD) dense_join_kernel(P p) {
  dense_join<P, D, JD, GR>(p, blockIdx.x);
}

template <int D, class P>
static void launch_dense_join(const P& p, hipStream_t st) {
  const unsigned rows = static_cast<unsigned>(p.b * p.q_h);
  if (p.nsplit > 64) hipLaunchKernelGGL((dense_join_kernel<P, D, 32, 32>), dim3(rows * (D / 32)), dim3(1024), 0, st, p);
  else hipLaunchKernelGGL((dense_join_kernel<P, D, D, 8>), dim3(rows), dim3(8 * D), 0, st, p);
}

}  // namespace saga
