// The softmax weight that every cached position gathers over a step's query heads.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace saga {

// w (+)= sum_h exp(x_h - M_h) / l_h of one (batch row, group of query heads), where M_h and l_h come from
// the softmax's partial (reference, sum) pairs.  A head without a finite sum (no position, a NaN
// score) adds nothing.  A thread takes 4 positions and adds their heads in order.  Every block
// joins its heads' partials itself (a launch less), under the loads of its first scores.
// Bound by the scores, 4 bytes a head and position: 32 x 65544 positions of 12 heads (109 MB)
// 22 us, 4.9 TB/s; 8 x 33024 6.3 (a position a thread: 38 and 8.9).
// Blocks of 256 threads.
inline int64_t attention_weights_blocks(const WeightsParams& p) { return static_cast<int64_t>(p.b) * p.G * ((p.L + 1023LL) / 1024); }

constexpr int kWeightHeads = 64;  // heads whose (M, 1 / l) are held at a time

__device__ __forceinline__ void attention_weights(const WeightsParams& p, int block) {
  constexpr int PER = 4, TH = 4;  // positions of a thread, heads whose scores are in flight at a time
  __shared__ float fm[kWeightHeads], fr[kWeightHeads];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nchunk = (p.L + 256 * PER - 1) / (256 * PER);
  const int row = block / nchunk, pos0 = (block - row * nchunk) * 256 * PER, pos = pos0 + tid * PER;
  const int bi = row / p.G, gi = row - bi * p.G, gq = p.q_h / p.G;
  int Leff = p.L;
  if (p.kv_len) Leff = min(Leff, max(p.kv_len[bi], 0));
  float* w = p.w + bi * p.w_sb + gi * p.w_sg + pos;
  if (pos0 >= Leff) {
    if (!p.add)
      for (int e = 0; e < PER; ++e)
        if (pos + e < p.L) w[e] = 0.f;
    return;
  }
  const int64_t r0 = static_cast<int64_t>(bi) * p.q_h + gi * gq;
  const float* x0 = p.scores + r0 * p.s_ld + min(pos, (Leff - 1) / PER * PER);
  f32x4 x[TH];
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < TH; ++i) x[i] = *reinterpret_cast<const f32x4*>(x0 + min(h + i, gq - 1) * p.s_ld);
  };
  load(0);
  float acc[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
  for (int hb = 0; hb < gq; hb += kWeightHeads) {
    const int n = min(gq - hb, kWeightHeads);
    if (hb) __syncthreads();
    for (int i = wave; i < n; i += 4) {
      const int64_t base = (r0 + hb + i) * p.nparts;
      float m = kNegInf, l = 0.f;  // (an empty part holds (-inf, 0), one of NaN scores a NaN sum)
      for (int q0 = lane; q0 < p.nparts; q0 += 256) {
        float pm[4], ps[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int64_t at = (base + min(q0 + 64 * u, p.nparts - 1)) * p.pstride;
          pm[u] = q0 + 64 * u < p.nparts ? p.pm[at] : kNegInf;
          ps[u] = q0 + 64 * u < p.nparts ? p.ps[at] : 0.f;
        }
        const float mn = fmaxf(fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])), m);
        l = m == kNegInf ? l : l * __expf(m - mn);
#pragma unroll
        for (int u = 0; u < 4; ++u) l += pm[u] == kNegInf ? ps[u] : ps[u] * __expf(pm[u] - mn);
        m = mn;
      }
      const float M = wave_max(m);
      l = wave_sum(m == kNegInf ? l : l * __expf(m - M));
      if (lane == 0) {
        const bool some = l > 0.f && l < __builtin_inff();
        fm[i] = some ? M : __builtin_inff();
        fr[i] = some ? 1.f / l : 0.f;
      }
    }
    __syncthreads();
    for (int h = 0; h < n; h += TH) {
      f32x4 y[TH];
#pragma unroll
      for (int i = 0; i < TH; ++i) y[i] = x[i];
      load(hb + h + TH);
#pragma unroll
      for (int i = 0; i < TH; ++i) {
        const int at = min(h + i, kWeightHeads - 1);
        const float m = fm[at], r = h + i < n ? fr[at] : 0.f;
        if (r > 0.f) {
#pragma unroll
          for (int e = 0; e < PER; ++e) acc[e] += __expf(y[i][e] - m) * r;
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    if (pos + e < Leff) w[e] = p.add ? w[e] + acc[e] : acc[e];
    else if (pos + e < p.L && !p.add) w[e] = 0.f;
  }
}

}  // namespace saga
