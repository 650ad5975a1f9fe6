// Dense decode attention over an 8-bit cache (e4m3 numbers c, a scale per block of positions
// and head), split over the positions.
//
// A block takes one batch row, one unit of query heads (at most 16, the columns of every product:
// NV whole value heads of one key head, or a run of heads that share both) and one split of the
// positions; its waves step through 32 positions each, which lie in one block of the cache,
// and meet in LDS.  e4m3 numbers are exact in 16 bits, so that both products of a step
// are MFMAs with exact products and fp32 sums, and the scales are one factor each:
//   * x[h, j] = (scale s_k) q_h . c_j: key rows straight from memory as the A operand, in the
//     query's type;
//   * softmax with a running reference and sum in fp32: the reference moves only when a score
//     exceeds it by kFp8Slack nats, so most steps exchange and rescale nothing;
//   * o[h, i] += sum_j (p_hj s_v) c_ji: p s_v of the head's own value head is split into three bf16 terms,
//     which hold its 24 bits, an MFMA each (the third, under the loads: 22.8 -> 23.0 us at 8 x 32769, 193.5 ->
//     194.8 with weights at 32 x 65541; with two, f32 outputs there were off by 2.4e-6, now by 4.4e-7).
//     Lane (m, s) loads dims [m d / 16, + d / 16) of positions 8 s .. 8 s + 7 and pairs neighbouring
//     positions with byte permutes, so that values pass through no LDS; MFMA e has dim m d / 16 + e
//     in row m.
// Kernel 2 joins the splits.  With weights per position asked for, a step's scores go to memory, and
// kernel 2 has blocks that turn them into weights beside those that join.
// Bound by the cache's bytes: 12 / 1 / 2 heads of 128, 32 x 65541 positions (806 MB) 144 us with its
// join, 5.6 TB/s, 8 x 32769 (101 MB) 23.2 + 4.0 (one of 17 steps over four waves, two launches).  With
// weights 191 + 23 at 32 x 65541: 100 MB of scores written between the reads (906 MB at 4.7 TB/s, where a
// copy gets 5.1) and read; whole lines a store, stores past the caches and waits that leave the
// stores out were the same.  Two blocks a CU: three or four spill.
#include <algorithm>

#include "dense_join.cuh"
#include "fp8.cuh"
#include "kernels.h"
#include "weights.cuh"

namespace saga {

constexpr float kFp8Slack = 8.f;  // a weight is at most e^8

// First query head of the unit `seg` of heads that share a key and a value head, cut
// at 16, and how many it holds.
__device__ __forceinline__ int fp8_segment(int seg, int q_h, int g, int g_v, int& count) {
  int h = 0;
  for (int i = 0;; ++i) {
    const int e = min(min((h / g + 1) * g, (h / g_v + 1) * g_v), min(h + 16, q_h));
    if (i == seg) {
      count = e - h;
      return h;
    }
    h = e;
  }
}

static int fp8_segments(int q_h, int g, int g_v) {
  int n = 0;
  for (int h = 0; h < q_h; ++n) h = std::min(std::min((h / g + 1) * g, (h / g_v + 1) * g_v), h + 16);
  return n;
}

// A mask value out of the aligned word that holds it.
__device__ __forceinline__ float fp8_mask_value(uint32_t word, uint32_t shift, int dt) {
  if (dt == SAGA_DTYPE_F32) return __uint_as_float(word);
  word >>= shift;
  if (dt == SAGA_DTYPE_BF16) return bf16_bits_to_f32(word & 0xffffu);
  if (dt == SAGA_DTYPE_F16) return f16_bits_to_f32(static_cast<uint16_t>(word));
  return (word & 0xffu) ? 1.f : 0.f;
}

// Two floats as a pair of bf16 numbers; a and b keep what the rounding left over.
__device__ __forceinline__ uint32_t fp8_split(float& a, float& b) {
  const uint32_t w = q4_bf16_pair(a, b);
  a -= bf16_bits_to_f32(w & 0xffffu);
  b -= bf16_bits_to_f32(w >> 16);
  return w;
}

template <int DT, int D, int NV, bool MASK, bool TRACE>
__global__ void __launch_bounds__(256, 2) dense_fp8_kernel(DenseFp8Params p) {
  constexpr int NP = D / 64;   // 16-byte pieces of a key row per lane
  constexpr int NJ = D / 32;   // MFMA steps of a row
  constexpr int E = D / 16;    // value dims of a lane
  constexpr int WROW = D + 4;
  __shared__ __attribute__((aligned(16))) float lds[4 * 16 * (WROW + 2)];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, s = lane >> 4;
  const int split = blockIdx.x % p.nsplit;
  const int unit = blockIdx.x / p.nsplit;
  const int bi = unit / p.nseg;
  int nh = NV * p.g_v, h0 = (unit - bi * p.nseg) * nh;
  if constexpr (NV == 1) h0 = fp8_segment(unit - bi * p.nseg, p.q_h, p.g, p.g_v, nh);
  const int kh = h0 / p.g, vh0 = h0 / p.g_v;
  int Leff = p.L;
  if (p.kv_len) Leff = min(Leff, max(p.kv_len[bi], 0));
  const int h = h0 + (col < nh ? col : 0);
  const int u_mine = NV == 1 ? 0 : h / p.g_v - vh0;

  // step j of a row: dims 64 (j / 2) + 16 s + 8 (j % 2) .. of lane group s
  u32x4 qf[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j)
    qf[j] = ld16(p.q + (bi * p.q_sb + static_cast<int64_t>(h) * p.q_sh + 64 * (j / 2) + 16 * s + 8 * (j % 2)) * 2);

  const int beg = split * p.split_len;
  const int end = min(beg + p.split_len, Leff);
  const int nstep = end > beg ? (end - beg + 31) / 32 : 0;

  // A step's rows lie within 2^31 bytes of its first: a buffer per stream and step, whose
  // size ends with the split, so that rows past it load zeros (and touch no memory).
  // Row m of key tile t is position 8 (m / 4) + 4 t + m % 4: the rows 4 s + r that a lane's
  // scores are of are then its positions 8 s + i, i = 4 t + r.
  const char* kc = p.kv.kc + bi * p.kv.kc_sb + kh * p.kv.kc_sh + beg * p.kv.kc_sl;
  const char* vc = p.kv.vc + bi * p.kv.vc_sb + vh0 * p.kv.vc_sh + beg * p.kv.vc_sl;
  const float* ks = p.kv.ks + bi * p.kv.ks_sb + kh * p.kv.ks_sh;
  const float* vs = p.kv.vs + bi * p.kv.vs_sb + (vh0 + u_mine) * p.kv.vs_sh;
  const int kcl = static_cast<int>(p.kv.kc_sl), vcl = static_cast<int>(p.kv.vc_sl);
  const int krow = 8 * (col >> 2) + (col & 3);
  const int koff[2] = {krow * kcl + 16 * s, (krow + 4) * kcl + 16 * s};
  int voff[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) voff[i] = (8 * s + i) * vcl + E * col;

  struct Step {
    u32x4 k[2][NP];
    uint32_t v[NV][8][E / 4];
    float sk, sv;
    uint32_t m[MASK ? 8 : 1];
  };
  // The mask of this lane's positions, of any type: the aligned word that holds a value, and its
  // shift, so that a step's loads are one run without branches (a load under a branch is
  // waited for at the join).  A batch row's mask lies within 2^31 bytes.
  const int mes = p.mask_dt == SAGA_DTYPE_F32 ? 4 : p.mask_dt == SAGA_DTYPE_BOOL ? 1 : 2;
  const uint32_t mstep = static_cast<uint32_t>(p.m_sl) * mes;
  const uint64_t maddr = reinterpret_cast<uint64_t>(p.mask) + bi * p.m_sb * mes;
  const int mbytes = MASK ? static_cast<int>(maddr & 3) + static_cast<int>((p.q_h - 1) * p.m_sh + (p.L - 1) * p.m_sl + 1) * mes : 0;
  const uint32_t moff = static_cast<uint32_t>(maddr & 3) + static_cast<uint32_t>(h * p.m_sh) * mes + 8 * s * mstep;
  auto load_step = [&](Step& r, int it) {
    const int c0 = 32 * it, rows = min(max(end - beg - c0, 0), 32);  // from beg
    auto buffer = [&](const char* base, int64_t stride) {
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base + c0 * stride), 0,
                                               rows ? (rows - 1) * static_cast<int>(stride) + D : 0, 0x00027000);
    };
    const auto kb = buffer(kc, p.kv.kc_sl);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int j = 0; j < NP; ++j) r.k[t][j] = __builtin_amdgcn_raw_buffer_load_b128(kb, koff[t] + 64 * j, 0, 0);
    const int block = min(beg + c0, p.L - 1) >> p.kv.shift;
    r.sk = ks[block];
    r.sv = vs[block];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const auto vb = buffer(vc + u * p.kv.vc_sh, p.kv.vc_sl);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (E == 8) {
          const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(vb, voff[i], 0, 0);
          r.v[u][i][0] = v.x, r.v[u][i][1] = v.y;
        } else {
          r.v[u][i][0] = __builtin_amdgcn_raw_buffer_load_b32(vb, voff[i], 0, 0);
        }
      }
    }
    if constexpr (MASK) {
      const int64_t at = static_cast<int64_t>(beg + c0) * mstep, left = ((mbytes + 3) & ~3) - at;
      const auto mb = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char*>((maddr & ~uint64_t{3}) + at), 0,
                                                        left > 0 ? static_cast<int>(left) : 0, 0x00027000);
#pragma unroll
      for (int i = 0; i < 8; ++i) r.m[i] = __builtin_amdgcn_raw_buffer_load_b32(mb, (moff + i * mstep) & ~3u, 0, 0);
    }
  };

  Step ra, rb;
  load_step(ra, w);
  __builtin_amdgcn_sched_barrier(0);

  f32x4 o[NV][E];
#pragma unroll
  for (int u = 0; u < NV; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) o[u][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = kNegInf, l_run = 0.f;  // the reference of head `col`; the sum of this lane's positions

  auto use_step = [&](Step& r, int it) {
    const int c0 = beg + 32 * it;
    const float by = r.sk * p.scale;
    float x[8];  // positions c0 + 8 s + i
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const u32x4 k = r.k[t][j / 2];
        a = mfma_16b<DT>(j % 2 ? fp8_frag<DT>(k.z, k.w) : fp8_frag<DT>(k.x, k.y), qf[j], a);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * t + i] = a[i] * by;
    }
    if constexpr (MASK) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] + fp8_mask_value(r.m[i], 8 * ((moff + i * mstep) & 3), p.mask_dt);
    }
    if (c0 + 32 > end) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + 8 * s + i >= end) x[i] = kNegInf;
    }
    if constexpr (TRACE) {
      if (col < nh) {
        float* row = p.scores + (static_cast<int64_t>(bi) * p.q_h + h) * p.scores_ld + c0 + 8 * s;
        *reinterpret_cast<f32x4*>(row) = f32x4{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4*>(row + 4) = f32x4{x[4], x[5], x[6], x[7]};
      }
    }
    float mt = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mt = fmaxf(mt, x[i]);
    if (__any(mt > m_run + kFp8Slack)) {  // (from -inf on: any score)
      mt = fmaxf(mt, __shfl_xor(mt, 16));
      mt = fmaxf(mt, __shfl_xor(mt, 32));
      const float m_new = fmaxf(m_run, mt);
      const float alpha = m_run == kNegInf ? (m_new == kNegInf ? 1.f : 0.f) : __expf(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) o[u][e] *= alpha;
    }
    const float m_ref = m_run == kNegInf ? 0.f : m_run;  // (no score yet: weights of 0)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = __expf(x[i] - m_ref);
      l_run += x[i];
      x[i] *= r.sv;
    }
    u32x4 pf[3];
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) pf[k][i] = fp8_split(x[2 * i], x[2 * i + 1]);
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int c = 0; c < E / 4; ++c)
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // dims 4 c + 2 half and the next, of positions 2 i and 2 i + 1
          u32x4 a, b;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t two = __builtin_amdgcn_perm(r.v[u][2 * i + 1][c], r.v[u][2 * i][c], half ? 0x07030602u : 0x05010400u);
            a[i] = fp8_pair<SAGA_DTYPE_BF16, false>(two);
            b[i] = fp8_pair<SAGA_DTYPE_BF16, true>(two);
          }
          const int e = 4 * c + 2 * half;
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            o[u][e] = mfma_16b<SAGA_DTYPE_BF16>(a, pf[k], o[u][e]);
            o[u][e + 1] = mfma_16b<SAGA_DTYPE_BF16>(b, pf[k], o[u][e + 1]);
          }
        }
  };

  for (int it = w; it < nstep; it += 8) {
    load_step(rb, it + 4);
    __builtin_amdgcn_sched_barrier(0);
    use_step(ra, it);
    if (it + 4 >= nstep) break;
    load_step(ra, it + 8);
    __builtin_amdgcn_sched_barrier(0);
    use_step(rb, it + 4);
  }

  float* Wo = lds;
  float (*Wm)[16] = reinterpret_cast<float (*)[16]>(Wo + 4 * 16 * WROW);
  float (*Wl)[16] = Wm + 4;
  // the lanes of a head hold its positions between them
  l_run += __shfl_xor(l_run, 16);
  l_run += __shfl_xor(l_run, 32);
  if (s == 0) {
    Wm[w][col] = m_run;
    Wl[w][col] = l_run;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)  // rows 4 s + r: dims E (4 s + r) ..
#pragma unroll
    for (int e0 = 0; e0 < E; e0 += 4) {
      f32x4 a;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = o[0][e0 + e][r];
#pragma unroll
        for (int u = 1; u < NV; ++u) a[e] = u_mine == u ? o[u][e0 + e][r] : a[e];
      }
      *reinterpret_cast<f32x4*>(Wo + (w * 16 + col) * WROW + E * (4 * s + r) + e0) = a;
    }
  __syncthreads();

  // join the four waves: the split's partial, or the output when nsplit == 1
  float2* ml = reinterpret_cast<float2*>(p.part + static_cast<int64_t>(p.b) * p.q_h * p.nsplit * D);
  for (int e = tid; e < nh * D; e += 256) {
    const int hh = e / D, dd = e - hh * D;
    float M = kNegInf;
#pragma unroll
    for (int q = 0; q < 4; ++q) M = fmaxf(M, Wm[q][hh]);
    float l = 0.f, a = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float f = Wm[q][hh] == kNegInf ? (Wl[q][hh] == 0.f ? 0.f : 1.f) : __expf(Wm[q][hh] - M);
      l += Wl[q][hh] * f;
      a += Wo[(q * 16 + hh) * WROW + dd] * f;
    }
    const int64_t at = (static_cast<int64_t>(bi) * p.q_h + h0 + hh) * p.nsplit + split;
    if (p.nsplit == 1)
      store_from_f32(p.out, p.out_dt, bi * p.o_sb + static_cast<int64_t>(h0 + hh) * p.o_sh + dd, q4_in_range(a / l, p.out_dt));
    else
      p.part[at * D + dd] = a;
    if ((TRACE || p.nsplit > 1) && dd == 0) ml[at] = float2{M, l};
  }
}

template <int D>
__global__ void __launch_bounds__(256) dense_fp8_finish_kernel(DenseFp8Params p, WeightsParams w, int joins) {
  if (static_cast<int>(blockIdx.x) < joins) dense_join<DenseFp8Params, D, 32, 8>(p, blockIdx.x);
  else attention_weights(w, blockIdx.x - joins);
}

template <int D>
static hipError_t launch_dense_fp8_finish(const DenseFp8Params& p, WeightsParams* w, hipStream_t st) {
  if (!w) {
    if (p.nsplit > 1) launch_dense_join<D>(p, st);
    return hipSuccess;
  }
  w->scores = p.scores;
  w->s_ld = p.scores_ld;
  w->pm = p.part + static_cast<int64_t>(p.b) * p.q_h * p.nsplit * D;
  w->ps = w->pm + 1;
  w->pstride = 2;
  w->nparts = p.nsplit;
  // (to 64 splits a join in blocks of 32 dims adds in the order of one block of D: the same bits as without
  // weights; more are joined by 32 groups)
  if (p.nsplit > 64) launch_dense_join<D>(p, st);
  const int64_t joins = p.nsplit > 1 && p.nsplit <= 64 ? static_cast<int64_t>(p.b) * p.q_h * (D / 32) : 0;
  const int64_t blocks = joins + attention_weights_blocks(*w);
  if (blocks >= (1LL << 24)) return hipErrorInvalidValue;  // a launch holds less than 2^32 threads
  hipLaunchKernelGGL(dense_fp8_finish_kernel<D>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, p, *w,
                     static_cast<int>(joins));
  return hipSuccess;
}

template <int DT, int D, int NV>
static void launch_dense_fp8_typed(const DenseFp8Params& p, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.b * p.nseg * p.nsplit));
  if (p.mask) {
    if (p.scores) hipLaunchKernelGGL((dense_fp8_kernel<DT, D, NV, true, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((dense_fp8_kernel<DT, D, NV, true, false>), grid, dim3(256), 0, st, p);
  } else {
    if (p.scores) hipLaunchKernelGGL((dense_fp8_kernel<DT, D, NV, false, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((dense_fp8_kernel<DT, D, NV, false, false>), grid, dim3(256), 0, st, p);
  }
}

template <int DT, int D>
static void launch_dense_fp8_units(const DenseFp8Params& p, int nv, hipStream_t st) {
  if constexpr (D == 64) {
    if (nv == 5) return launch_dense_fp8_typed<DT, D, 5>(p, st);
  }
  if (nv == 2) return launch_dense_fp8_typed<DT, D, 2>(p, st);
  launch_dense_fp8_typed<DT, D, 1>(p, st);
}

hipError_t launch_dense_decode_fp8(DenseFp8Params& p, WeightsParams* w, hipStream_t st) {
  // Units of several whole value heads read and score their keys once for all of them: 5 (d 64) or 2
  // where a key head's count divides by that and 16 columns hold their query heads
  int nv = 1;
  if (p.g % p.g_v == 0) {
    const int n = p.g / p.g_v;
    if (p.kv.d == 64 && n % 5 == 0 && 5 * p.g_v <= 16) nv = 5;
    else if (n % 2 == 0 && 2 * p.g_v <= 16) nv = 2;
  }
  int64_t ns, sl;
  if (nv > 1) {  // (not where that leaves most CUs without a block)
    p.nseg = p.q_h / (nv * p.g_v);
    dense_q4_plan(static_cast<int64_t>(p.b) * p.nseg, p.L, &ns, &sl);
    if (p.b * p.nseg * ns < 128) nv = 1;
  }
  if (nv == 1) p.nseg = fp8_segments(p.q_h, p.g, p.g_v);
  dense_q4_plan(static_cast<int64_t>(p.b) * p.nseg, p.L, &ns, &sl);
  p.nsplit = static_cast<int32_t>(ns);
  p.split_len = static_cast<int32_t>(sl);
  if (p.b * p.nseg * ns >= (1LL << 24)) return hipErrorInvalidValue;  // a launch holds less than 2^32 threads
  const bool bf = p.q_dt == SAGA_DTYPE_BF16;
  if (p.kv.d == 128) {
    if (bf) launch_dense_fp8_units<SAGA_DTYPE_BF16, 128>(p, nv, st);
    else launch_dense_fp8_units<SAGA_DTYPE_F16, 128>(p, nv, st);
    const hipError_t e = launch_dense_fp8_finish<128>(p, w, st);
    if (e != hipSuccess) return e;
  } else {
    if (bf) launch_dense_fp8_units<SAGA_DTYPE_BF16, 64>(p, nv, st);
    else launch_dense_fp8_units<SAGA_DTYPE_F16, 64>(p, nv, st);
    const hipError_t e = launch_dense_fp8_finish<64>(p, w, st);
    if (e != hipSuccess) return e;
  }
  return hipGetLastError();
}

}  // namespace saga
